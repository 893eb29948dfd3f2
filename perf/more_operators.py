"""Workloads of speculative decoding over the paged KV cache.

A step that checks a tree of drafted tokens makes four calls besides the plan and its
Linears: the cache write with a norm for each head of q and k (a layer), the attention in
which a drafted token sees the cached ones and its ancestors in the tree (a layer), the log
probabilities of the drafted tokens under the model's logits (a step), and the move of the
accepted path's keys and values to the places that follow the cached ones, in all layers,
with the pages of the others given back (a step).  ``run`` makes one of them, through
``llmengine_amd.capi`` where ``own`` is true and in plain torch operations where it is not.
Head counts, sizes and vocabularies are those of the benchmark's models (Llama-7B: 32 heads of
128, 32000 tokens; Qwen2.5-0.5B: 14 heads of 64 over 2 KV heads, 151936 tokens) or generic
grouped layouts.

The cache's layout is the framework's: pages hold, per KV head, tiles of 16 tokens; element
(token, d) of a K tile is at [d / 8][token][d % 8], of a V tile at
[token / 4 % 2][d][token / 8][token % 4].
"""
from __future__ import annotations

import math
import random

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
TILE = 16                               # tokens of a cache tile
WORD = 64                               # nodes of a word of a tree's mask
MAX_SCORES = 32 * 64 * 8 * 32768        # padded scores of the plain form, largest listed
MAX_CACHE = 8 * 32768 * 8 * 128         # padded cache elements, largest listed
MAX_LOGITS = 1024 * 151936
MAX_CELLS = 32 * 32 * 80 * 8 * 128      # elements of K in all layers' pages, largest listed


def listed():
    return [
        # The drafted tokens of a few requests, q/k/v in one buffer of the fused Linear.
        {"name": "write_normed_37", "kind": "write", "type": "bf16", "heads": 14,
         "kv_heads": 2, "dim": 64, "page": 16, "tokens": 37, "rope": "halves", "fused": True,
         "mix": 1},
        # A long prompt into an 8-bit cache.
        {"name": "write_normed_int8_8192", "kind": "write", "type": "int8", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "tokens": 8192, "rope": "halves",
         "fused": False, "mix": 2},
        # Smallest: one request, a tree of 8 drafted tokens over a short context.
        {"name": "tree_1x8", "kind": "tree", "type": "f16", "heads": 14, "kv_heads": 2,
         "dim": 64, "page": 16, "seqs": 1, "nodes": 8, "chunk": 0, "chunked": 0, "kv": 129,
         "window": 0, "mix": 3},
        # A batch of a 7B model, no grouped heads: 26 drafted tokens each.
        {"name": "tree_16x26", "kind": "tree", "type": "f16", "heads": 32, "kv_heads": 32,
         "dim": 128, "page": 16, "seqs": 16, "nodes": 26, "chunk": 0, "chunked": 0,
         "kv": 4096, "window": 0, "mix": 4},
        # Long contexts on an 8-bit cache, grouped heads, trees of 64: the largest case.
        {"name": "tree_int8_8x64", "kind": "tree", "type": "int8", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "seqs": 8, "nodes": 64, "chunk": 0, "chunked": 0,
         "kv": 32768, "window": 0, "mix": 5},
        # Small trees beside the chunk of a prompt, through a sliding window.
        {"name": "tree_bf16_mixed", "kind": "tree", "type": "bf16", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 32, "seqs": 16, "nodes": 11, "chunk": 300, "chunked": 1,
         "kv": 4096, "window": 1024, "mix": 6},
        # Wide trees, whose masks take several words, of few requests.
        {"name": "tree_3x200", "kind": "tree", "type": "f16", "heads": 28, "kv_heads": 4,
         "dim": 128, "page": 32, "seqs": 3, "nodes": 200, "chunk": 0, "chunked": 0,
         "kv": 9001, "window": 0, "mix": 7},
        # The token that one request got, with its probability only.
        {"name": "logprobs_1x151936", "kind": "logprobs", "rows": 1, "vocab": 151936,
         "given": 1, "top": 0, "temperature": 1.0, "padded": 0},
        # Drafted children of a batch's nodes, with alternatives, under a temperature.
        {"name": "logprobs_208x32000", "kind": "logprobs", "rows": 208, "vocab": 32000,
         "given": 4, "top": 5, "temperature": 0.7, "padded": 0},
        # Scoring of a whole prompt, with as many alternatives as interfaces give.
        {"name": "logprobs_1024x151936", "kind": "logprobs", "rows": 1024, "vocab": 151936,
         "given": 1, "top": 20, "temperature": 1.0, "padded": 271},
        # One request's path in the 24 layers of a 0.5B model.
        {"name": "keep_1x8", "kind": "keep", "type": "f16", "kv_heads": 2, "dim": 64,
         "page": 16, "layers": 24, "seqs": 1, "nodes": 8, "chunked": 0, "kv": 700, "mix": 11},
        # A batch's paths in 32 layers of an 8-bit cache.
        {"name": "keep_int8_32x64", "kind": "keep", "type": "int8", "kv_heads": 8, "dim": 128,
         "page": 16, "layers": 32, "seqs": 32, "nodes": 64, "chunked": 2, "kv": 4096,
         "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(heads, KV heads, head size)"""
    return rng.choice([(14, 2, 64), (32, 32, 128), (32, 8, 128), (16, 4, 96), (8, 1, 256),
                       (12, 12, 64), (28, 4, 128), (20, 5, 128)])


def draw(rng):
    kind = rng.choice(["write", "tree", "tree", "tree", "logprobs", "logprobs", "keep"])
    mix = rng.randint(0, 1 << 30)
    if kind == "logprobs":
        vocab = _log_int(rng, 1000, 262144)
        rows = max(1, min(_log_int(rng, 1, 4096), MAX_LOGITS // vocab))
        return {"kind": kind, "rows": rows, "vocab": vocab, "given": rng.choice([0, 1, 1, 3, 8]),
                "top": rng.choice([0, 1, 5, 20, 50, 128]),
                "temperature": rng.choice([1.0, 1.0, 0.6, 1.3]),
                "padded": rng.choice([0, 0, vocab // 50])}
    page = rng.choice([16, 32, 64, 128])
    heads, kv_heads, dim = _heads(rng)
    kv_type = rng.choice(["f16", "f16", "bf16", "int8"])
    if kind == "write":
        return {"kind": kind, "type": kv_type, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "page": page, "tokens": _log_int(rng, 1, 8192),
                "rope": rng.choice(["halves", "halves", "pairs", "none"]),
                "fused": rng.random() < 0.5, "mix": mix}
    nodes = _log_int(rng, 1, 256)
    if kind == "keep":
        nodes = min(nodes, 128)
        layers = _log_int(rng, 1, 80)
        held = (nodes + 2 * page) * kv_heads * dim * layers
        seqs = max(1, min(_log_int(rng, 1, 64), MAX_CELLS // held))
        return {"kind": kind, "type": kv_type, "kv_heads": kv_heads, "dim": dim, "page": page,
                "layers": layers, "seqs": seqs, "nodes": nodes,
                "chunked": rng.choice([0, 0, seqs // 4]), "kv": _log_int(rng, 1, 16000),
                "mix": mix}
    kv = _log_int(rng, 1, 32768) + nodes
    seqs = _log_int(rng, 1, 64)
    seqs = max(1, min(seqs, MAX_CACHE // (kv * kv_heads * dim),
                      MAX_SCORES // (kv * heads * nodes)))
    nodes = max(1, min(nodes, MAX_SCORES // (kv * heads * seqs)))
    chunk = chunked = 0
    if rng.random() < 0.25:
        chunk = min(_log_int(rng, 2, 1024), MAX_SCORES // (kv * heads * seqs))
        chunked = min(seqs, rng.randint(1, 3)) if 1 < chunk <= kv else 0
    return {"kind": kind, "type": kv_type, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "seqs": seqs, "nodes": nodes, "chunk": chunk if chunked else 0,
            "chunked": chunked, "kv": kv, "window": rng.choice([0, 0, 0, 100, 1024]), "mix": mix}


def _pages(length, page):
    return -(-length // page)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prefix(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _capi():
    from llmengine_amd import capi
    return capi


def _pool(case, pages, k, v, k_scale=None, v_scale=None):
    """The cache's handle: its buffers, and the framework's object for them."""
    pool = {"k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "pages": pages}
    if own:
        pool["cache"] = _capi().PagedCache(case["type"], pages, case["page"], case["kv_heads"],
                                           case["dim"], k, v, k_scale, v_scale)
    return pool


def _requests(case):
    """(new rows, tokens in all, whether they are a tree) of each request: the first `chunked`
    have a chunk of a prompt, the others a tree of nodes / 2 .. nodes drafted tokens; the first
    is as long as any, the others spread over a factor of 16."""
    rng = random.Random(case["mix"])
    out = []
    for b in range(case["seqs"]):
        total = case["kv"] if b == 0 else max(1, int(case["kv"] * 16 ** -rng.random()))
        tree = b >= case["chunked"]
        size = case["nodes"] if tree else case["chunk"]
        new = size if b in (0, case["chunked"]) else max(1, int(size * rng.uniform(0.5, 1)))
        out.append((new, max(total, new), tree))
    return out


def _tree(rng, n):
    """Parents of n drafted tokens, the root first, some branches longer than others."""
    return [-1] + [rng.randrange(max(0, i - 1 - rng.randrange(12)), i) for i in range(1, n)]


# ---- the write ------------------------------------------------------------------------------

def _prepare_write(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, G, D, page, T = (case["heads"], case["kv_heads"], case["dim"], case["page"],
                        case["tokens"])
    # Rows as the Linears leave them: of different sizes from head to head.
    size = torch.exp(torch.randn(H + 2 * G, 1, generator=gen, device="cuda"))
    qkv = torch.randn(T, H + 2 * G, D, generator=gen, device="cuda") * size
    q, k, v = qkv.view(T, -1).split([H * D, G * D, G * D], dim=1)
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    norms = [1.0 + 0.3 * torch.randn(D, generator=gen, device="cuda") for _ in range(2)]
    # Up to 32 sequences; a chunk starts anywhere in its sequence, its pages anywhere.
    rng = random.Random(case["mix"])
    seqs = min(32, max(1, T // 64)) if T > 32 else T
    cuts = [0] + sorted(rng.sample(range(1, T), seqs - 1)) + [T]
    pages = sum(_pages(b - a, page) + 1 for a, b in zip(cuts, cuts[1:]))
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    positions, slots, at = [], [], 0
    for a, b in zip(cuts, cuts[1:]):
        start = rng.randrange(0, 8000)
        n = _pages(start % page + b - a, page)
        mine = order[at:at + n]
        at += n
        positions += range(start, start + b - a)
        slots += [mine[i // page] * page + i % page
                  for i in range(start % page, start % page + b - a)]
    limit = 8000 + T
    st = {"case": case, "q": q, "k": k, "v": v, "q_norm": norms[0], "k_norm": norms[1],
          "eps": 1e-6, "positions": _int32(positions), "slots": _int32(slots),
          "q_out": torch.empty(T, H * D, device="cuda"), "rope": None, "limit": 0}
    if case["rope"] != "none":
        angle = (torch.arange(limit, device="cuda", dtype=torch.float64)[:, None] *
                 1e6 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        st["rope"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
        st["limit"] = limit
    cells = pages * G * page
    k, v = (torch.zeros(cells * D, dtype=TYPES[case["type"]], device="cuda") for _ in range(2))
    scales = [None, None]
    if case["type"] == "int8":
        scales = [torch.zeros(cells, device="cuda") for _ in range(2)]
    st["pool"] = _pool(case, pages, k, v, *scales)
    return st


def _normed_rotated(x, weight, st, mode):
    """[T, heads, D] normed over D and rotated in 64 bits: values beside the borders of 8-bit
    cells."""
    x = x.double()
    x = x / (x.square().mean(-1, keepdim=True) + st["eps"]).sqrt() * weight.double()
    if mode == "none":
        return x
    cos, sin = st["rope"][st["positions"].long()].double()[:, None].unbind(-1)
    D = x.shape[-1]
    a, b = (x[..., :D // 2], x[..., D // 2:]) if mode == "halves" else (x[..., 0::2],
                                                                       x[..., 1::2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    return (torch.cat([ra, rb], -1) if mode == "halves"
            else torch.stack([ra, rb], -1).flatten(-2))


def _places(slot, case):
    """Flat index of the K and V elements of slots in the cache, and of their scales."""
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    head = torch.arange(G, device="cuda")
    cell = (slot // page)[:, None] * G + head          # (page, head)
    row, off = slot % page // TILE, slot % TILE
    tile = (cell * (page // TILE) + row[:, None]) * (TILE * D)
    d = torch.arange(D, device="cuda")
    at_k = tile[..., None] + (d // 8 * (TILE * 8) + d % 8) + (off * 8)[:, None, None]
    at_v = (tile[..., None] + d * 8
            + (off // 4 % 2 * (D * 8) + off // 8 * 4 + off % 4)[:, None, None])
    return at_k, at_v, cell * page + (slot % page)[:, None]


def _run_write(st):
    case, pool = st["case"], st["pool"]
    H, G, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    out = [st["q_out"], pool["k"], pool["v"]]
    if case["type"] == "int8":
        out += [pool["k_scale"], pool["v_scale"]]
    if own:
        _capi().paged_kv_write_normed(pool["cache"], st["q"], st["q_out"], H, st["k"], st["v"],
                                      st["q_norm"], st["k_norm"], st["eps"], st["rope"],
                                      st["limit"], D, case["rope"], st["positions"],
                                      st["slots"], T)
        return out
    q = _normed_rotated(st["q"].reshape(T, H, D), st["q_norm"], st, case["rope"])
    st["q_out"].copy_(q.flatten(1))
    k = _normed_rotated(st["k"].reshape(T, G, D), st["k_norm"], st, case["rope"]).float()
    v = st["v"].reshape(T, G, D)
    at_k, at_v, at_s = _places(st["slots"].long(), case)
    if case["type"] == "int8":
        k_scale, v_scale = (x.abs().amax(-1) * (1.0 / 127.0) for x in (k, v))
        pool["k_scale"][at_s], pool["v_scale"][at_s] = k_scale, v_scale
        k, v = ((x / s[..., None]).round() for x, s in ((k, k_scale), (v, v_scale)))
    pool["k"][at_k] = k.to(pool["k"].dtype)
    pool["v"][at_v] = v.to(pool["v"].dtype)
    return out


def _exact_write(case, seed):
    """From the definitions of norm, rotation and cells; 8-bit cells are whole numbers, which
    have no value in 64 bits."""
    st = _prepare_write(case, seed)
    H, G, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    turn = torch.ones(T, 1, max(1, D // 2), dtype=torch.complex128, device="cuda")
    if case["rope"] != "none":
        turn = torch.view_as_complex(st["rope"].double())[st["positions"].long()][:, None]
    halves = case["rope"] == "halves"

    def turned(x, n, weight):
        x = x.double().reshape(T, n, D)
        length = torch.linalg.vector_norm(x, dim=-1, keepdim=True)
        x = weight.double() * (x * torch.rsqrt(length * length / D + st["eps"]))
        pairs = x.reshape(T, n, 2, D // 2).transpose(2, 3) if halves else x.reshape(
            T, n, D // 2, 2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return (y.transpose(2, 3) if halves else y).reshape(T, n, D)

    k, v = turned(st["k"], G, st["k_norm"]), st["v"].double().reshape(T, G, D)
    q = turned(st["q"], H, st["q_norm"]).flatten(1)
    page = case["page"]
    slot = st["slots"].long()
    at = (slot // page, slice(None), slot % page)
    if case["type"] == "int8":
        out = [q, None, None]
        for x in (k, v):
            cells = torch.zeros(st["pool"]["pages"], G, page, dtype=torch.float64, device="cuda")
            cells[at] = x.abs().amax(-1) / 127
            out.append(cells.flatten())
        return out
    cells = torch.zeros(2, st["pool"]["pages"], G, page, D, dtype=torch.float64, device="cuda")
    cells[0][at], cells[1][at] = k, v
    k = cells[0].reshape(-1, TILE, D // 8, 8).transpose(1, 2)
    v = cells[1].reshape(-1, 2, 2, 4, D).permute(0, 2, 4, 1, 3)
    return [q, k.flatten(), v.flatten()]


# ---- the attention of a tree ----------------------------------------------------------------

def _prepare_tree(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    requests = _requests(case)
    need = [_pages(total, page) for _, total, _ in requests]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    max_pages = max(need) + 2
    table = torch.full((case["seqs"], max_pages), -1, dtype=torch.int32, device="cuda")
    for b, (at, n) in enumerate(zip(_prefix(need), need)):
        table[b, :n] = order[at:at + n]
    # Masks of the trees' rows, 64 nodes a word, and the rows' positions.
    rng = random.Random(seed)
    words = max([_pages(n, WORD) for n, _, tree in requests if tree], default=1)
    masks, positions = [], []
    for new, total, tree in requests:
        if not tree:
            masks += [0] * new
            positions += range(total - new, total)
            continue
        seen, depth = [], []
        for i, p in enumerate(_tree(rng, new)):
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            depth.append(depth[p] + 1 if p >= 0 else 0)
        masks += seen
        positions += [total - new + d for d in depth]
    signed = [[m >> WORD * w & (1 << WORD) - 1 for w in range(words)] for m in masks]
    signed = [[x - (1 << WORD) if x >> (WORD - 1) else x for x in row] for row in signed]
    T = len(masks)
    # Logits of a standard deviation of 2, so that some keys carry most of a row.
    q = 2.0 * torch.randn(T, H * D, generator=gen, device="cuda")
    size = (pages * G * page * D,)
    k_scale = v_scale = None
    if case["type"] == "int8":
        k, v = (torch.randint(-127, 128, size, generator=gen, device="cuda", dtype=torch.int8)
                for _ in range(2))
        k_scale, v_scale = ((0.5 + torch.rand(pages * G * page, generator=gen, device="cuda"))
                            / 73.0 for _ in range(2))
    else:
        k, v = (torch.randn(size, generator=gen, device="cuda", dtype=TYPES[case["type"]])
                for _ in range(2))
    return {"case": case, "q": q, "out": torch.empty_like(q), "table": table, "tokens": T,
            "max_pages": max_pages, "requests": requests, "words": words,
            "most": max(n for n, _, _ in requests),
            "mask": torch.tensor(signed, dtype=torch.int64, device="cuda"),
            "masks": masks, "depths": positions, "positions": _int32(positions),
            "trees": _int32([int(tree) for _, _, tree in requests]),
            "kv_lens": _int32([total for _, total, _ in requests]),
            "cu": _int32(_prefix([new for new, _, _ in requests])),
            "pool": _pool(case, pages, k, v, k_scale, v_scale)}


def _run_tree(st):
    case, pool = st["case"], st["pool"]
    H, G, D, page, B = (case["heads"], case["kv_heads"], case["dim"], case["page"],
                        case["seqs"])
    scale = D ** -0.5
    if own:
        _capi().paged_tree_attention(pool["cache"], st["q"], st["out"], H, scale,
                                     case["window"], st["table"], st["max_pages"],
                                     st["kv_lens"], st["cu"], B, st["tokens"], st["mask"],
                                     st["words"], st["positions"], st["trees"])
        return st["out"]
    # The pages of every request, in order: [B, G, keys, D] in 32 bits.
    pages = st["table"].long().clamp(min=0)
    keys = pages.shape[1] * page
    k = pool["k"].view(-1, G, page // TILE, D // 8, TILE, 8)[pages]
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(B, G, keys, D).float()
    v = pool["v"].view(-1, G, page // TILE, 2, D, 2, 4)[pages]
    v = v.permute(0, 2, 1, 3, 6, 4, 7, 5).reshape(B, G, keys, D).float()
    if case["type"] == "int8":
        k, v = (x * s.view(-1, G, page)[pages].transpose(1, 2).reshape(B, G, keys, 1)
                for x, s in ((k, pool["k_scale"]), (v, pool["v_scale"])))
    # The queries, padded to the most rows: [B, G, rows of a KV head's query heads, D].
    cu, kv_lens, n = st["cu"].long(), st["kv_lens"].long(), st["most"]
    i = torch.arange(n, device="cuda")
    new = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp(max=st["tokens"] - 1)
    q = st["q"][at].view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    scores = ((q @ k.transpose(-1, -2).contiguous()) * scale).view(B, G, H // G, n, keys)
    # What a row sees: cached keys, and new ones by its mask or up to itself.
    base = (kv_lens - new)[:, None, None]
    j = torch.arange(keys, device="cuda")
    node = j - base                                             # [B, 1, keys]
    bits = st["words"] * WORD
    word = st["mask"][at].gather(2, (node // WORD).clamp(0, st["words"] - 1).expand(B, n, keys))
    by_mask = (word >> (node % WORD) & 1).bool() & (node < bits)
    pos = st["positions"][at].long()[..., None]
    tree = (st["trees"] != 0)[:, None, None]
    cached = node < 0
    if case["window"] > 0:
        cached = cached & (j > pos - case["window"])
        causal = (node <= i[:, None]) & (j > pos - case["window"])
    else:
        causal = node <= i[:, None]
    seen = torch.where(tree, cached | (by_mask & (node >= 0)), causal)
    seen &= j < kv_lens[:, None, None]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = v.masked_fill_((j >= kv_lens[:, None])[:, None, :, None], 0.0)
    out = (p.view(B, G, -1, keys) @ v).view(B, G, H // G, n, D)
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, H * D)
    st["out"].copy_(out[i[None] < new[:, None]])
    return st["out"]


def _exact_tree(case, seed):
    """One request and KV head after the other, in 64 bits, what a row sees from the sets of
    its ancestors."""
    st = _prepare_tree(case, seed)
    G, D, page, pool = case["kv_heads"], case["dim"], case["page"], st["pool"]
    R = case["heads"] // G
    q = st["q"].double().view(-1, G, R, D)
    out = torch.zeros_like(q)
    first = 0
    for b, (new, total, tree) in enumerate(st["requests"]):
        n, base = _pages(total, page), total - new
        mine = st["table"][b, :n].long()
        hidden = torch.zeros(new, total, dtype=torch.bool)
        for i in range(new):
            mask = st["masks"][first + i] if tree else (2 << i) - 1
            hidden[i, base:] = torch.tensor([not mask >> c & 1 for c in range(new)])
            if case["window"]:
                past = max(0, st["depths"][first + i] - case["window"] + 1)
                hidden[i, :min(past, base) if tree else past] = True
        hidden = hidden.cuda()
        for g in range(G):
            def cells(name, dims, order):
                x = pool[name].view(-1, G, *dims)[mine, g].double()
                return x.permute(order).reshape(n * page, -1)[:total]
            k = cells("k", (page // TILE, D // 8, TILE, 8), (0, 1, 3, 2, 4))
            v = cells("v", (page // TILE, 2, D, 2, 4), (0, 1, 4, 2, 5, 3))
            if case["type"] == "int8":
                k = k * cells("k_scale", (page,), (0, 1))
                v = v * cells("v_scale", (page,), (0, 1))
            for r in range(R):
                s = q[first:first + new, g, r] @ k.T / math.sqrt(D)
                out[first:first + new, g, r] = torch.softmax(
                    s.masked_fill(hidden, -math.inf), -1) @ v
        first += new
    return out.view(first, -1)


# ---- log probabilities ----------------------------------------------------------------------

def _prepare_logprobs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    R, n, m, top = case["rows"], case["vocab"], case["given"], case["top"]
    # A row's largest logits stand out more or less: entropies from near 0 to near log n.
    spread = 0.5 + 5.0 * torch.rand(R, 1, generator=gen, device="cuda")
    logits = torch.randn(R, n, generator=gen, device="cuda").mul_(spread)
    if case["padded"]:       # ids that a vocabulary is rounded up by, never allowed
        logits[:, n - case["padded"]:] = float("-inf")
    tokens = torch.randint(0, n - case["padded"], (R, m), generator=gen, device="cuda",
                           dtype=torch.int32)
    if m:                    # one of the likely ones, as drafts are
        tokens[:, 0] = logits.argmax(1)
    st = {"case": case, "logits": logits, "tokens": tokens}
    for name, cols, dtype in (("logprobs", m, torch.float32), ("top_ids", top, torch.int32),
                              ("top_logprobs", top, torch.float32)):
        st[name] = torch.empty(R, cols, dtype=dtype, device="cuda")
    st["entropy"] = torch.empty(R, device="cuda")
    return st


def _inverse(case):
    """1 / temperature, in 32 bits as the logits are."""
    return (1.0 / torch.tensor(case["temperature"], dtype=torch.float32)).item()


def _run_logprobs(st):
    case, x = st["case"], st["logits"]
    out = [st[name] for name in ("logprobs", "entropy", "top_ids", "top_logprobs")
           if st[name].numel()]
    R, n, m, top = case["rows"], case["vocab"], case["given"], case["top"]
    if own:
        _capi().token_logprobs(x, R, n, st["tokens"] if m else None, m, top,
                               st["logprobs"] if m else None, st["entropy"],
                               st["top_ids"] if top else None,
                               st["top_logprobs"] if top else None,
                               temperature=case["temperature"])
        return out
    if case["temperature"] != 1.0:
        x = x * _inverse(case)
    # Distances from the maximum, whose sums are long ones.
    low = x - x.amax(1, keepdim=True)
    p = low.exp()
    total = p.sum(1, dtype=torch.float64)
    mean = (p * torch.where(p > 0, low, 0.0)).sum(1, dtype=torch.float64) / total
    log_total = total.log()
    st["entropy"].copy_(log_total - mean)
    if m:
        st["logprobs"].copy_(low.gather(1, st["tokens"].long()).double() - log_total[:, None])
    if top:
        # Distinct whole numbers in the order of (logit, then the lower id).
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, ~bits & 0xffffffff, bits | 0x80000000) - (1 << 31)
        key = (order << 32) | (0x7fffffff - torch.arange(n, device="cuda"))
        ids = 0x7fffffff - (key.topk(top, 1).values & 0xffffffff)
        st["top_ids"].copy_(ids)
        st["top_logprobs"].copy_(low.gather(1, ids).double() - log_total[:, None])
    return out


def _exact_logprobs(case, seed):
    """log softmax in 64 bits, some rows at a time."""
    st = _prepare_logprobs(case, seed)
    out, top = [[], [], [], []], case["top"]
    for at in range(0, case["rows"], 64):
        x = st["logits"][at:at + 64].double()
        if case["temperature"] != 1.0:
            x = x * _inverse(case)
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        p = logp.exp()
        out[0].append(logp.gather(1, st["tokens"][at:at + 64].long()))
        out[1].append(-(p * torch.where(p > 0, logp, 0.0)).sum(1))
        out[3].append(logp.sort(1, descending=True).values[:, :top])
    given, entropy, ids, top_logprobs = (torch.cat(x) if x else None for x in out)
    return (([given] if case["given"] else []) + [entropy] +
            ([ids, top_logprobs] if top else []))


# ---- the accepted path ----------------------------------------------------------------------

def _prepare_keep(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rng, G, D, page, L = (random.Random(seed), case["kv_heads"], case["dim"], case["page"],
                          case["layers"])
    requests = _requests({**case, "chunk": case["nodes"]})
    # The pages with new rows lie in the cache, those before them are not touched.
    first = [(total - new) // page for new, total, _ in requests]
    need = [_pages(total, page) for _, total, _ in requests]
    pages = sum(n - f for f, n in zip(first, need)) + 4
    order = list(range(pages))
    rng.shuffle(order)
    max_pages = max(need) + 1
    table = torch.full((case["seqs"], max_pages), -1, dtype=torch.int32)
    at = 4
    for b, (f, n) in enumerate(zip(first, need)):
        table[b, f:n] = torch.tensor(order[at:at + n - f])
        at += n - f
    # Accepted nodes: each stays where it is or comes from behind the path, so that a call
    # again on the same cache moves the same values.
    keep, counts = [], []
    width = case["nodes"]
    for new, _, tree in requests:
        if not tree:
            counts.append(-1)
            keep.append([0] * width)
            continue
        count = min(new, 1 + min(rng.randrange(8), rng.randrange(8)))
        stay = rng.randint(1, count)
        moved = min(count - stay, max(0, new - count))
        path = list(range(stay)) + sorted(rng.sample(range(count, new), moved)) \
            if moved else list(range(stay))
        counts.append(len(path))
        keep.append(path + [-1] * (width - len(path)))
    size = (L, pages * G * page * D)
    k_scale = v_scale = None
    if case["type"] == "int8":
        k, v = (torch.randint(-127, 128, size, generator=gen, device="cuda", dtype=torch.int8)
                for _ in range(2))
        k_scale, v_scale = (torch.rand(L, pages * G * page, generator=gen, device="cuda")
                            for _ in range(2))
    else:
        k, v = (torch.randn(size, generator=gen, device="cuda", dtype=TYPES[case["type"]])
                for _ in range(2))
    st = {"case": case, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale,
          "pages": pages, "max_pages": max_pages, "table": table.cuda(), "requests": requests,
          "paths": keep, "keep": _int32(keep), "counts": _int32(counts), "width": width,
          "kv_lens": _int32([total for _, total, _ in requests]),
          "cu": _int32(_prefix([new for new, _, _ in requests])),
          "granted": _int32([1] * case["seqs"]),
          "kept_lens": torch.zeros(case["seqs"], dtype=torch.int32, device="cuda"),
          "stack": _int32(order[:4] + [-1] * (pages - 4)), "count": _int32([4]),
          "count_out": _int32([0])}
    if own:
        capi = _capi()
        st["caches"] = capi.PagedCaches([
            capi.PagedCache(case["type"], pages, page, G, D, k[i], v[i],
                            None if k_scale is None else k_scale[i],
                            None if v_scale is None else v_scale[i]) for i in range(L)])
    return st


def _run_keep(st):
    case = st["case"]
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    out = [st["k"], st["v"], st["kept_lens"], st["stack"], st["count_out"]]
    if case["type"] == "int8":
        out += [st["k_scale"], st["v_scale"]]
    if own:
        _capi().paged_kv_keep(st["caches"], st["table"], st["max_pages"], st["kv_lens"],
                              st["cu"], st["granted"], case["seqs"], st["keep"], st["width"],
                              st["counts"], st["kept_lens"], st["stack"], st["count"],
                              st["count_out"])
        return out
    kv_lens, table = st["kv_lens"].long(), st["table"].long()
    new = (st["cu"][1:] - st["cu"][:-1]).long()
    base = (kv_lens - new)[:, None]
    some = st["counts"] >= 0
    kept = torch.where(some, kv_lens - new + st["counts"], kv_lens)
    i = torch.arange(st["width"], device="cuda")
    on_path = (i < st["counts"][:, None]) & some[:, None]
    b, i = on_path.nonzero(as_tuple=True)
    frm, to = base[b, 0] + st["keep"].long()[b, i], base[b, 0] + i
    b, frm, to = b[frm != to], frm[frm != to], to[frm != to]
    k_from, v_from, s_from = _places(table[b, frm // page] * page + frm % page, case)
    k_to, v_to, s_to = _places(table[b, to // page] * page + to % page, case)
    for name, x_from, x_to in (("k", k_from, k_to), ("v", v_from, v_to),
                               ("k_scale", s_from, s_to), ("v_scale", s_from, s_to)):
        if st[name] is not None:
            st[name][:, x_to] = st[name][:, x_from]
    # Pages past the kept length go on top of the stack, in the order of the requests.
    col = torch.arange(st["max_pages"], device="cuda")
    back = ((col >= ((kept + page - 1) // page)[:, None]) &
            (col < ((kv_lens + page - 1) // page)[:, None])).flatten()
    pages, count = st["pages"], st["count"].long()
    place = torch.where(back, count + back.long().cumsum(0) - 1, pages)
    stack = torch.cat([st["stack"], st["stack"][:1]])
    stack.scatter_(0, place, torch.where(back, st["table"].flatten(), -1))
    st["stack"].copy_(stack[:pages])
    st["count_out"].copy_(count + back.sum())
    st["kept_lens"].copy_(kept)
    return out


def _exact_keep(case, seed):
    """The values moved one by one; whole numbers are found on the host."""
    st = _prepare_keep(case, seed)
    G, D, page, L = case["kv_heads"], case["dim"], case["page"], case["layers"]
    table, lens, back = st["table"].tolist(), [], []
    moves = []
    for b, (new, total, tree) in enumerate(st["requests"]):
        path = [i for i in st["paths"][b] if i >= 0] if tree else range(new)
        at = [table[b][p // page] * page + p % page if table[b][p // page] >= 0 else -1
              for p in range(total - new, total)]
        moves += [(at[i], at[j]) for j, i in enumerate(path)]
        lens.append(total - new + len(path))
        back += table[b][_pages(lens[-1], page):_pages(total, page)]
    frm, to = (torch.tensor(x, device="cuda") for x in zip(*moves))
    floating = case["type"] != "int8"
    out = [None, None]
    if floating:
        x = st["k"].double().view(L, -1, G, page // TILE, D // 8, TILE, 8)
        x = x.permute(0, 1, 3, 5, 2, 4, 6).reshape(L, -1, G, D // 8, 8)   # [slot, G, ...]
        x[:, to] = x[:, frm]
        x = x.view(L, -1, page // TILE, TILE, G, D // 8, 8).permute(0, 1, 4, 2, 5, 3, 6)
        out[0] = x.reshape(L, -1)
        x = st["v"].double().view(L, -1, G, page // TILE, 2, D, 2, 4)
        x = x.permute(0, 1, 3, 6, 4, 7, 2, 5).reshape(L, -1, G, D)
        x[:, to] = x[:, frm]
        x = x.view(L, -1, page // TILE, 2, 2, 4, G, D).permute(0, 1, 6, 2, 4, 7, 3, 5)
        out[1] = x.reshape(L, -1)
    stack = st["stack"].tolist()
    stack[4:4 + len(back)] = back
    out += [_int32(lens), _int32(stack), _int32([4 + len(back)])]
    if not floating:
        for name in ("k_scale", "v_scale"):
            x = st[name].double().view(L, -1, G, page).transpose(2, 3).reshape(L, -1, G)
            x[:, to] = x[:, frm]
            out.append(x.view(L, -1, page, G).transpose(2, 3).reshape(L, -1))
    return out


# ---- what the tools call --------------------------------------------------------------------

def prepare(case, seed):
    return {"write": _prepare_write, "tree": _prepare_tree, "logprobs": _prepare_logprobs,
            "keep": _prepare_keep}[case["kind"]](case, seed)


def run(state):
    return {"write": _run_write, "tree": _run_tree, "logprobs": _run_logprobs,
            "keep": _run_keep}[state["case"]["kind"]](state)


def exact(case, seed):
    return {"write": _exact_write, "tree": _exact_tree, "logprobs": _exact_logprobs,
            "keep": _exact_keep}[case["kind"]](case, seed)


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["kind"] == "logprobs":
        R, n, m, top = case["rows"], case["vocab"], case["given"], case["top"]
        return {"bytes": R * (4 * n + 8 * m + 8 * top + 4), "flops": 6 * R * n}
    G, D = case["kv_heads"], case["dim"]
    cell = {"f16": 2 * D, "bf16": 2 * D, "int8": D + 4}[case["type"]]
    if case["kind"] == "keep":
        rows = sum(n for n, _, _ in _requests({**case, "chunk": case["nodes"]}))
        moved = 2 * case["seqs"]      # about as many rows change their place
        return {"bytes": case["layers"] * moved * G * 2 * 2 * cell + 4 * rows
                + 24 * case["seqs"], "flops": 0}
    H = case["heads"]
    if case["kind"] == "write":
        row = 4 * D * (2 * H + 2 * G) + 2 * G * cell + 8
        flops = 4 * D * (H + G)
        if case["rope"] != "none":
            row += 4 * D
            flops += 3 * D * (H + G)
        return {"bytes": case["tokens"] * row + 8 * D, "flops": case["tokens"] * flops}
    keys = pairs = tokens = 0
    for new, total, tree in _requests(case):
        reach = case["window"] or total
        keys += min(total, reach + new - 1)
        if tree:     # a node's ancestors are few beside the cached keys
            pairs += new * (min(total - new, reach) + 1)
        else:
            pairs += sum(min(p + 1, reach) for p in range(total - new, total))
        tokens += new
    return {"bytes": keys * G * 2 * cell + tokens * (8 * H * D + 12) + 4 * keys // case["page"],
            "flops": 4 * D * H * pairs}
