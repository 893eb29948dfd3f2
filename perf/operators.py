"""Workloads of the paged KV cache: page planning, the rotary cache write, and attention.

A serving step of a decoder layer makes three calls besides its Linears: the plan (pages
for each request's new tokens, the slot of every token), the write (q and k rotated, k and
v put into their slots of the cache) and the attention of the new tokens over the cache.
``run`` makes one of them, through ``llmengine_amd.capi`` where ``own`` is true and in plain
torch operations where it is not.  Head counts and sizes are those of the benchmark's
models (Llama-7B: 32 heads of 128; Qwen2.5-0.5B: 14 heads of 64 over 2 KV heads) or a
generic grouped layout (32 heads of 128 over 8 KV heads).

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
TILE = 16                 # tokens of a cache tile
MAX_PAIRS = 32 * 128 * 2048 * (10240 - 1024)  # heads * dim * (query, key) pairs, largest listed
MAX_SCORES = 32 * 2048 * 10240                # padded scores of the plain form, largest listed
MAX_CACHE = 8 * 32768 * 8 * 128               # padded cache elements, largest listed


def listed():
    return [
        # A decode batch of 64 requests: most need no page, some start one.
        {"name": "plan_decode_64", "kind": "plan", "seqs": 64, "chunk": 1, "chunked": 0,
         "kv": 4096, "page": 16, "release": 2, "short": False, "mix": 1},
        # Admission of many prompts at once, finished requests among them, pages running out.
        {"name": "plan_prompts_512", "kind": "plan", "seqs": 512, "chunk": 512, "chunked": 64,
         "kv": 8192, "page": 32, "release": 40, "short": True, "mix": 2},
        # The write of a decode step: 32 tokens of a 7B model, q/k/v in buffers of their own.
        {"name": "write_decode_32", "kind": "write", "type": "f16", "heads": 32,
         "kv_heads": 32, "dim": 128, "page": 16, "tokens": 32, "rope": "pairs",
         "fused": False, "mix": 3},
        # A prompt of odd length of a 0.5B model, q/k/v in one buffer of the fused Linear.
        {"name": "write_prompt_1531", "kind": "write", "type": "bf16", "heads": 14,
         "kv_heads": 2, "dim": 64, "page": 32, "tokens": 1531, "rope": "halves",
         "fused": True, "mix": 4},
        # A long prompt into an 8-bit cache.
        {"name": "write_prompt_int8_8192", "kind": "write", "type": "int8", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "tokens": 8192, "rope": "halves",
         "fused": False, "mix": 5},
        # Smallest: one request of a 0.5B model, one token over a short context.
        {"name": "attn_decode_1x129", "kind": "attention", "type": "f16", "heads": 14,
         "kv_heads": 2, "dim": 64, "page": 16, "seqs": 1, "chunk": 1, "chunked": 0,
         "kv": 129, "window": 0, "mix": 6},
        # A decode batch of a 7B model, no grouped heads, lengths up to 4096.
        {"name": "attn_decode_32x4096", "kind": "attention", "type": "f16", "heads": 32,
         "kv_heads": 32, "dim": 128, "page": 16, "seqs": 32, "chunk": 1, "chunked": 0,
         "kv": 4096, "window": 0, "mix": 7},
        # A few long contexts on an 8-bit cache, grouped heads: the KV axis has to be split.
        {"name": "attn_decode_int8_8x32768", "kind": "attention", "type": "int8", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "seqs": 8, "chunk": 1, "chunked": 0,
         "kv": 32768, "window": 0, "mix": 8},
        # A decode batch with the chunk of a prompt in it.
        {"name": "attn_mixed_bf16", "kind": "attention", "type": "bf16", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 32, "seqs": 16, "chunk": 300, "chunked": 1,
         "kv": 4096, "window": 0, "mix": 9},
        # Prompts of odd length through a sliding window, 8-bit cache.
        {"name": "attn_window_int8_3x777", "kind": "attention", "type": "int8", "heads": 14,
         "kv_heads": 2, "dim": 64, "page": 16, "seqs": 3, "chunk": 777, "chunked": 3,
         "kv": 2500, "window": 512, "mix": 10},
        # The last chunk of a long prompt: the largest case.
        {"name": "attn_chunk_2048x10240", "kind": "attention", "type": "f16", "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "seqs": 1, "chunk": 2048, "chunked": 1,
         "kv": 10240, "window": 0, "mix": 11},
        # A whole prompt with nothing cached before it, no grouped heads.
        {"name": "attn_prompt_4x512", "kind": "attention", "type": "f16", "heads": 32,
         "kv_heads": 32, "dim": 128, "page": 16, "seqs": 4, "chunk": 512, "chunked": 4,
         "kv": 512, "window": 0, "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    """(heads, KV heads, head size)"""
    return rng.choice([(14, 2, 64), (32, 32, 128), (32, 8, 128), (16, 4, 96), (8, 1, 256),
                       (12, 12, 64), (28, 4, 128), (20, 5, 128)])


def draw(rng):
    kind = rng.choice(["plan", "write", "attention", "attention", "attention"])
    mix = rng.randint(0, 1 << 30)
    page = rng.choice([16, 32, 64, 128])
    if kind == "plan":
        seqs = _log_int(rng, 1, 1000)
        chunk = _log_int(rng, 1, 512)
        return {"kind": kind, "seqs": seqs, "chunk": chunk,
                "chunked": rng.randint(0, min(seqs, 64)), "kv": _log_int(rng, 600, 16000),
                "page": page, "release": rng.randint(0, seqs // 8),
                "short": rng.random() < 0.3, "mix": mix}
    heads, kv_heads, dim = _heads(rng)
    kv_type = rng.choice(["f16", "f16", "bf16", "int8"])
    if kind == "write":
        return {"kind": kind, "type": kv_type, "heads": heads, "kv_heads": kv_heads,
                "dim": dim, "page": page, "tokens": _log_int(rng, 1, 8192),
                "rope": rng.choice(["halves", "pairs", "none"]),
                "fused": rng.random() < 0.5, "mix": mix}
    kv = _log_int(rng, 1, 32768)
    seqs = _log_int(rng, 1, 64)
    chunk = 1 if rng.random() < 0.4 else min(kv, _log_int(rng, 2, 2048))
    seqs = max(1, min(seqs, MAX_CACHE // (kv * kv_heads * dim)))
    chunk = max(1, min(chunk, MAX_SCORES // (kv * seqs * heads)))
    chunked = 0 if chunk == 1 else rng.choice([1, seqs, rng.randint(1, seqs)])
    chunk = max(1, min(chunk, MAX_PAIRS // (max(1, chunked) * heads * dim * kv)))
    return {"kind": kind, "type": kv_type, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": page, "seqs": seqs, "chunk": chunk, "chunked": chunked if chunk > 1 else 0,
            "kv": kv, "window": rng.choice([0, 0, 0, 100, 1024]), "mix": mix}


def _lengths(case):
    """(new tokens, tokens in all) of each sequence: `chunked` of them with a chunk, the others
    decoding one token; the first is as long as any, the others spread over a factor of 16.
    Of several chunks the later ones are shorter, as prompts are."""
    rng = random.Random(case["mix"])
    out = []
    for b in range(case["seqs"]):
        total = case["kv"] if b == 0 else max(1, int(case["kv"] * 16 ** -rng.random()))
        new = 1
        if b < case["chunked"]:
            new = case["chunk"] if b == 0 else max(1, int(case["chunk"] * rng.uniform(0.4, 1)))
            total = max(total, new)
        out.append((new, total))
    return out


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


# ---- the plan -------------------------------------------------------------------------------

def _prepare_plan(case, seed):
    gen = random.Random(seed)
    lens = [(new, max(1, total - new)) for new, total in _lengths(case)]
    news, cached = [n for n, _ in lens], [c for _, c in lens]
    for b in random.Random(case["mix"]).sample(range(case["seqs"]), case["release"]):
        news[b] = -1
    page = case["page"]
    have = [_pages(c, page) for c in cached]
    add = [0 if n < 0 else _pages(c + n, page) - h for n, c, h in zip(news, cached, have)]
    back = sum(h for n, h in zip(news, have) if n < 0)
    # Enough free pages for all, or for about two thirds of what is asked.
    free = max(0, sum(add) * 2 // 3 - back) if case["short"] else sum(add) + 64
    pages = sum(have) + free
    order = list(range(pages))
    gen.shuffle(order)
    max_pages = max(_pages(c + max(n, 0), page) for n, c in zip(news, cached)) + 8
    rows, at = [], free
    for h in have:
        rows.append(order[at:at + h] + [-1] * (max_pages - h))
        at += h
    stack = order[:free] + [-1] * (pages - free)
    tokens = sum(n for n in news if n > 0)
    st = {"case": case, "tokens": tokens, "pages": pages, "max_pages": max_pages,
          "cached": _int32(cached), "new": _int32(news), "table": _int32(rows),
          "stack": _int32(stack), "count": _int32([free])}
    for name, n in (("count_out", 1), ("kv_lens", case["seqs"]), ("cu", case["seqs"] + 1),
                    ("positions", tokens), ("slots", tokens), ("granted", case["seqs"])):
        st[name] = torch.empty(n, dtype=torch.int32, device="cuda")
    return st


def _run_plan(st):
    case = st["case"]
    if own:
        _capi().paged_plan(st["cached"], st["new"], case["seqs"], st["table"], st["max_pages"],
                           case["page"], st["pages"], st["stack"], st["count"],
                           st["count_out"], st["tokens"], st["kv_lens"], st["cu"],
                           st["positions"], st["slots"], st["granted"])
        return {n: st[n] for n in ("table", "stack", "count_out", "kv_lens", "cu", "positions",
                                   "slots", "granted")}
    page, pages, table = case["page"], st["pages"], st["table"].long()
    cached, new, count = st["cached"].long(), st["new"].long(), st["count"].long()
    released, want = new < 0, new.clamp(min=0)
    have, need = (cached + page - 1) // page, (cached + want + page - 1) // page
    col = torch.arange(st["max_pages"], device="cuda")
    # Released pages go on top of the stack, in the order of the requests.
    back = (col < have[:, None]) & released[:, None]
    rank = back.flatten().long().cumsum(0) - 1
    place = torch.where(back.flatten(), count + rank, pages)
    stack = torch.cat([st["stack"].long(), st["stack"].long()[:1]])
    stack = stack.scatter(0, place, torch.where(back.flatten(), table.flatten(), -1))[:pages]
    count = count + back.sum()
    # Pages from the top of the stack, in the order of the requests, while they last.
    add = torch.where(released, 0, need - have)
    upto = add.cumsum(0)
    granted = released | (add == 0) | (upto <= count)
    took = torch.where(granted, upto, 0).max().clamp(min=0)
    fresh = (col >= have[:, None]) & (col < need[:, None]) & (granted & ~released)[:, None]
    at = count - 1 - ((upto - add - have)[:, None] + col)
    table = torch.where(fresh, stack[at.clamp(0, pages - 1)], table)
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), want.cumsum(0)])
    t = torch.arange(st["tokens"], device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = cached[b] + t - cu[b]
    ok = granted[b]
    slots = table[b, (pos // page).clamp(max=st["max_pages"] - 1)] * page + pos % page
    kv_lens = torch.where(granted & ~released, cached + want, 0)
    out = {"table": table, "stack": stack, "count_out": (count - took), "kv_lens": kv_lens,
           "cu": cu, "positions": torch.where(ok, pos, 0), "slots": torch.where(ok, slots, -1),
           "granted": granted}
    return {n: x.int() for n, x in out.items()}


def _exact_plan(case, seed):
    """The plan request by request, on the host."""
    st = _prepare_plan(case, seed)
    page = case["page"]
    cached, new = st["cached"].tolist(), st["new"].tolist()
    table, whole = st["table"].tolist(), st["stack"].tolist()
    stack, tail = whole[:st["count"].item()], whole
    for b, n in enumerate(new):
        if n < 0:
            stack += table[b][:_pages(cached[b], page)]
    tail[:len(stack)] = stack
    asked, total = 0, len(stack)
    lens, granted, positions, slots = [], [], [], []
    for b, n in enumerate(new):
        if n < 0:
            lens.append(0)
            granted.append(1)
            continue
        first, last = _pages(cached[b], page), _pages(cached[b] + n, page)
        asked += last - first
        ok = last == first or asked <= total
        if ok:
            for j in range(first, last):
                table[b][j] = stack.pop()
        granted.append(int(ok))
        lens.append(cached[b] + n if ok else 0)
        for i in range(cached[b], cached[b] + n):
            positions.append(i if ok else 0)
            slots.append(table[b][i // page] * page + i % page if ok else -1)
    cu = _prefix([max(n, 0) for n in new])
    out = {"table": table, "stack": tail, "count_out": [len(stack)], "kv_lens": lens, "cu": cu,
           "positions": positions, "slots": slots, "granted": granted}
    return {n: _int32(x) for n, x in out.items()}


# ---- the write ------------------------------------------------------------------------------

def _prepare_write(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, G, D, page, T = (case["heads"], case["kv_heads"], case["dim"], case["page"],
                        case["tokens"])
    if case["fused"]:
        qkv = torch.randn(T, (H + 2 * G) * D, generator=gen, device="cuda")
        q, k, v = qkv.split([H * D, G * D, G * D], dim=1)
    else:
        q, k, v = (torch.randn(T, n * D, generator=gen, device="cuda") for n in (H, G, G))
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
    st = {"case": case, "q": q, "k": k, "v": v, "positions": _int32(positions),
          "slots": _int32(slots), "q_out": torch.empty(T, H * D, device="cuda"),
          "rope": None, "limit": 0}
    if case["rope"] != "none":
        angle = (torch.arange(limit, device="cuda", dtype=torch.float64)[:, None] *
                 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D))
        st["rope"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
        st["limit"] = limit
    cells = pages * G * page
    k, v = (torch.zeros(cells * D, dtype=TYPES[case["type"]], device="cuda") for _ in range(2))
    scales = [None, None]
    if case["type"] == "int8":
        scales = [torch.zeros(cells, device="cuda") for _ in range(2)]
    st["pool"] = _pool(case, pages, k, v, *scales)
    return st


def _rotated(x, st, mode):
    """Rotary embedding of [T, heads, D], in 64 bits."""
    x = x.double()
    if mode == "none":
        return x
    cos, sin = st["rope"][st["positions"].long()].double()[:, None].unbind(-1)
    D = x.shape[-1]
    a, b = (x[..., :D // 2], x[..., D // 2:]) if mode == "halves" else (x[..., 0::2],
                                                                       x[..., 1::2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    return (torch.cat([ra, rb], -1) if mode == "halves"
            else torch.stack([ra, rb], -1).flatten(-2))


def _places(st, case):
    """Flat index of every token's K and V elements in the cache, and of its scale."""
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    slot = st["slots"].long()
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
    if own:
        _capi().paged_kv_write(pool["cache"], st["q"], st["q_out"], H, st["k"], st["v"],
                               st["rope"], st["limit"], D, case["rope"], st["positions"],
                               st["slots"], T)
        out = [st["q_out"], pool["k"], pool["v"]]
        return out + ([pool["k_scale"], pool["v_scale"]] if case["type"] == "int8" else [])
    st["q_out"].copy_(_rotated(st["q"].reshape(T, H, D), st, case["rope"]).flatten(1))
    k = _rotated(st["k"].reshape(T, G, D), st, case["rope"]).float()
    v = st["v"].reshape(T, G, D)
    at_k, at_v, at_s = _places(st, case)
    out = [st["q_out"], pool["k"], pool["v"]]
    if case["type"] == "int8":
        k_scale, v_scale = (x.abs().amax(-1) * (1.0 / 127.0) for x in (k, v))
        pool["k_scale"][at_s], pool["v_scale"][at_s] = k_scale, v_scale
        k, v = ((x / s[..., None]).round() for x, s in ((k, k_scale), (v, v_scale)))
        out += [pool["k_scale"], pool["v_scale"]]
    pool["k"][at_k] = k.to(pool["k"].dtype)
    pool["v"][at_v] = v.to(pool["v"].dtype)
    return out


def _exact_write(case, seed):
    """Token by token from the definition of the rotation and of the cells; 8-bit cells are
    whole numbers, which have no value in 64 bits."""
    st = _prepare_write(case, seed)
    H, G, D, T = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    turn = torch.ones(T, 1, max(1, D // 2), dtype=torch.complex128, device="cuda")
    if case["rope"] != "none":
        turn = torch.view_as_complex(st["rope"].double())[st["positions"].long()][:, None]
    halves = case["rope"] == "halves"

    def turned(x, n):
        x = x.double().reshape(T, n, D)
        pairs = x.reshape(T, n, 2, D // 2).transpose(2, 3) if halves else x.reshape(
            T, n, D // 2, 2)
        y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return (y.transpose(2, 3) if halves else y).reshape(T, n, D)

    k, v = turned(st["k"], G), st["v"].double().reshape(T, G, D)
    q = turned(st["q"], H).flatten(1)
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


# ---- the attention --------------------------------------------------------------------------

def _prepare_attention(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    H, G, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    lens = _lengths(case)
    need = [_pages(total, page) for _, total in lens]
    pages = sum(need) + 8
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    max_pages = max(need) + 2
    table = torch.full((case["seqs"], max_pages), -1, dtype=torch.int32, device="cuda")
    for b, (at, n) in enumerate(zip(_prefix(need), need)):
        table[b, :n] = order[at:at + n]
    T = sum(new for new, _ in lens)
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
            "max_pages": max_pages, "lens": lens, "most": max(n for n, _ in lens),
            "kv_lens": _int32([total for _, total in lens]),
            "cu": _int32(_prefix([new for new, _ in lens])),
            "pool": _pool(case, pages, k, v, k_scale, v_scale)}


def _run_attention(st):
    case, pool = st["case"], st["pool"]
    H, G, D, page, B = (case["heads"], case["kv_heads"], case["dim"], case["page"],
                        case["seqs"])
    scale = D ** -0.5
    if own:
        _capi().paged_attention(pool["cache"], st["q"], st["out"], H, scale, case["window"],
                                st["table"], st["max_pages"], st["kv_lens"], st["cu"], B,
                                st["tokens"])
        return st["out"]
    # The pages of every sequence, in order: [B, G, keys, D] in 32 bits.
    pages = st["table"].long().clamp(min=0)
    keys = pages.shape[1] * page
    k = pool["k"].view(-1, G, page // TILE, D // 8, TILE, 8)[pages]
    k = k.permute(0, 2, 1, 3, 5, 4, 6).reshape(B, G, keys, D).float()
    v = pool["v"].view(-1, G, page // TILE, 2, D, 2, 4)[pages]
    v = v.permute(0, 2, 1, 3, 6, 4, 7, 5).reshape(B, G, keys, D).float()
    if case["type"] == "int8":
        k, v = (x * s.view(-1, G, page)[pages].transpose(1, 2).reshape(B, G, keys, 1)
                for x, s in ((k, pool["k_scale"]), (v, pool["v_scale"])))
    # The queries, padded to the longest chunk: [B, G, rows of a KV head's query heads, D].
    cu, kv_lens, n = st["cu"].long(), st["kv_lens"].long(), st["most"]
    i = torch.arange(n, device="cuda")
    new = cu[1:] - cu[:-1]
    at = (cu[:-1, None] + i).clamp(max=st["tokens"] - 1)
    q = st["q"][at].view(B, n, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    scores = ((q @ k.transpose(-1, -2).contiguous()) * scale).view(B, G, H // G, n, keys)
    pos = (kv_lens - new)[:, None] + i
    j = torch.arange(keys, device="cuda")
    seen = (j <= pos[..., None]) & (j < kv_lens[:, None, None])
    if case["window"] > 0:
        seen &= j > pos[..., None] - case["window"]
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


def _exact_attention(case, seed):
    """One sequence and KV head after the other, in 64 bits."""
    st = _prepare_attention(case, seed)
    G, D, page, pool = case["kv_heads"], case["dim"], case["page"], st["pool"]
    R = case["heads"] // G
    q = st["q"].double().view(-1, G, R, D)
    out = torch.zeros_like(q)
    first = 0
    for b, (new, total) in enumerate(st["lens"]):
        n = _pages(total, page)
        mine = st["table"][b, :n].long()
        lo = max(0, total - new + 1 - case["window"]) if case["window"] else 0
        for g in range(G):
            def cells(name, dims, order):
                x = pool[name].view(-1, G, *dims)[mine, g].double()
                return x.permute(order).reshape(n * page, -1)[lo:total]
            k = cells("k", (page // TILE, D // 8, TILE, 8), (0, 1, 3, 2, 4))
            v = cells("v", (page // TILE, 2, D, 2, 4), (0, 1, 4, 2, 5, 3))
            if case["type"] == "int8":
                k = k * cells("k_scale", (page,), (0, 1))
                v = v * cells("v_scale", (page,), (0, 1))
            pos = total - new + torch.arange(new, device="cuda")[:, None]
            j = torch.arange(lo, total, device="cuda")
            hidden = j > pos
            if case["window"]:
                hidden |= j <= pos - case["window"]
            for r in range(R):
                s = q[first:first + new, g, r] @ k.T / math.sqrt(D)
                out[first:first + new, g, r] = torch.softmax(
                    s.masked_fill(hidden, -math.inf), -1) @ v
        first += new
    return out.view(first, -1)


# ---- what the tools call --------------------------------------------------------------------

def prepare(case, seed):
    return {"plan": _prepare_plan, "write": _prepare_write,
            "attention": _prepare_attention}[case["kind"]](case, seed)


def run(state):
    return {"plan": _run_plan, "write": _run_write,
            "attention": _run_attention}[state["case"]["kind"]](state)


def exact(case, seed):
    return {"plan": _exact_plan, "write": _exact_write,
            "attention": _exact_attention}[case["kind"]](case, seed)


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["kind"] == "plan":
        lens = _lengths(case)
        tokens, seqs = sum(n for n, _ in lens), case["seqs"]
        pages = sum(_pages(t, case["page"]) - _pages(t - n, case["page"]) for n, t in lens)
        return {"bytes": 4 * (5 * seqs + 2 * tokens + 2 * pages), "flops": 0}
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    cell = {"f16": 2 * D, "bf16": 2 * D, "int8": D + 4}[case["type"]]
    if case["kind"] == "write":
        row = 4 * D * (2 * H + 2 * G) + 2 * G * cell + 8
        flops = 0
        if case["rope"] != "none":
            row += 4 * D
            flops = 3 * D * (H + G)
        return {"bytes": case["tokens"] * row, "flops": case["tokens"] * flops}
    keys = pairs = tokens = 0
    for new, total in _lengths(case):
        reach = case["window"] or total
        keys += min(total, reach + new - 1)
        pairs += sum(min(p + 1, reach) for p in range(total - new, total))
        tokens += new
    return {"bytes": keys * G * 2 * cell + tokens * 8 * H * D + 4 * keys // case["page"],
            "flops": 4 * D * H * pairs}
