"""GPU numerics of trees of drafted tokens over the paged KV cache (include/mle_paged.h): the
attention against softmax in 64 bits over what each row's mask names, the move of an accepted
path against a host loop over the requests, the cache write with norms against the formula in
extended precision, and a run of them against decoding token by token.

Tolerance of the attention: that of the attention of runs of tokens (derived beside its tests):
2 max|v| (ds + 2^-20 + (keys / 8 + 64) 2^-24), ds = (D + 16) 2^-22 scale max_j sum_d |q_d k_jd|.
"""
import math

import numpy as np
import pytest

from helpers import empty_f32, note, own_stream, to_dev
from llmengine_amd import capi
from test_gpu_paged import (TYPES, cells_of, i32, make_cache, plan_case, plan_host, prefix, put,
                            rotate_host, stored_host)

pytestmark = pytest.mark.gpu


def tree_masks(rng, n, kind="tree"):
    """(seen [n, n], depth [n]) of n new rows: what each sees of them."""
    seen, depth = np.zeros((n, n), bool), np.zeros(n, np.int64)
    for i in range(n):
        if kind in ("tree", "flat"):
            p = -1 if i == 0 else 0 if kind == "flat" else int(rng.integers(max(0, i - 9), i))
            if p >= 0:
                seen[i] = seen[p]
                depth[i] = depth[p] + 1
            seen[i, i] = True
        elif kind == "chain":
            seen[i, :i + 1], depth[i] = True, i
        elif kind == "any":            # not a tree: any rows at all, later ones among them
            seen[i] = rng.random(n) < 0.4
            depth[i] = rng.integers(0, n)
    return seen, depth                 # "none": a row sees no new row, itself included


def words_of(seen, words):
    """Masks as [n, words] int64; bits past the words are left out."""
    n = seen.shape[0]
    out = np.zeros((n, words), np.uint64)
    for j in range(min(seen.shape[1], 64 * words)):
        out[:, j // 64] |= seen[:, j].astype(np.uint64) << np.uint64(j % 64)
    return out.view(np.int64)


def attention_host(q, k, v, seen, scale):
    """q [n, H, D], k/v [keys, G, D] in 64 bits, seen [n, keys]; (out, tolerance)."""
    n, H, D = q.shape
    R = H // k.shape[1]
    out, tol = np.zeros((n, H, D)), 0.0
    use = seen.any(0)
    if not use.any():
        return out, tol
    for h in range(H):
        kk, vv = k[:, h // R], v[:, h // R]
        s = np.where(seen, scale * (q[:, h].astype(np.float64) @ kk.T), -np.inf)
        top = s.max(-1, keepdims=True)
        e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        z = e.sum(-1, keepdims=True)
        out[:, h] = (e @ vv) / np.where(z > 0, z, 1)
        ds = (D + 16) * 2.0 ** -22 * abs(scale) * (np.abs(q[:, h]) @ np.abs(kk[use]).T).max()
        tol = max(tol, 2 * np.abs(vv[use]).max()
                  * (ds + 2.0 ** -20 + (use.sum() / 8 + 64) * 2.0 ** -24))
    return out, tol


class Trees:
    """Requests (new, total, kind) in a poisoned cache; kind "run" is causal, else as
    tree_masks has it."""

    def __init__(self, dev, kv_type, H, G, D, page, lens, window=0, seed=1, words=None,
                 bad_pages=(), all_trees=False, scale=None, shuffle_masks=True):
        rng = np.random.default_rng(seed)
        self.dev, self.H, self.G, self.D, self.page, self.lens = dev, H, G, D, page, lens
        self.window, self.scale = window, D ** -0.5 if scale is None else scale
        need = [-(-t // page) for _, t, _ in lens]
        pages = sum(need) + 3
        self.cache = make_cache(rng, dev, kv_type, pages, page, G, D)
        order = rng.permutation(pages)
        self.max_pages = max(need + [1]) + 2
        table = np.full((len(lens), self.max_pages), -1, np.int64)
        T = self.T = sum(n for n, _, _ in lens)
        self.words = words or max([1] + [-(-n // 64) for n, _, kind in lens if kind != "run"])
        q = (2.0 * rng.standard_normal((T, H, D))).astype(np.float32)
        # Bits past the rows of a request, and masks of runs, may be anything.
        masks = rng.integers(-2 ** 63, 2 ** 63, (T, self.words), dtype=np.int64)
        positions = np.zeros(T, np.int64)
        self.want, self.tol, at, row = np.zeros((T, H, D)), 0.0, 0, 0
        self.seen = []
        for b, ((n, total, kind), np_) in enumerate(zip(lens, need)):
            table[b, :np_] = order[at:at + np_]
            at += np_
            k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
            ok = np.ones(total, bool)
            if total:
                slots = table[b, np.arange(total) // page] * page + np.arange(total) % page
                k, v = put(self.cache, kv_type, page, slots, k, v)
            for bb, j in bad_pages:
                if bb == b and j < np_:
                    table[b, j] = -5 if j % 2 else pages + 3
                    ok[j * page:(j + 1) * page] = False
            base = total - n
            key = np.arange(total)
            if kind == "run":
                pos = base + np.arange(n)
                seen = key[None] <= pos[:, None]
                if window:
                    seen &= key[None] > pos[:, None] - window
            else:
                new, depth = tree_masks(rng, n, kind)
                pos = base + depth
                seen = np.zeros((n, total), bool)
                seen[:, :base] = key[None, :base] > pos[:, None] - window if window else True
                new[:, 64 * self.words:] = False
                seen[:, base:] = new
                mine = words_of(new, self.words)
                keep = words_of(np.ones((n, n), bool), self.words)
                masks[row:row + n] = (masks[row:row + n] & ~keep) | mine if n else 0
            positions[row:row + n] = pos
            seen &= ok[None]
            self.seen.append(seen)
            if n:
                o, tol = attention_host(q[row:row + n], k, v, seen, self.scale)
                self.want[row:row + n] = o
                self.tol = max(self.tol, tol)
            row += n
        self.q = to_dev(q.reshape(T, H * D), dev)
        self.table = i32(table, dev)
        self.kv_lens = i32([t for _, t, _ in lens], dev)
        self.cu = i32(prefix([n for n, _, _ in lens]), dev)
        self.mask = to_dev(masks, dev)
        self.positions = i32(positions, dev)
        self.trees = None if all_trees else i32([int(k != "run") for _, _, k in lens], dev)

    def run(self, out=None, q=None, stream=None, **kw):
        out = empty_f32((self.T, self.H * self.D), self.dev) if out is None else out
        a = dict(row_positions=self.positions if self.window else None, trees=self.trees)
        a.update(kw)
        capi.paged_tree_attention(self.cache, self.q if q is None else q, out, self.H,
                                  self.scale, self.window, self.table, self.max_pages,
                                  self.kv_lens, self.cu, len(self.lens), self.T, self.mask,
                                  self.words, a["row_positions"], a["trees"], stream=stream)
        return out

    def check(self, out):
        import torch
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(self.want.shape).astype(np.float64)
        assert np.isfinite(got).all()
        err = np.abs(got - self.want).max()
        assert err <= self.tol, (err, self.tol)


LAYOUTS = [(14, 2, 64), (4, 4, 128), (8, 2, 128), (8, 4, 96), (8, 1, 256), (64, 1, 64), (3, 3, 96)]


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D", LAYOUTS)
@pytest.mark.parametrize("lens,page,window", [
    ([(1, 1, "tree")], 16, 0),
    ([(8, 129, "tree"), (1, 1, "tree"), (3, 3, "flat"), (26, 700, "tree")], 16, 0),
    ([(70, 70, "tree"), (5, 90, "any"), (0, 50, "tree"), (64, 333, "tree"), (17, 190, "run")],
     32, 0),
    ([(130, 300, "tree"), (9, 17, "chain"), (6, 1000, "tree"), (90, 200, "run")], 48, 100)])
def test_tree_attention(dev, kv_type, H, G, D, lens, page, window):
    note(f"tree {kv_type} H={H} G={G} D={D} lens={lens} page={page} window={window}")
    b = Trees(dev, kv_type, H, G, D, page, lens, window=window, seed=H + D)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257])
def test_tree_sizes_and_offsets(dev, kv_type, n):
    """Trees that begin anywhere in a tile, a page, a unit of keys, and end there."""
    note(f"tree sizes {kv_type} n={n}")
    for base in (0, 1, 15, 31, 33, 63, 64, 79, 500):
        b = Trees(dev, kv_type, 4, 4, 64, 16, [(n, n + base, "tree"), (2, 40, "any")],
                  seed=n + base, all_trees=True)
        b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_long_context(dev, kv_type):
    """A few trees over long contexts: parts of a tile joined; several words of mask."""
    for lens in ([(8, 9000, "tree")], [(40, 6000, "tree"), (3, 5000, "tree")],
                 [(200, 5000, "tree")]):
        note(f"tree long {kv_type} {lens}")
        b = Trees(dev, kv_type, 8, 2, 128, 64, lens, seed=5)
        b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_tree_tiles_in_many_parts(dev, kv_type, D):
    """One tile, or two, of every height in so many parts that groups of them are joined
    first; the sums do not depend on which workgroup comes last."""
    for lens in ([(4, 12000, "tree")], [(7, 14001, "tree")], [(13, 9000, "tree")],
                 [(50, 11000, "tree")], [(60, 5000, "tree"), (11, 7777, "run")],
                 [(66, 9009, "tree")]):
        note(f"tree many parts {kv_type} D={D} {lens}")
        b = Trees(dev, kv_type, 2, 1, D, 64, lens, seed=D)
        out = b.run().clone()
        b.check(out)
        for _ in range(4):
            assert bool((b.run() == out).all())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("n", [3, 40, 150])
def test_tree_rows_that_see_nothing(dev, kv_type, n):
    """Masks without a bit, over no cached token, are rows of zeros; over cached ones they see
    those; through a window past all of them again nothing."""
    note(f"tree rows that see nothing {kv_type} n={n}")
    b = Trees(dev, kv_type, 4, 2, 64, 16, [(n, n, "none"), (n, n + 30, "none")])
    out = b.run()
    b.check(out)
    assert (out[:n] == 0).all()
    # Positions are held to those of the new rows: the last one sees no cached key through a
    # window of 1, the first one's window of 1 holds none either.
    c = Trees(dev, kv_type, 4, 2, 64, 16, [(n, n + 30, "none")], window=1)
    out = c.run(row_positions=i32([2 ** 31 - 1, -5, 0] * n, dev)[:n])
    c.want[:], c.tol = 0, 0
    c.check(out)


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_masks_of_too_few_words(dev, kv_type):
    """Nodes past the mask's words are seen by none, not by themselves either."""
    note(f"tree short masks {kv_type}")
    b = Trees(dev, kv_type, 4, 2, 64, 16, [(100, 180, "tree"), (200, 200, "tree")], words=1)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_bad_pages_and_short_lengths(dev, kv_type):
    """Keys in pages outside the cache are hidden; a request whose rows are more than its
    length (refused by the plan: 0) has rows of zeros where nothing is there."""
    note(f"tree bad pages {kv_type}")
    b = Trees(dev, kv_type, 4, 2, 64, 16, [(5, 100, "tree"), (60, 150, "tree")],
              bad_pages=[(0, 0), (0, 6), (1, 5), (1, 8)])
    b.check(b.run())
    c = Trees(dev, kv_type, 4, 2, 64, 16, [(5, 100, "tree"), (60, 150, "tree")])
    c.kv_lens.copy_(i32([0, 150], dev))
    out = c.run()
    c.want[:5] = 0
    c.check(out)
    c.kv_lens.copy_(i32([-7, -2 ** 31], dev))
    c.want[:] = 0
    c.check(c.run())


@pytest.mark.parametrize("kv_type", ("f16", "bf16"))
@pytest.mark.parametrize("n,D", [(5, 64), (60, 64), (140, 64), (14, 128), (14, 256), (30, 256)])
def test_tree_non_finite_values(dev, kv_type, n, D):
    """A node's NaN or infinite K or V reaches the nodes that see it and no other."""
    import torch
    G, H, page, total = 2, 4, 16, n + 45
    for what, value in (("k", float("nan")), ("v", float("nan")), ("v", float("inf")),
                        ("k", float("inf"))):
        note(f"tree non-finite {kv_type} {what}={value} n={n}")
        b = Trees(dev, kv_type, H, G, D, page, [(n, total, "tree")], seed=n)
        at = total - n + n // 2
        slot = int(b.table[0, at // page]) * page + at % page
        p, r, tile = slot // page, slot % 16, slot % page // 16
        if what == "k":
            b.cache.k.view(-1, G, page // 16, D // 8, 16, 8)[p, 0, tile, 3, r, 5] = value
        else:
            b.cache.v.view(-1, G, page // 16, 2, D, 2, 4)[
                p, 0, tile, r // 4 % 2, 29, r // 8, r % 4] = value
        out = b.run()
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(n, H, D)
        hit = b.seen[0][:, at]
        assert hit.any() and not hit.all()
        mine = slice(0, H // G)
        assert np.abs(got[~hit] - b.want[~hit]).max() <= b.tol
        assert np.abs(got[:, H // G:] - b.want[:, H // G:]).max() <= b.tol
        if what == "k":
            if math.isnan(value):
                assert np.isnan(got[hit][:, mine]).all()
            continue
        x = got[hit][:, mine][..., 29]
        assert (np.isnan(x) if math.isnan(value) else x == value).all()
        other = np.arange(D) != 29
        assert np.abs(got[hit][:, mine][..., other]
                      - b.want[hit][:, mine][..., other]).max() <= b.tol


def test_tree_non_finite_scales(dev):
    """8-bit caches: a node of NaN scales reaches the nodes that see it and no other."""
    import torch
    for n in (6, 50):
        b = Trees(dev, "int8", 4, 2, 64, 16, [(n, n + 20, "tree")], seed=3)
        at = 20 + n // 2
        slot = int(b.table[0, at // 16]) * 16 + at % 16
        for s in (b.cache.k_scale, b.cache.v_scale):
            s.view(-1, 2, 16)[slot // 16, 0, slot % 16] = float("nan")
        note(f"tree NaN scales n={n}")
        out = b.run()
        torch.cuda.synchronize()
        got, hit = out.cpu().numpy().reshape(n, 4, 64), b.seen[0][:, at]
        assert np.isnan(got[hit][:, :2]).all()
        assert np.abs(got[~hit] - b.want[~hit]).max() <= b.tol
        assert np.abs(got[:, 2:] - b.want[:, 2:]).max() <= b.tol


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_chain_and_run_agree(dev, kv_type):
    """A tree without branches is a run of tokens: the bits of the attention of runs."""
    import torch
    for lens, window in (([(1, 700), (9, 3000), (2, 2)], 0), ([(100, 700), (33, 60)], 0),
                         ([(7, 500), (70, 900)], 90)):
        note(f"tree chain {kv_type} {lens}")
        b = Trees(dev, kv_type, 8, 2, 64, 32, [(n, t, "chain") for n, t in lens])
        c = Trees(dev, kv_type, 8, 2, 64, 32, [(n, t, "run") for n, t in lens], window=window)
        runs = empty_f32((c.T, 512), dev)
        capi.paged_attention(c.cache, c.q, runs, 8, c.scale, window, c.table, c.max_pages,
                             c.kv_lens, c.cu, len(lens), c.T)
        c.check(c.run())
        c.check(runs)
        if window == 0:
            runs = empty_f32((b.T, 512), dev)
            capi.paged_attention(b.cache, b.q, runs, 8, b.scale, 0, b.table, b.max_pages,
                                 b.kv_lens, b.cu, len(lens), b.T)
            b.check(b.run())
            b.check(runs)
        torch.cuda.synchronize()


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_strides_streams_and_repeats(dev, kv_type):
    """Strided rows, out over q, another stream, the same bits on every run; rows behind the
    last request are left as they were."""
    import torch
    b = Trees(dev, kv_type, 8, 2, 64, 32, [(4, 3000, "tree"), (40, 700, "tree"), (2, 90, "run")])
    note(f"tree strides {kv_type}")
    first = b.run()
    b.check(first)
    wide_q = torch.zeros(b.T + 3, 8 * 64 + 20, device=dev)
    wide_q[:b.T, :512] = b.q
    wide_out = empty_f32((b.T + 3, 8 * 64 + 4), dev)
    T, mask = b.T, b.mask
    b.T, b.mask = T + 3, torch.cat([mask, mask[:3]])  # rows that no request has
    b.run(out=wide_out[:, :512], q=wide_q[:, :512])
    b.T, b.mask = T, mask
    torch.cuda.synchronize()
    assert torch.equal(wide_out[:T, :512], first) and torch.isnan(wide_out[:, 512:]).all()
    assert torch.isnan(wide_out[T:]).all()
    same = b.q.clone()
    b.run(out=same, q=same)
    torch.cuda.synchronize()
    assert torch.equal(same, first)
    stream = own_stream()
    for _ in range(3):
        other = empty_f32(first.shape, dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            b.run(out=other)
        stream.synchronize()
        assert torch.equal(other, first)


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_graph_replays(dev, kv_type):
    """A captured call follows masks, lengths and kinds on the device; eager calls between."""
    import torch
    b = Trees(dev, kv_type, 8, 2, 64, 32, [(4, 3000, "tree"), (40, 700, "tree"), (2, 90, "run")])
    c = Trees(dev, kv_type, 8, 2, 64, 32, [(4, 1000, "any"), (40, 300, "run"), (2, 70, "tree")],
              seed=2)
    eager = [x.run() for x in (b, c)]
    stream = own_stream()
    capi.workspace_reserve(*capi.paged_attention_workspace_size(b.cache, 8, 3, b.T),
                           stream=stream)
    torch.cuda.synchronize()
    note(f"tree captured {kv_type}")
    held = {n: getattr(b, n).clone() for n in ("q", "table", "kv_lens", "mask", "trees")}
    out = empty_f32(eager[0].shape, dev)
    cache_c = [c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        capi.paged_tree_attention(b.cache, held["q"], out, 8, b.scale, 0, held["table"],
                                  b.max_pages, held["kv_lens"], b.cu, 3, b.T, held["mask"], 1,
                                  None, held["trees"], stream=stream)
    for rep in range(4):
        if rep == 2:
            table = torch.full_like(held["table"], -1)
            table[:, :c.max_pages] = c.table
            held["table"].copy_(table)
            for n in ("q", "kv_lens", "mask", "trees"):
                held[n].copy_(getattr(c, n))
            for x, y in zip((b.cache.k, b.cache.v, b.cache.k_scale, b.cache.v_scale), cache_c):
                if y is not None:
                    x[:y.numel()].copy_(y)
        out.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        extra = c.run()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[rep // 2]), rep
        assert torch.equal(extra, eager[1])


# ---- the accepted path ----

def keep_host(cells, table, page, num_pages, kv_lens, news, granted, keep, counts, lens, stack,
              count):
    """The header's rules, request by request; cells: arrays [layers, slots, ...]."""
    cells, stack, lens = [x.copy() for x in cells], stack.copy(), list(lens)
    top, max_pages = min(max(count, 0), num_pages), table.shape[1]

    def slot(b, pos):
        if pos // page >= max_pages:
            return -1
        p = table[b, pos // page]
        return p * page + pos % page if 0 <= p < num_pages else -1
    for b, n in enumerate(news):
        if not granted[b]:
            continue
        kv = max(int(kv_lens[b]), 0)
        if n <= 0 or kv < n or counts[b] < 0:
            lens[b] = kv
            continue
        path = []
        for i in range(min(int(counts[b]), keep.shape[1], n)):
            if not (path[-1] if path else -1) < keep[b, i] < n:
                break
            path.append(int(keep[b, i]))
        base = kv - n
        moves = [(slot(b, base + r), slot(b, base + i)) for i, r in enumerate(path) if i != r]
        for f, t in moves:
            if f >= 0 and t >= 0:
                for x in cells:
                    x[:, t] = x[:, f]
        lens[b] = base + len(path)
        for j in range(-(-lens[b] // page), min(-(-kv // page), max_pages)):
            if top < num_pages:
                stack[top] = table[b, j]
                top += 1
    return cells, lens, stack, top


def keep_case(rng, dev, kv_type, layers, G, D, page, requests, stride):
    """Random caches, and requests (new, total, path or None) in pages of them."""
    import torch
    need = [-(-t // page) for _, t, _ in requests]
    pages, max_pages, B = sum(need) + 5, max(need + [1]) + 1, len(requests)
    order = rng.permutation(pages)
    table, at = np.full((B, max_pages), -1, np.int64), 2
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    stack = np.full(pages, -1, np.int64)
    stack[:2] = order[:2]
    caches = [capi.PagedCache.allocate(kv_type, pages, page, G, D, dev) for _ in range(layers)]
    for c in caches:
        for x in (c.k, c.v, c.k_scale, c.v_scale):
            if x is not None:
                x.copy_(torch.from_numpy(rng.integers(-120, 120, x.shape)).to(dev))
    keep = rng.integers(-2, 9, (B, stride))
    counts = np.zeros(B, np.int64)
    for b, (n, _, path) in enumerate(requests):
        counts[b] = -1 if path is None else len(path)
        if path:
            keep[b, :min(len(path), stride)] = path[:stride]
    return caches, table, stack, keep, counts, pages


def cells_host(caches, page, G, D):
    out = []
    for i in range(4):
        parts = [cells_of(c, c.struct.num_pages, page, G, D)[i] for c in caches]
        if parts[0] is not None:
            out.append(np.stack([p.float().cpu().numpy() for p in parts]))
    return out


class Keep:
    def __init__(self, dev, rng, kv_type, layers, G, D, page, requests, stride):
        self.page, self.G, self.D, self.requests, self.stride = page, G, D, requests, stride
        (self.caches, self.table, self.stack, self.keep, self.counts,
         self.pages) = keep_case(rng, dev, kv_type, layers, G, D, page, requests, stride)
        self.B, self.dev = len(requests), dev
        self.kv = np.array([t for _, t, _ in requests])
        self.news = [n for n, _, _ in requests]
        self.granted = np.ones(self.B, np.int64)
        self.lens = np.full(self.B, -77)

    def run(self, free_count=2, in_place=False, stack=True, stream=None):
        import torch
        d = self.dev
        lens, st = i32(self.lens, d), i32(self.stack, d)
        count, out = i32([free_count], d), i32([-9], d)
        group = capi.PagedCaches(self.caches)
        capi.paged_kv_keep(group, i32(self.table, d), self.table.shape[1], i32(self.kv, d),
                           i32(prefix(self.news), d), i32(self.granted, d), self.B,
                           i32(self.keep, d), self.stride, i32(self.counts, d), lens,
                           st if stack else None, count if stack else None,
                           (count if in_place else out) if stack else None, stream=stream)
        torch.cuda.synchronize()
        return (cells_host(self.caches, self.page, self.G, self.D), lens.cpu().tolist(),
                st.cpu().numpy(), int((count if in_place else out).item()))

    def check(self, free_count=2, **kw):
        want = keep_host(cells_host(self.caches, self.page, self.G, self.D), self.table,
                         self.page, self.pages, self.kv, self.news, self.granted, self.keep,
                         self.counts, self.lens, self.stack, free_count)
        got = self.run(free_count, **kw)
        for g, w in zip(got[0], want[0]):
            np.testing.assert_array_equal(g, w)
        assert got[1] == want[1]
        if kw.get("stack", True):
            np.testing.assert_array_equal(got[2], want[2])
            assert got[3] == want[3]
        return got


def path_of(rng, n, most):
    return sorted(rng.choice(n, rng.integers(0, min(n, most) + 1), replace=False).tolist())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("G,D,page,layers,B,n,longest", [
    (2, 64, 16, 3, 1, 8, 40), (1, 96, 32, 2, 7, 30, 300), (3, 128, 16, 5, 20, 64, 200),
    (1, 256, 48, 1, 5, 200, 100), (2, 128, 16, 66, 3, 5, 20), (1, 64, 16, 1, 300, 12, 60)])
def test_keep_matches_host_loop(dev, kv_type, G, D, page, layers, B, n, longest):
    note(f"keep {kv_type} G={G} D={D} page={page} layers={layers} B={B} n={n}")
    rng = np.random.default_rng(B + D)
    requests = []
    for b in range(B):
        new = int(rng.integers(1, n + 1))
        total = new + int(rng.integers(0, longest))
        kind = rng.integers(0, 8)
        path = (None if kind == 0 else list(range(new)) if kind == 1 else
                list(range(new))[-6:] if kind == 2 else path_of(rng, new, 24))
        requests.append((new, total, path) if kind != 7 else (0, total, path))
    k = Keep(dev, rng, kv_type, layers, G, D, page, requests, stride=max(24, n))
    k.granted[rng.integers(0, B)] = 0
    k.check(in_place=bool(B % 2))


@pytest.mark.parametrize("kv_type", TYPES)
def test_keep_ends_bad_paths(dev, kv_type):
    """Entries that do not increase, lie outside the rows, counts past the row's stride,
    lengths below the rows, requests that were refused, pages outside the cache, a full stack."""
    rng = np.random.default_rng(8)
    note(f"keep bad paths {kv_type}")
    requests = [(20, 50, [0, 3, 3, 5]), (20, 41, [0, 7, 2]), (9, 60, [-1, 2]), (9, 33, [0, 9, 10]),
                (40, 90, list(range(1, 40))), (12, 30, [2, 5, 11]), (5, 25, [4]), (3, 3, [0, 2]),
                (6, 70, []), (17, 17, [16])]
    k = Keep(dev, rng, kv_type, 2, 2, 64, 16, requests, stride=13)
    k.counts[1] = 2 ** 31 - 1
    k.kv[5] = 4                       # fewer than its rows
    k.kv[6] = 0
    k.granted[7] = 0
    k.table[4, 3] = -1                # rows of it lie in no page
    k.table[4, 5] = k.pages + 9
    k.check()
    for free in (k.pages - 1, k.pages, k.pages + 50, -3):
        k.check(free_count=free)
    k.check(stack=False)


def test_keep_captured(dev):
    """Replays follow paths and lengths on the device; the lengths take the old ones' place."""
    import torch
    rng = np.random.default_rng(4)
    k = Keep(dev, rng, "f16", 3, 2, 64, 16,
             [(9, 30, [0, 4, 7]), (30, 77, [0, 1, 20]), (4, 9, None)], stride=8)
    start = [[x.clone() for x in (c.k, c.v)] for c in k.caches]
    group = capi.PagedCaches(k.caches)
    held = [i32(x, dev) for x in (k.table, k.kv, prefix(k.news), k.granted, k.keep, k.counts,
                                  k.lens, k.stack, [2])]
    first = [x.clone() for x in held]
    stream = own_stream()
    note("keep captured")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        capi.paged_kv_keep(group, held[0], k.table.shape[1], held[1], held[2], held[3], 3,
                           held[4], 8, held[5], held[6], held[7], held[8], held[8],
                           stream=stream)
    for rep in range(4):
        for x, y in zip(held, first):
            x.copy_(y)
        for c, s in zip(k.caches, start):
            c.k.copy_(s[0]), c.v.copy_(s[1])
        k.keep[0, :3] = [0, 2 + rep, 8]
        held[4].copy_(i32(k.keep, dev))
        want = keep_host(cells_host(k.caches, 16, 2, 64), k.table, 16, k.pages, k.kv, k.news,
                         k.granted, k.keep, k.counts, k.lens, k.stack, 2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for g, w in zip(cells_host(k.caches, 16, 2, 64), want[0]):
            np.testing.assert_array_equal(g, w)
        assert held[6].tolist() == want[1] and held[8].item() == want[3]
        np.testing.assert_array_equal(held[7].cpu().numpy(), want[2])


# ---- the write with norms ----

def normed_host(x, w, eps, rope, pos, rope_dim, mode):
    """Extended precision; (value, bound of the rounding to fp32 and of 64-bit work)."""
    x = x.astype(np.longdouble)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.longdouble(np.float32(eps)))
    y = y * w.astype(np.longdouble)
    size = np.abs(y)
    if mode != "none":
        t = rope[pos].astype(np.longdouble)[:, None]
        c, s = t[..., 0], t[..., 1]
        h = rope_dim // 2
        ia = np.arange(h) if mode == "halves" else 2 * np.arange(h)
        ib = ia + h if mode == "halves" else ia + 1
        a, b = y[..., ia].copy(), y[..., ib].copy()
        y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
        size[..., ia] = size[..., ib] = np.abs(a) + np.abs(b)
    return y, np.abs(y) * 2.0 ** -24 + size * 2.0 ** -47 + 2.0 ** -149


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D,rope_dim,mode,page,T,fused", [
    (14, 2, 64, 64, "halves", 16, 1, False), (4, 4, 128, 128, "pairs", 32, 37, True),
    (6, 3, 96, 64, "halves", 16, 130, True), (8, 1, 256, 256, "pairs", 64, 67, False),
    (5, 5, 64, 64, "none", 48, 29, False), (2, 1, 128, 8, "halves", 16, 300, True),
    (3, 1, 96, 96, "pairs", 16, 18, False)])
def test_normed_write(dev, kv_type, H, G, D, rope_dim, mode, page, T, fused):
    import torch
    note(f"normed write {kv_type} H={H} G={G} D={D} rope={rope_dim}/{mode} page={page} T={T}")
    rng = np.random.default_rng(T + D)
    n = H + 2 * G
    qkv = rng.standard_normal((T, n, D)).astype(np.float32)
    qkv *= np.float32(10.0) ** rng.integers(-12, 12, (T, n, 1)).astype(np.float32)
    qkv[T // 2, 0] = 0                # a head of zeros: over sqrt(eps)
    qkv[T - 1, n - 1] = 0             # a V row of zeros
    wq, wk = (rng.standard_normal(D).astype(np.float32) for _ in range(2))
    limit, eps = 500, 1e-5
    rope = rng.uniform(-1, 1, (limit, rope_dim // 2, 2)).astype(np.float32)
    pages = T // page + 8
    slots = rng.permutation(pages * page)[:T].astype(np.int64)
    run = min(T, page) // 4 * 4       # some whole places of four tokens
    slots[:run] = (pages - 1) * page + np.arange(run)
    used = np.isin(slots[run:], slots[:run])
    slots[run:][used] = -1
    pos = rng.integers(0, limit, T)
    if T > 10:
        slots[T - 2] = pages * page
        pos[7] = limit if mode != "none" else pos[7]
    dq = to_dev(qkv.reshape(T, -1), dev)
    parts = [dq[:, :H * D], dq[:, H * D:(H + G) * D], dq[:, (H + G) * D:]]
    if not fused:
        parts = [x.contiguous() for x in parts]
    cache = capi.PagedCache.allocate(kv_type, pages, page, G, D, dev)
    q_out = empty_f32((T, H * D), dev)
    capi.paged_kv_write_normed(cache, parts[0], q_out, H, parts[1], parts[2], to_dev(wq, dev),
                               to_dev(wk, dev), eps, None if mode == "none" else to_dev(rope, dev),
                               limit, rope_dim, mode, i32(pos, dev), i32(slots, dev), T)
    torch.cuda.synchronize()
    placed = pos < limit
    safe = np.where(placed, pos, 0)
    want, bound = normed_host(qkv[:, :H], wq, eps, rope, safe, rope_dim, mode)
    want[~placed] = 0
    got = q_out.cpu().numpy().reshape(T, H, D)
    assert (np.abs(got - want) <= bound).all()
    k, k_bound = normed_host(qkv[:, H:H + G], wk, eps, rope, safe, rope_dim, mode)
    kc, vc, ks, vs = [None if x is None else x.cpu().double().numpy()
                      for x in cells_of(cache, pages, page, G, D)]
    kept = placed & (slots >= 0) & (slots < pages * page)
    at = slots[kept]
    vw, vws = stored_host(qkv[kept, H + G:], kv_type)
    np.testing.assert_array_equal(vc[at], vw.double().numpy())
    k, k_bound = k[kept], k_bound[kept]
    if kv_type == "int8":
        np.testing.assert_array_equal(vs[at], np.where(vws > 2.0 ** -64, vws, 0).astype(np.float64))
        # s is amax / 127 with three roundings; q a whole number at most half a step away, but
        # for the rounding of k, s and their quotient.
        amax = np.abs(k).max(-1)
        assert (np.abs(ks[at] - amax / 127) <= amax / 127 * 2.0 ** -22).all()
        s = ks[at][..., None]
        assert (np.abs(kc[at] * s - k) <= s * (0.5 + 127 * 2.0 ** -22)).all()
    else:
        # The fp32 value rounded again, whichever fp32 value 64-bit work may come to.
        slack = k_bound - np.abs(k) * 2.0 ** -24
        ends = [torch.from_numpy((k + d).astype(np.float32)).to(cache.k.dtype).double().numpy()
                for d in (-slack, slack)]
        assert ((kc[at] == ends[0]) | (kc[at] == ends[1])).all()
    rest = np.ones(pages * page, bool)
    rest[at] = False
    assert (kc[rest] == 0).all() and (vc[rest] == 0).all()


@pytest.mark.parametrize("kv_type", TYPES)
def test_normed_write_in_place_and_non_finite(dev, kv_type):
    """q in place; heads with NaN or infinity are NaN where the formula has it, and no other
    head; eps 0 over a head of zeros is NaN; head_dim 96 leaves lanes without elements."""
    import torch
    H, G, D, T, page = 3, 2, 96, 9, 16
    rng = np.random.default_rng(3)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    k, v = (rng.standard_normal((T, G, D)).astype(np.float32) for _ in range(2))
    k[2, 1, 5], v[3, 0, 63], k[4, 0, 0], q[5, 2, 8], q[1, 0] = np.nan, np.inf, -np.inf, np.inf, 0
    w = np.ones(D, np.float32)
    for eps in (1e-6, 0.0):
        note(f"normed write non-finite {kv_type} eps={eps}")
        cache = capi.PagedCache.allocate(kv_type, 2, page, G, D, dev)
        dq = to_dev(q.reshape(T, -1), dev)
        capi.paged_kv_write_normed(cache, dq, dq, H, to_dev(k.reshape(T, -1), dev),
                                   to_dev(v.reshape(T, -1), dev), to_dev(w, dev), to_dev(w, dev),
                                   eps, None, 0, D, "none", None, i32(np.arange(T) + 3, dev), T)
        torch.cuda.synchronize()
        got = dq.cpu().numpy().reshape(T, H, D)
        with np.errstate(all="ignore"):
            want, bound = normed_host(q, w, eps, None, None, D, "none")
        bad = np.isnan(want.astype(np.float64))
        assert bad[5, 2, 8] and not bad[5, 2, 9] and bad[1, 0].all() == (eps == 0.0)
        np.testing.assert_array_equal(np.isnan(got), bad)
        assert (np.abs(got - want) <= bound)[~bad].all()
        kc, vc, ks, vs = cells_of(cache, 2, page, G, D)
        rows = (kc.float() if ks is None else kc.float() * ks[..., None]).cpu().numpy()[3:3 + T]
        with np.errstate(all="ignore"):
            want, _ = normed_host(k, w, eps, None, None, D, "none")
        nan_rows = np.isnan(want.astype(np.float64)).any(-1)
        np.testing.assert_array_equal(np.isnan(rows).any(-1), nan_rows)


def test_normed_write_captured(dev):
    """Replays read the rows, positions and slots that are there then."""
    import torch
    H, G, D, T, page = 4, 2, 64, 7, 16
    rng = np.random.default_rng(6)
    hold = [torch.zeros(T, n * D, device=dev) for n in (H, G, G)]
    w = to_dev(rng.standard_normal(D).astype(np.float32), dev)
    rope = to_dev(rng.uniform(-1, 1, (50, D // 2, 2)).astype(np.float32), dev)
    pos, slots = i32([0] * T, dev), i32([0] * T, dev)
    caches = [capi.PagedCache.allocate("int8", 4, page, G, D, dev) for _ in range(2)]
    outs = [empty_f32((T, H * D), dev) for _ in range(2)]

    def call(i, stream=None):
        capi.paged_kv_write_normed(caches[i], hold[0], outs[i], H, hold[1], hold[2], w, w, 1e-6,
                                   rope, 50, D, "halves", pos, slots, T, stream=stream)
    stream = own_stream()
    note("normed write captured")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(0, stream)
    for rep in range(3):
        for x in hold:
            x.copy_(torch.randn(x.shape, device=dev))
        pos.copy_(i32(rng.integers(0, 50, T), dev))
        slots.copy_(i32(rng.permutation(4 * page)[:T], dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        call(1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        for n in ("k", "v", "k_scale", "v_scale"):
            assert torch.equal(getattr(caches[0], n), getattr(caches[1], n))


# ---- all of it together ----

@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("window", [0, 20])
def test_steps_of_speculation(dev, kv_type, window):
    """Two layers, three requests, several steps: a prompt each, then trees whose accepted path
    is kept; every layer's cache then holds the accepted tokens in order, in fewest pages, and
    the attention of each step is that of the tokens a row descends from."""
    import torch
    H, G, D, page, B, layers, max_pages, pages = 4, 2, 64, 16, 3, 2, 8, 20
    rng = np.random.default_rng(11 + window)
    rope = torch.empty(200, D // 2, 2, device=dev)
    capi.rope_table(rope, 200, D)
    rope_h = rope.cpu().numpy()
    wq, wk = (1 + 0.2 * rng.standard_normal(D)).astype(np.float32), np.ones(D, np.float32)
    caches = [capi.PagedCache.allocate(kv_type, pages, page, G, D, dev) for _ in range(layers)]
    group = capi.PagedCaches(caches)
    table = i32(np.full((B, max_pages), -1), dev)
    stack, count, lens = i32(np.arange(pages), dev), i32([pages], dev), i32([0] * B, dev)
    held = [[(np.zeros((0, G, D)),) * 2 for _ in range(B)] for _ in range(layers)]
    scale, total = D ** -0.5, [0] * B
    for step in range(6):
        news = [17, 40, 3] if step == 0 else [8, 1 + 5 * step, 30]
        kinds = [0, 0, 0] if step == 0 else [1, 1, step % 2]
        T = sum(news)
        note(f"speculation {kv_type} window={window} step {step} {news}")
        kv, granted = (i32([0] * B, dev) for _ in range(2))
        cu, pos, slots = i32([0] * (B + 1), dev), i32([0] * T, dev), i32([0] * T, dev)
        capi.paged_plan(lens, i32(news, dev), B, table, max_pages, page, pages, stack, count,
                        count, T, kv, cu, pos, slots, granted)
        masks, depth, seen = np.zeros((T, 1), np.int64), np.zeros(T, np.int64), []
        first = prefix(news)
        for b, n in enumerate(news):
            new, d = tree_masks(rng, n, "tree" if kinds[b] else "chain")
            masks[first[b]:first[b + 1]] = words_of(new, 1)
            depth[first[b]:first[b + 1]] = d
            seen.append(new)
        index = np.concatenate([np.arange(n) for n in news])
        pos = pos + i32(depth - index, dev)
        trees = i32(kinds, dev)
        for layer, cache in enumerate(caches):
            qkv = rng.standard_normal((T, H + 2 * G, D)).astype(np.float32)
            d = to_dev(qkv.reshape(T, -1), dev)
            q, k, v = d.split([H * D, G * D, G * D], dim=1)
            capi.paged_kv_write_normed(cache, q, q, H, k, v, to_dev(wq, dev), to_dev(wk, dev),
                                       1e-6, rope, 200, D, "halves", pos, slots, T)
            out = empty_f32((T, H * D), dev)
            capi.paged_tree_attention(cache, q, out, H, scale, window, table, max_pages, kv, cu,
                                      B, T, to_dev(masks, dev), 1, pos, trees)
            torch.cuda.synchronize()
            p = pos.cpu().numpy()
            q_host = q.cpu().numpy().reshape(T, H, D)
            want_q, bound = normed_host(qkv[:, :H], wq, 1e-6, rope_h, p, D, "halves")
            assert (np.abs(q_host - want_q) <= bound).all()
            k_host, _ = normed_host(qkv[:, H:H + G], wk, 1e-6, rope_h, p, D, "halves")
            k_host = k_host.astype(np.float32)
            got = out.cpu().numpy().reshape(T, H, D)
            for b, n in enumerate(news):
                rows = slice(first[b], first[b + 1])
                new = []
                for x in (k_host[rows], qkv[rows, H + G:]):
                    c, s = stored_host(x, kv_type)
                    c = c.double().numpy()
                    new.append(c if s is None else c * s.double().numpy()[..., None])
                kk, vv = (np.concatenate([h, x]) for h, x in zip(held[layer][b], new))
                base = len(held[layer][b][0])
                see = np.ones((n, base + n), bool)
                see[:, base:] = seen[b]
                if window:
                    # A run's window covers its own rows too, a tree's masks alone decide.
                    reach = base if kinds[b] else base + n
                    see[:, :reach] &= np.arange(reach)[None] > p[rows][:, None] - window
                o, tol = attention_host(q_host[rows], kk, vv, see, scale)
                # One rounding of k may fall to the other side: a step of its type.
                step_k = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7, "int8": 1 / 127}[kv_type]
                ds = scale * np.abs(q_host[rows]).sum(-1).max() * 2.0 ** -24 * step_k * 2
                assert np.abs(got[rows] - o).max() <= tol + 4 * ds * np.abs(vv).max()
                held[layer][b] = [kk, vv]
        # A path from the root down, one request's tree rejected to its root.
        keep, counts = np.full((B, 40), -1), np.full(B, -1)
        for b, n in enumerate(news):
            if not kinds[b]:
                continue
            leaf = int(rng.integers(0, n)) if b else 0
            path = np.flatnonzero(seen[b][leaf])
            keep[b, :len(path)], counts[b] = path, len(path)
        capi.paged_kv_keep(group, table, max_pages, kv, cu, granted, B, i32(keep, dev), 40,
                           i32(counts, dev), lens, stack, count, count)
        torch.cuda.synchronize()
        for b, n in enumerate(news):
            rows = np.arange(n) if counts[b] < 0 else keep[b, :counts[b]]
            for layer in range(layers):
                base = len(held[layer][b][0]) - n
                order = np.concatenate([np.arange(base), base + rows])
                held[layer][b] = [x[order] for x in held[layer][b]]
            total[b] = len(held[0][b][0])
        assert lens.tolist() == total
        assert count.item() == pages - sum(-(-t // page) for t in total)
        tab, free = table.cpu().numpy(), set(stack.cpu().numpy()[:count.item()].tolist())
        assert len(free) == count.item()
        for layer, cache in enumerate(caches):
            kc, vc, ks, vs = [None if x is None else x.cpu().double().numpy()
                              for x in cells_of(cache, pages, page, G, D)]
            for b in range(B):
                mine = tab[b, :-(-total[b] // page)]
                assert not free & set(mine.tolist())
                at = mine[np.arange(total[b]) // page] * page + np.arange(total[b]) % page
                for x, s, want, exact in ((kc, ks, held[layer][b][0], False),
                                          (vc, vs, held[layer][b][1], True)):
                    x = x[at] if s is None else x[at] * s[at][..., None]
                    # k: a step of its type where a rounding fell to the other side.
                    slack = 0.0 if exact else 2.0 * {"f16": 2.0 ** -10, "bf16": 2.0 ** -7,
                                                     "int8": 1 / 127}[kv_type]
                    assert (np.abs(x - want) <= slack * np.abs(want).max(initial=0)).all()


@pytest.mark.parametrize("kv_type", ["int8", "f16"])
def test_far_pages(dev, kv_type):
    """Pages more than 2^32 elements and bytes into a cache: the write, the attention and the
    move do there what they do in near pages, bit for bit."""
    import torch
    H, G, D, page, T, pages = 16, 8, 256, 64, 100, 4
    first = 2 ** 32 // (G * page * D) + 9
    note(f"far pages {kv_type}")
    rng = np.random.default_rng(3)
    host = rng.standard_normal((T, (H + 2 * G) * D)).astype(np.float32)
    mask, depth = tree_masks(rng, T, "tree")
    path = np.flatnonzero(mask[T - 1])
    w = torch.ones(D, device=dev)
    outs = []
    for start in (0, first):
        cache = capi.PagedCache.allocate(kv_type, start + pages, page, G, D, dev)
        q, k, v = to_dev(host, dev).split([H * D, G * D, G * D], dim=1)
        order = start + np.array([2, 0, 3, 1])
        table, kv, cu = i32(order[None], dev), i32([150], dev), i32([0, T], dev)
        at = 50 + np.arange(T)
        slots = i32(order[at // page] * page + at % page, dev)
        capi.paged_kv_write_normed(cache, q, q, H, k, v, w, w, 1e-6, None, 0, D, "none", None,
                                   slots, T)
        out = empty_f32((T, H * D), dev)
        capi.paged_tree_attention(cache, q, out, H, D ** -0.5, 0, table, pages, kv, cu, 1, T,
                                  to_dev(words_of(mask, 2), dev), 2)
        kept, count = i32([0], dev), i32([0], dev)
        stack = i32(np.full(start + pages, -1), dev)
        capi.paged_kv_keep(capi.PagedCaches([cache]), table, pages, kv, cu, i32([1], dev), 1,
                           i32(path[None], dev), len(path), i32([len(path)], dev), kept, stack,
                           count, count)
        torch.cuda.synchronize()
        part = [x[start * (x.numel() // (start + pages)):].clone()
                for x in (cache.k, cache.v, cache.k_scale, cache.v_scale) if x is not None]
        near = [x[:start * (x.numel() // (start + pages))] for x in (cache.k, cache.v)]
        assert not any(bool(x.view(torch.uint8)[i::4096].any()) for x in near for i in (0, 2049))
        n = int(count.item())
        outs.append(part + [out, kept, stack[:n] - start])
        del cache, near
    assert len(outs[0][-1]) > 0 and outs[0][-2].item() == 50 + len(path)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_calls_at_once_and_others_between(dev):
    """Calls on two streams at once have workspaces of their own; calls of other kinds on the
    same stream find its counters as they leave them."""
    import torch
    big = Trees(dev, "f16", 2, 1, 128, 64, [(50, 11000, "tree")], seed=4)
    few = Trees(dev, "f16", 2, 1, 128, 64, [(4, 12000, "tree"), (13, 700, "tree")], seed=5)
    x = torch.randn(3, 40000, device=dev)
    want = [b.run().clone() for b in (big, few)]
    ids = torch.empty(3, dtype=torch.int32, device=dev)
    lp, tok = empty_f32((3, 1), dev), i32([[5], [39999], [0]], dev)
    streams = [own_stream(), own_stream()]
    outs = [[empty_f32(w.shape, dev) for _ in range(8)] for w in want]
    torch.cuda.synchronize()
    note("trees on two streams, other calls between")
    for i in range(8):
        for b, s, o in zip((big, few), streams, outs):
            b.run(out=o[i], stream=s)
        capi.argmax(x, 3, 40000, ids, stream=streams[0])
        capi.token_logprobs(x, 3, 40000, tok, 1, 0, lp, None, None, None, stream=streams[0])
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for y in o:
            assert torch.equal(y, w)
    assert torch.equal(ids.long(), x.argmax(1))
    # A term's error is (distance to the maximum + 1) 2^-22, and no two of 120000 normal values
    # are 11 apart.
    right = torch.log_softmax(x.double(), 1).gather(1, tok.long())
    assert bool(((lp - right).abs() <= 2.0 ** -22 * 12 + right.abs() * 2.0 ** -24).all())


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_many_requests(dev, kv_type):
    """More requests than a workgroup has threads, trees of every size, runs and none in turn."""
    rng = np.random.default_rng(9)
    kinds = ["tree", "run", "any", "chain", "none"]
    for B in (257, 700):
        lens = []
        for b in range(B):
            n = int(rng.choice([0, 1, 2, 5, 16, 17, 33, 70]))
            lens.append((n, n + int(rng.choice([0, 1, 40, 100])), kinds[b % 5]))
        note(f"tree many requests {kv_type} {B}")
        b = Trees(dev, kv_type, 2, 1, 64, 16, lens, seed=B, window=30 if B == 700 else 0)
        b.check(b.run())


def test_tree_widest_masks(dev):
    """More nodes than the widest masks name: the last ones are seen by none."""
    n = 64 * 64 + 70
    note("tree widest masks")
    b = Trees(dev, "f16", 1, 1, 64, 64, [(n, n + 100, "tree"), (3, 9, "tree")], words=64)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_tree_joined_groups_weigh_parts_by_their_own_maxima(dev, kv_type, D):
    """Tiles of 9 to 32 rows in more than 12 parts, a group of which is joined into the place of
    its first one while other waves may still read that one's maxima and sums.  Logits of a
    standard deviation of 8: the parts' maxima are apart by more than the tolerance, so that
    sums weighed by another part's show; the same bits on every run."""
    for n, total in ((9, 12000), (13, 9000), (16, 14001), (17, 11000), (26, 8000), (32, 15000)):
        note(f"tree joined groups {kv_type} D={D} {n} over {total}")
        b = Trees(dev, kv_type, 1, 1, D, 64, [(n, total, "tree")], seed=n, scale=4 * D ** -0.5)
        out = b.run().clone()
        b.check(out)
        for _ in range(12):
            assert bool((b.run() == out).all())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("D", [96, 128, 256])
def test_tree_several_tiles_a_workgroup(dev, kv_type, D):
    """More tiles than workgroups, several one after the other in each: trees of 17 to 64 rows
    only, whose next loads go out before a tile is joined, and all heights in turn with runs
    between; the same bits again."""
    rng = np.random.default_rng(D)
    some = [(n, n + int(rng.choice([0, 3, 60, 200])), "tree")
            for n in rng.integers(17, 65, 300).tolist()]
    kinds = ["tree", "any", "run", "chain", "tree", "none", "tree"]
    mixed = []
    for b in range(300):
        n = int(rng.choice([0, 1, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 40, 70]))
        mixed.append((n, n + int(rng.choice([0, 1, 40, 150])), kinds[b % 7]))
    for lens, H, G, window in ((some, 2, 2, 50), (mixed, 6, 3, 0)):
        note(f"tree several tiles {kv_type} D={D} H={H} G={G} window={window}")
        b = Trees(dev, kv_type, H, G, D, 16, lens, seed=D + H, window=window)
        out = b.run().clone()
        b.check(out)
        for _ in range(3):
            assert bool((b.run() == out).all())


@pytest.mark.parametrize("kv_type", TYPES)
def test_tree_chain_is_near_the_run(dev, kv_type):
    """A tree without branches is a run of tokens.  The tiles, cuts and joins of the two calls
    differ, so their sums do, each by the tolerance at most."""
    import torch
    for lens, D in (([(1, 700), (9, 3000), (2, 2)], 64), ([(100, 700), (33, 60)], 128),
                    ([(40, 900), (17, 5000)], 256)):
        note(f"tree chain and run {kv_type} {lens}")
        b = Trees(dev, kv_type, 4, 2, D, 32, [(n, t, "chain") for n, t in lens], seed=D)
        trees, runs = b.run(), empty_f32((b.T, 4 * D), dev)
        capi.paged_attention(b.cache, b.q, runs, 4, b.scale, 0, b.table, b.max_pages, b.kv_lens,
                             b.cu, len(lens), b.T)
        torch.cuda.synchronize()
        assert (trees - runs).abs().max().item() <= 2 * b.tol
