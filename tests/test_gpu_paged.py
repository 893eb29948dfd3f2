"""GPU numerics of the paged KV cache (include/mle_paged.h) against plain implementations.

The plan is compared entry by entry with a host loop over the requests, the write bit by bit
with the rotation and the cell formats in 64 bits, and the attention with softmax in 64 bits
over the values that the cache holds.

Tolerance of the attention: the kernel's q differs from the fp32 one by less than 2^-22 of a
row's largest element, products are exact, and sums of D terms in fp32 are off by less than
(D + 8) 2^-24 of the sum of magnitudes; a logit is so off by less than
ds = (D + 16) 2^-22 scale max_j sum_d |q_d k_jd|.  Weights e^s are off by ds + 2^-20 relative
(exp2 of a rounded product, the 8-bit scales' logarithms), sums over the keys by their number
n of partial sums (at most keys / 8 + 64) times 2^-24, and both numerator and denominator are
off so: |error| <= 2 max|v| (ds + 2^-20 + (keys / 8 + 64) 2^-24).
"""
import math

import numpy as np
import pytest

from helpers import empty_f32, note, own_stream, slower_by, to_dev
from llmengine_amd import capi

pytestmark = pytest.mark.gpu

TYPES = ("f16", "bf16", "int8")


def i32(values, dev):
    return to_dev(np.asarray(values, np.int32), dev)


def prefix(values):
    return np.concatenate([[0], np.cumsum(values)]).astype(np.int64)


# ---- the plan ----

def plan_host(cached, new, table, page, num_pages, stack, count, tokens):
    """The header's rules, request by request."""
    B, max_pages = table.shape
    table, stack = table.copy(), stack.copy()
    top = min(max(count, 0), num_pages)
    for b in range(B):
        if new[b] < 0:
            for j in range(min(-(-max(cached[b], 0) // page), max_pages)):
                if top < num_pages:
                    stack[top] = table[b, j]
                    top += 1
    whole, asked, rows = top, 0, 0
    kv, granted, cu = [], [], [0]
    pos, slots = np.zeros(tokens, np.int32), np.full(tokens, -1, np.int32)
    for b in range(B):
        want, first = max(int(new[b]), 0), rows
        rows += want
        cu.append(min(rows, tokens))
        if new[b] < 0:
            kv.append(0)
            granted.append(1)
            continue
        have, need = -(-int(cached[b]) // page), -(-(int(cached[b]) + want) // page)
        ok = rows <= tokens and need <= max_pages
        if ok:
            asked += need - have
            ok = need == have or asked <= whole
        if ok:
            for j in range(have, need):
                table[b, j] = stack[whole - 1 - (asked - need + j)]
                top = whole - asked
            for i in range(want):
                p = int(cached[b]) + i
                pos[first + i] = p
                pg = table[b, p // page]
                slots[first + i] = pg * page + p % page if 0 <= pg < num_pages else -1
        kv.append(int(cached[b]) + want if ok else 0)
        granted.append(int(ok))
    return table, stack, top, kv, cu, pos, slots, granted


def plan_case(rng, B, page, lens, news, free, max_pages, extra=0):
    have = [-(-c // page) for c in lens]
    num_pages = sum(have) + free + extra
    order = rng.permutation(num_pages).astype(np.int32)
    table = np.full((B, max_pages), -1, np.int32)
    at = free
    for b, h in enumerate(have):
        table[b, :h] = order[at:at + h]
        at += h
    stack = np.full(num_pages, -1, np.int32)
    stack[:free] = order[:free]
    return table, stack, num_pages


def run_plan(dev, cached, new, table, page, num_pages, stack, count, tokens):
    import torch
    B, max_pages = table.shape
    d = dict(cached=i32(cached, dev), new=i32(new, dev), table=i32(table, dev),
             stack=i32(stack, dev), count=i32([count], dev))
    out = {n: torch.full((max(k, 1),), -7, dtype=torch.int32, device=dev)
           for n, k in (("count", 1), ("kv", B), ("cu", B + 1), ("pos", tokens),
                        ("slots", tokens), ("granted", B))}
    for _ in range(2):  # a repeated call gives the same
        capi.paged_plan(d["cached"], d["new"], B, d["table"], max_pages, page, num_pages,
                        d["stack"], d["count"], out["count"], tokens, out["kv"], out["cu"],
                        out["pos"], out["slots"], out["granted"])
    torch.cuda.synchronize()
    o = {n: x.cpu().numpy() for n, x in out.items()}
    return (d["table"].cpu().numpy(), d["stack"].cpu().numpy(), int(o["count"][0]), o["kv"],
            o["cu"], o["pos"][:tokens], o["slots"][:tokens], o["granted"])


@pytest.mark.parametrize("B,page,longest,most_new,short,finished,slack", [
    (1, 16, 1, 1, False, 0, 0), (1, 16, 40, 0, False, 0, 3), (5, 16, 100, 40, True, 1, 0),
    (64, 32, 900, 1, False, 3, 0), (65, 48, 300, 1, True, 9, 5), (300, 16, 200, 60, True, 30, 0),
    (1025, 16, 90, 3, True, 70, 0), (2500, 32, 50, 2, False, 100, 11),
    (40, 128, 2000, 600, True, 4, 0), (3, 1024, 5000, 9000, False, 0, 1)])
def test_plan_matches_host_loop(dev, B, page, longest, most_new, short, finished, slack):
    note(f"plan B={B} page={page} longest={longest} new={most_new} short={short}")
    rng = np.random.default_rng(B * 7 + page)
    cached = rng.integers(0, longest + 1, B)
    new = rng.integers(0, most_new + 1, B)
    new[rng.choice(B, finished, replace=False)] = -1
    asked = sum(-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new) if n > 0)
    free = asked * 2 // 3 if short else asked + 3
    max_pages = max(-(-(c + max(n, 0)) // page) for c, n in zip(cached, new)) + 1
    table, stack, num_pages = plan_case(rng, B, page, cached, new, free, max_pages)
    tokens = int(np.maximum(new, 0).sum()) + slack
    args = (cached, new, table, page, num_pages, stack, free, tokens)
    for got, want in zip(run_plan(dev, *args), plan_host(*args)):
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("tokens_of_one", [3, 700])
def test_plan_captured(dev, tokens_of_one):
    """Replays follow the lengths on the device, with one workgroup and with several; the new
    free count takes the place of the old one."""
    import torch
    rng = np.random.default_rng(tokens_of_one)
    B, page = 12, 16
    cached = rng.integers(0, 200, B)
    new = np.full(B, tokens_of_one)
    new[[2, 7]] = -1
    tokens, max_pages = 10 * tokens_of_one, 64
    table, stack, num_pages = plan_case(rng, B, page, cached, new, 480, max_pages)
    held = [i32(x, dev) for x in (cached, new, table, stack, [480])]
    start = [x.clone() for x in held]
    out = [torch.zeros(n, dtype=torch.int32, device=dev) for n in (B, B + 1, tokens, tokens, B)]
    stream = torch.cuda.Stream()
    capi.workspace_reserve(256, 32, stream=stream)
    torch.cuda.synchronize()
    note(f"plan captured {tokens}")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        capi.paged_plan(held[0], held[1], B, held[2], max_pages, page, num_pages, held[3],
                        held[4], held[4], tokens, *out, stream=stream)
    for rep in range(4):
        lens = (cached + 5 * rep) * (new >= 0) + cached * (new < 0)
        for x, y in zip(held, start):
            x.copy_(y)
        held[0].copy_(i32(lens, dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [held[2], held[3], held[4], *out]
        want = plan_host(lens, new, table, page, num_pages, stack, 480, tokens)
        for g, w in zip(got, want):
            np.testing.assert_array_equal(g.cpu().numpy().reshape(-1),
                                          np.asarray(w).reshape(-1))


def test_plan_refuses_what_does_not_fit(dev):
    """Requests past max_pages, rows past `tokens`, negative lengths and bad page numbers."""
    rng = np.random.default_rng(5)
    cached, new = np.array([20, 10, 33, 0, 7]), np.array([5, 100, 3, 16, 2])
    table, stack, num_pages = plan_case(rng, 5, 16, cached, new, 6, 4)
    table[2, 2] = num_pages + 5          # row 2 lies in a page outside the cache
    for tokens in (126, 124, 60, 5, 0):  # all rows, then fewer and fewer of them
        note(f"plan refusals tokens={tokens}")
        args = (cached, new, table, 16, num_pages, stack, 6, tokens)
        for got, want in zip(run_plan(dev, *args), plan_host(*args)):
            np.testing.assert_array_equal(got, want)


def test_plan_rows_past_the_end_refuse_only_requests_with_rows(dev):
    """Requests without new tokens have no row that passes `tokens`: behind one that does,
    they keep their lengths, and their pages where they hold any."""
    cached, new = [20, 5, 33, 0, 7, 16], [3, 90, 0, 0, 2, -1]
    table, stack, num_pages = plan_case(np.random.default_rng(2), 6, 16, cached, new, 12, 8)
    for tokens in (95, 94, 10, 3, 2, 0):
        note(f"plan rows past the end tokens={tokens}")
        got = run_plan(dev, np.array(cached), np.array(new), table, 16, num_pages, stack, 12,
                       tokens)
        kv, cu, granted = got[3], got[4], got[7]
        ok = [rows <= tokens for rows in (3, 93, 0, 0, 95)] + [True]
        assert granted.tolist() == [int(x) for x in ok]
        assert kv.tolist() == [(c + max(n, 0)) * (x and n >= 0)
                               for c, n, x in zip(cached, new, ok)]
        assert cu.tolist() == [0] + [min(r, tokens) for r in (3, 93, 93, 93, 95, 95)]
        assert got[2] == 12 + 1 - 5 * ok[1]  # 5 to 95 tokens: 5 pages more


# ---- rotations and the write ----

@pytest.mark.parametrize("rope_dim,theta,factors", [(64, 10000.0, False), (128, 5e5, True),
                                                    (8, 1e6, False)])
def test_rope_table(dev, rope_dim, theta, factors):
    import torch
    half, n = rope_dim // 2, 9001
    f = np.linspace(1, 8, half).astype(np.float32) if factors else None
    table = empty_f32((n, half, 2), dev)
    capi.rope_table(table, n, rope_dim, theta, to_dev(f, dev) if factors else None)
    torch.cuda.synchronize()
    a = np.arange(n)[:, None] * theta ** (-np.arange(half) / half)
    if factors:
        a = a / f.astype(np.float64)
    want = np.stack([np.cos(a), np.sin(a)], -1)
    # Angles up to 9001 are off by a few ulps of 64 bits (2^-38); then one rounding.
    np.testing.assert_allclose(table.cpu().numpy(), want, rtol=2.0 ** -24, atol=2.0 ** -36)


def rotate_host(x, rope, pos, rope_dim, mode):
    """x [T, heads, D] fp32; exact products and sums (53 bits hold them), one rounding."""
    if mode == "none":
        return x
    out = x.copy()
    t = rope[pos].astype(np.longdouble)[:, None]
    c, s = t[..., 0], t[..., 1]
    h = rope_dim // 2
    ia = np.arange(h) if mode == "halves" else 2 * np.arange(h)
    ib = ia + h if mode == "halves" else ia + 1
    a, b = x[..., ia].astype(np.longdouble), x[..., ib].astype(np.longdouble)
    out[..., ia] = (a * c - b * s).astype(np.float64).astype(np.float32)
    out[..., ib] = (a * s + b * c).astype(np.float64).astype(np.float32)
    return out


def cells_of(cache, pages, page, G, D):
    """(K, V) of a cache as [slot, G, D] tensors in the cache's type, by the header's layout,
    and the scales as [slot, G] (or None)."""
    k = cache.k.view(pages, G, page // 16, D // 8, 16, 8).permute(0, 2, 4, 1, 3, 5)
    v = cache.v.view(pages, G, page // 16, 2, D, 2, 4).permute(0, 2, 5, 3, 6, 1, 4)
    scales = [None if s is None else s.view(pages, G, page).permute(0, 2, 1).reshape(-1, G)
              for s in (cache.k_scale, cache.v_scale)]
    return k.reshape(-1, G, D), v.reshape(-1, G, D), *scales


def stored_host(x, kv_type):
    """[T, G, D] fp32 -> (cells, scales) as the header says."""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x))
    if kv_type != "int8":
        return t.to({"f16": torch.float16, "bf16": torch.bfloat16}[kv_type]), None
    amax = t.abs().amax(-1)
    s = amax * torch.tensor(1.0 / 127.0, dtype=torch.float32)
    q = torch.where(s[..., None] > 0, (t / s[..., None]).round(), 0.0).clamp(-127, 127)
    return q.to(torch.int8), s


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D,rope_dim,mode,page,T,fused", [
    (14, 2, 64, 64, "halves", 16, 1, False), (4, 4, 128, 128, "pairs", 32, 37, True),
    (6, 3, 96, 64, "halves", 16, 130, True), (8, 1, 256, 256, "pairs", 64, 67, False),
    (5, 5, 64, 64, "none", 48, 29, False), (2, 1, 128, 8, "halves", 16, 300, True),
    (3, 1, 96, 96, "pairs", 16, 18, False)])
def test_write_bits(dev, kv_type, H, G, D, rope_dim, mode, page, T, fused):
    import torch
    note(f"write {kv_type} H={H} G={G} D={D} rope={rope_dim}/{mode} page={page} T={T}")
    rng = np.random.default_rng(T + D)
    n = H + 2 * G
    qkv = rng.standard_normal((T, n, D)).astype(np.float32)
    qkv[T // 2, H:] *= 1e-3
    qkv[T - 1, n - 1] = 0            # a V row of zeros
    limit = 500
    rope = rng.uniform(-1, 1, (limit, rope_dim // 2, 2)).astype(np.float32)
    # Runs of consecutive slots from any offset, some rows nowhere, one past the rope's end.
    pages = T // page * 2 + 8 * (T // 40 + 1)
    free = rng.permutation(pages)
    pos, slots, at, p = [], [], 0, int(rng.integers(0, 9))
    for t in range(T):
        if t % 41 == 40:
            p, at = int(rng.integers(0, 60)), at + p // page + 1
        pos.append(p)
        slots.append(free[(at + p // page) % pages] * page + p % page)
        p += 1
    pos, slots = np.array(pos, np.int64) % limit, np.array(slots, np.int64)
    if T > 10:
        slots[5], slots[9] = -1, pages * page
        pos[7] = limit if mode != "none" else pos[7]
    dq = to_dev(qkv.reshape(T, -1), dev)
    parts = [dq[:, :H * D], dq[:, H * D:(H + G) * D], dq[:, (H + G) * D:]]
    if not fused:
        parts = [x.contiguous() for x in parts]
    cache = capi.PagedCache.allocate(kv_type, pages, page, G, D, dev)
    q_out = empty_f32((T, H * D), dev)
    capi.paged_kv_write(cache, parts[0], q_out, H, parts[1], parts[2],
                        None if mode == "none" else to_dev(rope, dev), limit, rope_dim, mode,
                        i32(pos, dev), i32(slots, dev), T)
    torch.cuda.synchronize()
    placed = pos < limit
    safe = np.where(placed, pos, 0)
    want_q = rotate_host(qkv[:, :H], rope, safe, rope_dim, mode)
    want_q[~placed] = 0
    np.testing.assert_array_equal(q_out.cpu().numpy().reshape(T, H, D), want_q)
    k = rotate_host(qkv[:, H:H + G], rope, safe, rope_dim, mode)
    got = [None if x is None else x.cpu() for x in cells_of(cache, pages, page, G, D)]
    want = [torch.zeros_like(x) if x is not None else None for x in got]
    kept = placed & (slots >= 0) & (slots < pages * page)
    last = {int(s): t for t, s in enumerate(slots) if kept[t]}
    rows, ts = list(last), list(last.values())
    if len(set(slots[kept])) != kept.sum():
        pytest.fail("the test's slots repeat")
    for i, x in ((0, k), (1, qkv[:, H + G:])):
        c, s = stored_host(x, kv_type)
        want[i][rows] = c[ts]
        if s is not None:
            want[2 + i][rows] = s[ts]
    for g, w in zip(got, want):
        if w is not None:
            assert torch.equal(g, w)


@pytest.mark.parametrize("kv_type", TYPES)
def test_write_in_place_and_non_finite(dev, kv_type):
    """q rotated in place; rows with NaN or infinity read back as such, never as numbers."""
    import torch
    H, G, D, T, page = 3, 2, 64, 9, 16
    rng = np.random.default_rng(3)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    k, v = (rng.standard_normal((T, G, D)).astype(np.float32) for _ in range(2))
    k[2, 1, 5], v[3, 0, 63], v[8, 1, 0], k[4, 0, 0] = np.nan, np.inf, np.nan, -np.inf
    rope = rng.uniform(-1, 1, (T, D // 2, 2)).astype(np.float32)
    cache = capi.PagedCache.allocate(kv_type, 2, page, G, D, dev)
    dq = to_dev(q.reshape(T, -1), dev)
    capi.paged_kv_write(cache, dq, dq, H, to_dev(k.reshape(T, -1), dev),
                        to_dev(v.reshape(T, -1), dev), to_dev(rope, dev), T, D, "halves",
                        i32(np.arange(T), dev), i32(np.arange(T) + 3, dev), T)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(dq.cpu().numpy().reshape(T, H, D),
                                  rotate_host(q, rope, np.arange(T), D, "halves"))
    ck, cv, ks, vs = cells_of(cache, 2, page, G, D)
    values = [x.float() if s is None else x.float() * s[..., None] for x, s in ((ck, ks),
                                                                               (cv, vs))]
    want_bad = [np.zeros((T, G), bool) for _ in range(2)]
    for i, x in ((0, k), (1, v)):
        want_bad[i] = ~np.isfinite(x).all(-1)
    for x, bad in zip(values, want_bad):
        finite = torch.isfinite(x).all(-1).cpu().numpy()[3:3 + T]
        np.testing.assert_array_equal(~finite, bad)


# ---- the attention ----

def make_cache(rng, dev, kv_type, pages, page, G, D, poison=True):
    """A cache that holds NaN wherever fill_pages does not put values."""
    import torch
    cache = capi.PagedCache.allocate(kv_type, pages, page, G, D, dev)
    if poison:
        if kv_type == "int8":
            cache.k.fill_(-128), cache.v.fill_(127)
            cache.k_scale.fill_(float("nan")), cache.v_scale.fill_(float("nan"))
        else:
            cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    return cache


def put(cache, kv_type, page, slots, k, v):
    """k, v [n, G, D] fp32 into `slots`; returns what the cache holds of them, 64 bits."""
    import torch
    G, D = k.shape[1:]
    slots = torch.as_tensor(slots, device=cache.k.device)
    p, t = slots // page, slots % page
    kc = cache.k.view(-1, G, page // 16, D // 8, 16, 8)
    vc = cache.v.view(-1, G, page // 16, 2, D, 2, 4)
    r, tile = t % 16, t // 16
    out = []
    for x, is_k in ((k, True), (v, False)):
        c, s = stored_host(x, kv_type)
        c = c.to(cache.k.device)
        if is_k:
            kc[p, :, tile, :, r] = c.view(-1, G, D // 8, 8)
        else:
            vc[p, :, tile, r // 4 % 2, :, r // 8, r % 4] = c
        if s is not None:
            (cache.k_scale if is_k else cache.v_scale).view(-1, G, page)[p, :, t] = \
                s.to(cache.k.device)
            out.append(c.cpu().double().numpy() * s.double().numpy()[..., None])
        else:
            out.append(c.cpu().double().numpy())
    return out


def attention_host(q, k, v, pos, window, scale, ok=None):
    """q [n, H, D], k/v [keys, G, D] in 64 bits; returns (out, tolerance)."""
    n, H, D = q.shape
    R = H // k.shape[1]
    j = np.arange(k.shape[0])
    seen = j[None] <= pos[:, None]
    if window:
        seen &= j[None] > pos[:, None] - window
    if ok is not None:
        seen &= ok[None]
    out, tol = np.zeros((n, H, D)), 0.0
    for h in range(H):
        kk, vv = k[:, h // R], v[:, h // R]
        s = scale * (q[:, h].astype(np.float64) @ kk.T)
        s = np.where(seen, s, -np.inf)
        top = s.max(-1, keepdims=True) if s.shape[1] else np.full((n, 1), -np.inf)
        e = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
        z = e.sum(-1, keepdims=True)
        out[:, h] = (e @ vv) / np.where(z > 0, z, 1)
        if not seen.any():
            continue
        use = seen.any(0)
        ds = (D + 16) * 2.0 ** -22 * abs(scale) * (np.abs(q[:, h]) @ np.abs(kk[use]).T).max()
        tol = max(tol, 2 * np.abs(vv[use]).max()
                  * (ds + 2.0 ** -20 + (use.sum() / 8 + 64) * 2.0 ** -24))
    return out, tol


class Batch:
    """A batch of sequences (new, total) in a poisoned cache, and its expected outputs."""

    def __init__(self, dev, kv_type, H, G, D, page, lens, window=0, seed=1, q_scale=2.0,
                 bad_pages=(), pages_extra=3, first_page=0, scale=None, v_spread=False):
        import torch
        rng = np.random.default_rng(seed)
        self.dev, self.H, self.G, self.D, self.page, self.lens = dev, H, G, D, page, lens
        self.window, self.scale = window, D ** -0.5 if scale is None else scale
        need = [-(-t // page) for _, t in lens]
        pages = first_page + sum(need) + pages_extra
        self.cache = make_cache(rng, dev, kv_type, pages, page, G, D, poison=first_page == 0)
        order = first_page + rng.permutation(pages - first_page)
        self.max_pages = max(need + [1]) + 2
        table = np.full((len(lens), self.max_pages), -1, np.int64)
        T = sum(n for n, _ in lens)
        self.T = T
        q = (q_scale * rng.standard_normal((T, H, D))).astype(np.float32)
        self.want, self.tol, at, row = np.zeros((T, H, D)), 0.0, 0, 0
        for b, ((n, total), np_) in enumerate(zip(lens, need)):
            table[b, :np_] = order[at:at + np_]
            at += np_
            k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
            if v_spread:  # rows of V of very different sizes
                v *= 10.0 ** rng.uniform(-4, 3, (total, 1, 1)).astype(np.float32)
            ok = np.ones(total, bool)
            if total:
                slots = table[b, np.arange(total) // page] * page + np.arange(total) % page
                k, v = put(self.cache, kv_type, page, slots, k, v)
            for bb, j in bad_pages:
                if bb == b and j < np_:
                    table[b, j] = -5 if j % 2 else pages + 3
                    ok[j * page:(j + 1) * page] = False
            pos = total - n + np.arange(n)
            if n:
                o, tol = attention_host(q[row:row + n], k, v, pos, window, self.scale, ok)
                self.want[row:row + n] = o
                self.tol = max(self.tol, tol)
            row += n
        self.q = to_dev(q.reshape(T, H * D), dev)
        self.table = i32(table, dev)
        self.kv_lens = i32([t for _, t in lens], dev)
        self.cu = i32(prefix([n for n, _ in lens]), dev)

    def run(self, out=None, q=None, stream=None):
        out = empty_f32((self.T, self.H * self.D), self.dev) if out is None else out
        capi.paged_attention(self.cache, self.q if q is None else q, out, self.H, self.scale,
                             self.window, self.table, self.max_pages, self.kv_lens, self.cu,
                             len(self.lens), self.T, stream=stream)
        return out

    def check(self, out):
        import torch
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(self.want.shape).astype(np.float64)
        assert np.isfinite(got).all()
        err = np.abs(got - self.want).max()
        assert err <= self.tol, (err, self.tol)


LAYOUTS = [(14, 2, 64), (4, 4, 128), (8, 2, 128), (8, 4, 96), (8, 1, 256), (6, 6, 64),
           (7, 1, 128), (64, 1, 64), (3, 3, 96)]


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D", LAYOUTS)
@pytest.mark.parametrize("lens,page,window", [
    ([(1, 1)], 16, 0), ([(1, 129), (1, 1), (1, 16), (1, 700)], 16, 0),
    ([(1, 333), (70, 70), (0, 50), (1, 64), (17, 190)], 32, 0),
    ([(130, 300), (1, 17), (1, 1000)], 48, 100)])
def test_attention(dev, kv_type, H, G, D, lens, page, window):
    note(f"attention {kv_type} H={H} G={G} D={D} lens={lens} page={page} window={window}")
    b = Batch(dev, kv_type, H, G, D, page, lens, window, seed=D + H)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens,page,window", [
    ([(1, 9000)], 64, 0), ([(1, 5000), (3, 2100), (2, 33)], 128, 0), ([(257, 1500)], 16, 1),
    ([(40, 40)] * 5, 16, 7), ([(1, 4095), (300, 2049)], 1024, 1024), ([(64, 64)], 16, 0)])
def test_attention_lengths(dev, kv_type, lens, page, window):
    note(f"attention lengths {kv_type} lens={lens} page={page} window={window}")
    b = Batch(dev, kv_type, 8, 2, 64, page, lens, window, seed=sum(t for _, t in lens))
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D", [(2, 2, 64), (2, 1, 96), (3, 1, 128), (5, 1, 64), (8, 1, 256),
                                   (1, 1, 256), (16, 1, 128), (24, 1, 96), (7, 1, 96)])
@pytest.mark.parametrize("new,total,window", [(1, 6000, 0), (2, 5000, 0), (1, 7000, 3000)])
def test_attention_of_few_rows_in_many_parts(dev, kv_type, H, G, D, new, total, window):
    """One sequence: its keys go to as many workgroups as they are worth, then are joined."""
    note(f"attention in parts {kv_type} H={H} G={G} D={D} {new} of {total} window={window}")
    b = Batch(dev, kv_type, H, G, D, 32, [(new, total)], window, seed=total + D)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_many_sequences(dev, kv_type):
    """More sequences than a workgroup has threads, most of them short, some without rows."""
    rng = np.random.default_rng(9)
    lens = [(int(rng.integers(0, 3)), int(rng.integers(2, 60))) for _ in range(700)]
    lens[30], lens[650] = (50, 90), (1, 1500)
    note(f"attention many sequences {kv_type}")
    b = Batch(dev, kv_type, 4, 2, 64, 16, lens)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_bad_pages_hide_their_keys(dev, kv_type):
    lens = [(1, 300), (40, 200), (1, 40), (5, 90)]
    bad = [(0, 0), (0, 7), (1, 3), (1, 12), (2, 0), (2, 1), (2, 2), (3, 5)]
    for window in (0, 30):
        note(f"attention bad pages {kv_type} window={window}")
        b = Batch(dev, kv_type, 8, 2, 128, 16, lens, window, bad_pages=bad)
        b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_rows_without_keys(dev, kv_type):
    """Rows before the first token (kv_lens below the new rows: refused requests) are zero,
    rows outside every sequence are not written."""
    import torch
    b = Batch(dev, kv_type, 4, 2, 64, 16, [(1, 20), (30, 40), (2, 50), (20, 33)])
    b.kv_lens = i32([20, 0, 50, 5], dev)
    note(f"attention rows without keys {kv_type}")
    out = empty_f32((b.T + 4, b.H * b.D), dev)
    capi.paged_attention(b.cache, torch.cat([b.q, b.q[:4]]), out, 4, b.scale, 0, b.table,
                         b.max_pages, b.kv_lens, b.cu, 4, b.T + 4)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(-1, 4, 64)
    assert np.isnan(got[b.T:]).all()
    assert (got[1:31] == 0).all() and (got[33:48] == 0).all()
    for rows in (slice(0, 1), slice(31, 33)):
        assert np.abs(got[rows] - b.want[rows]).max() <= b.tol
    assert np.isfinite(got[48:53]).all() and (got[48:53] != 0).any()


@pytest.mark.parametrize("kv_type", ("f16", "bf16"))
@pytest.mark.parametrize("H,G,n", [(4, 2, 5), (4, 2, 60), (4, 1, 140)])
def test_attention_non_finite_values(dev, kv_type, H, G, n):
    """A later token's NaN or infinite K or V reaches the rows that see it and no other."""
    import torch
    D, page, total = 64, 16, n + 45
    for what, value in (("k", float("nan")), ("v", float("nan")), ("v", float("inf")),
                        ("v", float("-inf"))):
        note(f"attention non-finite {kv_type} {what}={value} n={n}")
        b = Batch(dev, kv_type, H, G, D, page, [(n, total)], seed=n)
        at = total - n + n // 2           # seen by the second half of the rows
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
        first, mine = n // 2, slice(0, H // G)
        assert np.abs(got[:first] - b.want[:first]).max() <= b.tol
        if G > 1:
            assert np.abs(got[:, H // G:] - b.want[:, H // G:]).max() <= b.tol
        if what == "k":
            assert np.isnan(got[first:, mine]).all()
        else:
            hit = got[first:, mine, 29]
            assert (np.isnan(hit) if math.isnan(value) else hit == value).all()
            other = np.arange(D) != 29
            assert np.abs(got[first:, mine][..., other]
                          - b.want[first:, mine][..., other]).max() <= b.tol


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens", [[(1, 300), (3, 70)], [(90, 300)]])
def test_attention_scales_and_magnitudes(dev, kv_type, lens):
    """Scales of zero, below zero and large; q of very small and very large values; V rows of
    sizes from 1e-4 to 1e3."""
    for scale, q_scale, spread in ((0.0, 1.0, False), (-0.2, 1.0, False), (4.0, 1.0, False),
                                   (0.125, 1e-30, False), (1e-6, 3e5, True),
                                   (0.125, 2.0, True)):
        note(f"attention magnitudes {kv_type} scale={scale} q={q_scale} lens={lens}")
        b = Batch(dev, kv_type, 4, 2, 64, 16, lens, scale=scale, q_scale=q_scale,
                  v_spread=spread)
        b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens", [[(1, 40), (2, 300)], [(50, 200)]])
def test_attention_non_finite_q(dev, kv_type, lens):
    """A row with NaN in q is NaN in that head and leaves the others as they are."""
    import torch
    b = Batch(dev, kv_type, 4, 2, 64, 16, lens)
    note(f"attention NaN in q {kv_type}")
    row, h = b.T - 2, 1
    b.q.view(b.T, 4, 64)[row, h, 7] = float("nan")
    out = b.run()
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(b.T, 4, 64)
    assert np.isnan(got[row, h]).all()
    got[row, h] = b.want[row, h]
    assert np.abs(got - b.want).max() <= b.tol


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_strides_streams_and_repeats(dev, kv_type):
    """Strided rows, out over q, another stream, and the same bits on every run."""
    import torch
    b = Batch(dev, kv_type, 8, 2, 64, 32, [(1, 3000), (40, 700), (2, 90)])
    note(f"attention strides {kv_type}")
    first = b.run()
    b.check(first)
    wide_q = torch.zeros(b.T, 8 * 64 + 20, device=dev)
    wide_q[:, :512] = b.q
    wide_out = empty_f32((b.T, 8 * 64 + 4), dev)
    b.run(out=wide_out[:, :512], q=wide_q[:, :512])
    torch.cuda.synchronize()
    assert torch.equal(wide_out[:, :512], first) and torch.isnan(wide_out[:, 512:]).all()
    same = b.q.clone()
    b.run(out=same, q=same)
    torch.cuda.synchronize()
    assert torch.equal(same, first)
    stream = torch.cuda.Stream()
    for _ in range(5):
        other = empty_f32(first.shape, dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            b.run(out=other)
        stream.synchronize()
        assert torch.equal(other, first)


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_graph_replays(dev, kv_type):
    """A captured call follows the lengths on the device; eager calls run between replays."""
    import torch
    b = Batch(dev, kv_type, 8, 2, 64, 32, [(1, 3000), (40, 700), (2, 90)])
    c = Batch(dev, kv_type, 8, 2, 64, 32, [(1, 2000), (40, 300), (2, 70)], seed=2)
    eager = [x.run() for x in (b, c)]
    stream = torch.cuda.Stream()
    capi.workspace_reserve(*capi.paged_attention_workspace_size(b.cache, 8, 3, b.T),
                           stream=stream)
    torch.cuda.synchronize()
    note(f"attention captured {kv_type}")
    names = ("q", "table", "kv_lens")
    held = {n: getattr(b, n).clone() for n in names}
    out = empty_f32(eager[0].shape, dev)
    cache_c = [c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        capi.paged_attention(b.cache, held["q"], out, 8, b.scale, 0, held["table"], b.max_pages,
                             held["kv_lens"], b.cu, 3, b.T, stream=stream)
    for rep in range(4):
        if rep == 2:  # the same graph on other lengths and pages
            table = torch.full_like(held["table"], -1)
            table[:, :c.max_pages] = c.table
            held["table"].copy_(table)
            held["q"].copy_(c.q), held["kv_lens"].copy_(c.kv_lens)
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


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_capture_without_reservation_is_refused(dev):
    """Attention, and a plan of many rows, that would allocate their workspace in a capture."""
    import torch
    b = Batch(dev, "f16", 4, 2, 64, 16, [(1, 40)])
    out = empty_f32(b.q.shape, dev)
    words = [torch.zeros(5000, dtype=torch.int32, device=dev) for _ in range(11)]
    torch.cuda.synchronize()
    for call in (lambda s: b.run(out=out, stream=s),
                 lambda s: capi.paged_plan(*words[:2], 2, words[2], 4, 16, 8, *words[3:6], 5000,
                                           *words[6:11], stream=s)):
        stream = torch.cuda.Stream()
        with pytest.raises(capi.Q8_0Error) as err:
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                call(stream)
        assert "reserve it before capture" in str(err.value)
        assert capi.workspace_info(stream)[2] == 0


@pytest.mark.parametrize("kv_type", TYPES)
def test_attention_far_pages(dev, kv_type):
    """Pages whose elements lie past 2^31 of the cache's buffers."""
    G, D, page = 2, 64, 256
    first = 2 ** 31 // (G * page * D) + 5
    note(f"attention far pages {kv_type}")
    b = Batch(dev, kv_type, 4, G, D, page, [(1, 900), (30, 600)], first_page=first)
    b.check(b.run())


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D,lens,window", [
    (8, 2, 128, [(1, 700), (1, 64)], 0), (14, 2, 64, [(60, 400), (20, 20)], 100),
    (4, 4, 96, [(130, 130)], 0), (8, 1, 256, [(40, 300), (1, 50)], 0)])
def test_attention_relative_error(dev, kv_type, H, G, D, lens, window):
    """The whole output within 2^-16 relative L2: a lost part of q (2^-12 of it in f16, 2^-17
    in bf16 with two of three) or of the weights, or a value rounded to 16 bits anywhere, is
    above or at that, while rounding errors of logits below 32 (2^-24 each, a few hundred of
    them at random) are near 2^-19."""
    import torch
    note(f"attention relative error {kv_type} H={H} G={G} D={D} lens={lens}")
    b = Batch(dev, kv_type, H, G, D, 32, lens, window, seed=D)
    out = b.run()
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(b.want.shape).astype(np.float64)
    assert np.linalg.norm(got - b.want) <= 2.0 ** -16 * np.linalg.norm(b.want)


@pytest.mark.parametrize("n,total", [(1, 90), (3, 90), (60, 200)])
@pytest.mark.parametrize("which,value", [("k", float("nan")), ("v", float("nan")),
                                         ("v", float("inf"))])
def test_attention_non_finite_scales(dev, n, total, which, value):
    """An 8-bit row whose scale is not finite makes NaN of the rows that see it, no others."""
    import torch
    H, G, D, page = 4, 2, 64, 16
    note(f"attention scale {which}={value} n={n}")
    b = Batch(dev, "int8", H, G, D, page, [(n, total)], seed=n)
    at = total - n + n // 2
    slot = int(b.table[0, at // page]) * page + at % page
    scales = b.cache.k_scale if which == "k" else b.cache.v_scale
    scales.view(-1, G, page)[slot // page, 1, slot % page] = value
    if value == float("inf"):  # what a row with an infinity stores
        r, tile = slot % 16, slot % page // 16
        b.cache.v.view(-1, G, page // 16, 2, D, 2, 4)[slot // page, 1, tile, r // 4 % 2, :,
                                                      r // 8, r % 4] = 0
    out = b.run()
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(n, H, D)
    first, hit = n // 2, slice(H // G, H)
    assert np.isnan(got[first:, hit]).all()
    got[first:, hit] = b.want[first:, hit]
    assert np.abs(got - b.want).max() <= b.tol


# ---- the step as a whole ----

@pytest.mark.parametrize("kv_type", TYPES)
def test_steps_together(dev, kv_type):
    """Plan, write and attention over several steps: prompts, a chunk, decoding, a finished
    request whose pages the next one takes."""
    import torch
    H, G, D, page, pages, B = 4, 2, 64, 16, 24, 3
    note(f"steps {kv_type}")
    rng = np.random.default_rng(8)
    cache = make_cache(rng, dev, kv_type, pages, page, G, D)
    table = i32(np.full((B, 10), -1), dev)
    stack, count = i32(rng.permutation(pages), dev), i32([pages], dev)
    rope = empty_f32((200, D // 2, 2), dev)
    capi.rope_table(rope, 200, D)
    torch.cuda.synchronize()
    host_rope = rope.cpu().numpy()
    history = [[np.zeros((0, G, D))] * 2 for _ in range(B)]
    lens = np.zeros(B, int)
    for news in ([40, 17, 0], [1, 30, 60], [1, 1, 1], [-1, 1, 1], [90, 1, 1], [1, 1, 1]):
        T = sum(max(n, 0) for n in news)
        kv, cu, pos, slots, granted = (torch.zeros(n, dtype=torch.int32, device=dev)
                                       for n in (B, B + 1, T, T, B))
        capi.paged_plan(i32(lens, dev), i32(news, dev), B, table, 10, page, pages, stack,
                        count, count, T, kv, cu, pos, slots, granted)
        qkv = rng.standard_normal((T, H + 2 * G, D)).astype(np.float32)
        d = to_dev(qkv.reshape(T, -1), dev)
        q, k, v = d.split([H * D, G * D, G * D], dim=1)
        q_out, out = empty_f32((T, H * D), dev), empty_f32((T, H * D), dev)
        capi.paged_kv_write(cache, q, q_out, H, k, v, rope, 200, D, "halves", pos, slots, T)
        capi.paged_attention(cache, q_out, out, H, D ** -0.5, 0, table, 10, kv, cu, B, T)
        torch.cuda.synchronize()
        assert granted.cpu().tolist() == [1] * B
        got, row = out.cpu().numpy().reshape(T, H, D), 0
        for b, n in enumerate(news):
            if n < 0:
                history[b], lens[b] = [np.zeros((0, G, D))] * 2, 0
                continue
            p = lens[b] + np.arange(n)
            mine = qkv[row:row + n]
            new = [rotate_host(mine[:, H:H + G], host_rope, p, D, "halves"), mine[:, H + G:]]
            for i, x in enumerate(new):
                c, s = stored_host(x, kv_type)
                c = c.double().numpy() * (1.0 if s is None else s.double().numpy()[..., None])
                history[b][i] = np.concatenate([history[b][i], c])
            lens[b] += n
            if n:
                want, tol = attention_host(rotate_host(mine[:, :H], host_rope, p, D, "halves"),
                                           *history[b], p, 0, D ** -0.5)
                assert np.abs(got[row:row + n] - want).max() <= tol
            row += n
    assert count.item() == pages - sum(-(-int(n) // page) for n in lens)


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D,prompts", [(8, 4, 96, 40), (8, 4, 128, 40), (8, 4, 256, 0),
                                           (8, 4, 256, 30), (4, 4, 256, 90), (40, 2, 256, 20)])
def test_attention_many_segments_of_a_workgroup(dev, kv_type, H, G, D, prompts):
    """More tiles than workgroups at every head size, so that each goes through several of few
    rows, of many, and of both in turn, with what one keeps for the next."""
    rng = np.random.default_rng(D + prompts)
    n = 700 if D < 256 else 400
    lens = [(int(rng.integers(0, 3)), int(rng.integers(2, 90))) for _ in range(n)]
    for b in rng.choice(n, prompts, replace=False):
        new = int(rng.integers(10, 70))
        lens[b] = (new, new + int(rng.integers(0, 60)))
    lens[5], lens[n - 2] = (1, 1500), (90, 700)
    note(f"attention many segments {kv_type} H={H} G={G} D={D} prompts={prompts}")
    b = Batch(dev, kv_type, H, G, D, 16, lens)
    out = b.run()
    b.check(out)
    got = out.cpu().numpy().reshape(b.want.shape).astype(np.float64)
    assert np.linalg.norm(got - b.want) <= 2.0 ** -16 * np.linalg.norm(b.want)


@pytest.mark.parametrize("kv_type", ("f16", "bf16"))
@pytest.mark.parametrize("H,G,D,new,total,window", [
    (4, 2, 64, 1, 70, 0), (4, 2, 128, 3, 300, 0), (3, 1, 256, 5, 90, 40), (2, 2, 96, 2, 5000, 0),
    (4, 2, 64, 60, 200, 0), (4, 1, 128, 70, 300, 90), (2, 1, 96, 40, 130, 0),
    (2, 1, 256, 40, 130, 0)])
@pytest.mark.parametrize("scale", [0.1, -0.1])
def test_attention_infinities_in_k(dev, kv_type, H, G, D, new, total, window, scale):
    """An infinity in K makes a logit infinite: minus infinity gives its key the weight 0, plus
    infinity makes NaN of the rows that see it, and the other heads and rows stay."""
    import torch
    page = 16
    rng = np.random.default_rng(new + D)
    q = (2 * rng.standard_normal((new, H, D))).astype(np.float32)
    k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
    pos = total - new + np.arange(new)
    _, tol = attention_host(q, *(x.astype(np.float64) for x in (k, v)), pos, window, scale)
    finite_k = k.copy()
    for at in rng.choice(total, 1 + total // 40, replace=False):
        k[at, rng.integers(G), rng.integers(D)] = rng.choice([-np.inf, np.inf])
    at = total - new + new // 2    # among the keys that some of the rows do not see
    k[at, 0, 7], k[at, 0, D - 1] = np.inf, -np.inf
    for case in ("many", "one"):
        note(f"attention infinities in K {kv_type} {case} D={D} {new} of {total} scale={scale}")
        if case == "one":
            k = finite_k.copy()
            k[total - new, 0, 11] = np.inf
        pages = -(-total // page)
        slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
        cache = make_cache(rng, dev, kv_type, pages, page, G, D)
        held = put(cache, kv_type, page, slots, k, v)
        out = empty_f32((new, H * D), dev)
        capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, scale, window,
                             i32(slots[::page] // page, dev), pages, i32([total], dev),
                             i32([0, new], dev), 1, new)
        torch.cuda.synchronize()
        with np.errstate(invalid="ignore"):
            want = infinite_host(q, *held, pos, window, scale)
        got = out.cpu().numpy().reshape(want.shape).astype(np.float64)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        ok = ~np.isnan(want)
        assert np.abs(got[ok] - want[ok]).max(initial=0) <= tol


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("lens", [[(1, 3000)] * 8, [(500, 3000)]])
def test_attention_of_non_finite_q_takes_no_longer(dev, kv_type, lens):
    """Rows whose q is not finite are NaN after one pass over the keys: twice the time of finite
    ones is well above what they take, a pass more with products one by one far above that."""
    import torch
    note(f"attention time of NaN in q {kv_type} {lens}")
    b = Batch(dev, kv_type, 8, 2, 128, 32, lens)
    bad = b.q.clone()
    bad.view(b.T, 8, 128)[::3, ::2, 5] = float("nan")
    out = [empty_f32(b.q.shape, dev) for _ in range(2)]
    assert slower_by(lambda: b.run(out=out[0], q=bad), lambda: b.run(out=out[1])) <= 2
    got = torch.isnan(out[0].view(b.T, 8, 128))
    assert got[::3, ::2].all() and not got[1::3].any() and not got[:, 1::2].any()


def infinite_host(q, k, v, pos, window, scale):
    """Attention in 64 bits with infinities in K; a row whose weights are all 0 is zero."""
    H, R, out = q.shape[1], q.shape[1] // k.shape[1], []
    j = np.arange(len(k))
    seen = (j <= pos[:, None]) & ((j > pos[:, None] - window) if window else True)
    for h in range(H):
        s = np.where(seen, scale * (q[:, h].astype(np.float64) @ k[:, h // R].T), -np.inf)
        top = s.max(-1, keepdims=True)
        e = np.exp(s - np.where(top == -np.inf, 0, top))
        z = e.sum(-1, keepdims=True)
        out.append(e @ v[:, h // R] / np.where(z == 0, 1, z))
    return np.stack(out, 1)


def check_rows_of_any_logits(got, q, k, v, pos, window, scale):
    """Rows against 64 bits whatever their logits' size.  A logit is off by less than ds (see the
    module's head), so weights by factors of up to e^ds and a row by expm1(2 ds) of the largest
    value.  Where that is not small, rows whose two largest logits differ by more than the
    errors and 30 have the value of one key (the others' weights are below e^-30 each), and
    rows of which that cannot be said are passed over.  Returns the number of rows compared."""
    n, H, D = q.shape
    R, j, compared = H // k.shape[1], np.arange(len(k)), 0
    want, _ = attention_host(q, k, v, pos, window, scale)
    seen = (j <= pos[:, None]) & ((j > pos[:, None] - window) if window else True)
    assert np.isfinite(got).all()
    for h in range(H):
        kk, most = k[:, h // R], np.abs(v[:, h // R]).max()
        s = np.where(seen, scale * (q[:, h].astype(np.float64) @ kk.T), -np.inf)
        ds = (D + 16) * 2.0 ** -22 * abs(scale) * (np.abs(q[:, h]).astype(np.float64)
                                                   @ np.abs(kk).T).max(-1)
        top = np.sort(s, -1)[:, -2:]
        for i in range(n):
            tol = most * (np.expm1(2 * min(ds[i], 1)) + 2.0 ** -19
                          + (len(k) / 8 + 64) * 2.0 ** -23)
            if ds[i] > 2.0 ** -3:
                if top[i, 1] - top[i, 0] <= 2 * ds[i] + 30:
                    continue
                tol = most * 2.0 ** -20
            compared += 1
            assert np.abs(got[i, h] - want[i, h]).max() <= tol, (i, h)
    return compared


@pytest.mark.parametrize("kv_type", TYPES)
@pytest.mark.parametrize("H,G,D,new,total,window", [
    (4, 2, 64, 1, 300, 0), (4, 2, 128, 3, 90, 40), (2, 2, 256, 1, 6000, 0), (4, 2, 96, 60, 200, 0),
    (4, 1, 128, 70, 300, 0), (2, 1, 256, 40, 130, 0)])
@pytest.mark.parametrize("scale,size", [(0.11, 1e6), (-0.11, 1e9), (0.11, 1e10), (0.11, 1e15),
                                        (0.11, 1e30), (5e30, 1.0), (0.0, 1e30), (1e-37, 1e37),
                                        (1e-30, 1e-30)])
def test_attention_logits_of_any_size(dev, kv_type, H, G, D, new, total, window, scale, size):
    """Logits from 0 to 1e33: the largest one's weight is 1 however many bits it has."""
    import torch
    note(f"attention logits {kv_type} D={D} {new} of {total} scale={scale} q={size}")
    rng = np.random.default_rng(new + D)
    page, pages = 16, -(-total // 16)
    q = (size * rng.uniform(0.5, 2, (new, H, D)) * rng.choice([-1, 1], (new, H, D))
         ).astype(np.float32)
    k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
    slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
    cache = make_cache(rng, dev, kv_type, pages, page, G, D)
    held = put(cache, kv_type, page, slots, k, v)
    out = empty_f32((new, H * D), dev)
    capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, scale, window,
                         i32(slots[::page] // page, dev), pages, i32([total], dev),
                         i32([0, new], dev), 1, new)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(new, H, D).astype(np.float64)
    compared = check_rows_of_any_logits(got, q, *held, total - new + np.arange(new), window, scale)
    assert compared >= new * H // 2


@pytest.mark.parametrize("D,new,total,window", [(64, 1, 300, 0), (256, 2, 90, 0), (128, 3, 90, 40),
                                                (64, 60, 200, 0), (96, 40, 100, 0),
                                                (128, 50, 90, 0), (256, 40, 100, 30)])
@pytest.mark.parametrize("size,scale", [(-6, 0.11), (-20, 0.11), (-122, 0.11), (-6, 1e-37),
                                        (-20, 1e-30)])
def test_attention_largest_keys(dev, D, new, total, window, size, scale):
    """Keys up to the largest that bf16 holds, with rows of q of 2^size on which all products
    and logits are finite."""
    import torch
    H, G, page = 4, 2, 16
    note(f"attention largest keys D={D} {new} of {total} q=2^{size} scale={scale}")
    rng = np.random.default_rng(new + D)
    q = (2.0 ** size * rng.uniform(0.5, 2, (new, H, D)) * rng.choice([-1, 1], (new, H, D))
         ).astype(np.float32)
    k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
    k *= np.float32(2.0 ** 125)
    k[::7] = np.sign(k[::7]) * np.float32(torch.finfo(torch.bfloat16).max)
    k[3::7] *= np.float32(2.0 ** -120)
    pages = -(-total // page)
    slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
    cache = make_cache(rng, dev, "bf16", pages, page, G, D)
    held = put(cache, "bf16", page, slots, k, v)
    out = empty_f32((new, H * D), dev)
    capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, scale, window,
                         i32(slots[::page] // page, dev), pages, i32([total], dev),
                         i32([0, new], dev), 1, new)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(new, H, D).astype(np.float64)
    compared = check_rows_of_any_logits(got, q, *held, total - new + np.arange(new), window, scale)
    assert compared >= new * H // 2


@pytest.mark.parametrize("D,new,total,window", [(64, 1, 1, 0), (64, 1, 200, 0), (256, 2, 90, 0),
                                                (128, 3, 90, 40), (64, 60, 200, 0), (96, 40, 100, 1),
                                                (128, 50, 190, 0), (256, 40, 100, 30)])
@pytest.mark.parametrize("q_scale", [0.0, 2.0])
def test_attention_largest_values(dev, D, new, total, window, q_scale):
    """V as large as bf16 holds, of one sign in a dimension: the mean stays finite, over keys
    of one weight and of different ones."""
    import torch
    H, G, page = 4, 2, 16
    note(f"attention largest values D={D} {new} of {total} q={q_scale}")
    rng = np.random.default_rng(new + D)
    q = (q_scale * rng.standard_normal((new, H, D))).astype(np.float32)
    k = rng.standard_normal((total, G, D)).astype(np.float32)
    v = rng.uniform(0.9, 0.999, (total, G, D)) * rng.choice([-1, 1], (G, D))
    v = (v * torch.finfo(torch.bfloat16).max).astype(np.float32)
    pages = -(-total // page)
    slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
    cache = make_cache(rng, dev, "bf16", pages, page, G, D)
    held = put(cache, "bf16", page, slots, k, v)
    out = empty_f32((new, H * D), dev)
    capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, D ** -0.5, window,
                         i32(slots[::page] // page, dev), pages, i32([total], dev),
                         i32([0, new], dev), 1, new)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(new, H, D).astype(np.float64)
    want, tol = attention_host(q, *held, total - new + np.arange(new), window, D ** -0.5)
    assert np.isfinite(got).all() and np.abs(got - want).max() <= tol


@pytest.mark.parametrize("new,total", [(1, 500), (3, 300), (40, 400)])
@pytest.mark.parametrize("size", [1e-17, 1e-6, 1.0, 1e4, 1e7, 1e10, 1e13])
def test_attention_zero_value_rows(dev, new, total, size):
    """8-bit V rows of zeros have their weights beside rows of any size (within 2^-16 as in
    test_attention_relative_error)."""
    import torch
    H, G, D, page = 4, 2, 64, 16
    note(f"attention zero V rows {new} of {total} beside {size}")
    rng = np.random.default_rng(total)
    q = (2 * rng.standard_normal((new, H, D))).astype(np.float32)
    k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
    v *= np.float32(size)
    v[rng.random(total) < 0.7] = 0
    pages = -(-total // page)
    slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
    cache = make_cache(rng, dev, "int8", pages, page, G, D)
    held = put(cache, "int8", page, slots, k, v)
    out = empty_f32((new, H * D), dev)
    capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, D ** -0.5, 0,
                         i32(slots[::page] // page, dev), pages, i32([total], dev),
                         i32([0, new], dev), 1, new)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(new, H, D).astype(np.float64)
    want, _ = attention_host(q, *held, total - new + np.arange(new), 0, D ** -0.5)
    assert np.linalg.norm(got - want) <= 2.0 ** -16 * np.linalg.norm(want)


@pytest.mark.parametrize("kv_type", ("bf16", "int8"))
@pytest.mark.parametrize("new,total", [(1, 70), (3, 300), (40, 200)])
@pytest.mark.parametrize("low,high", [(1e-30, 1e-30), (1e-19, 1e-16), (3e-17, 3e-17),
                                      (1e-33, 1e-10), (1e-33, 1.0)])
def test_tiny_values(dev, kv_type, new, total, low, high):
    """V rows of any size down to 1e-33, written and attended: what comes out is what the cache
    holds, within 2^-16 of it (see test_attention_relative_error), and 8-bit rows of scales at
    or below 2^-64 are zeros of scale 0."""
    import torch
    note(f"tiny values {kv_type} {new} of {total} from {low} to {high}")
    H, G, D, page = 4, 2, 64, 16
    rng = np.random.default_rng(total)
    q = (2 * rng.standard_normal((new, H, D))).astype(np.float32)
    k, v = (rng.standard_normal((total, G, D)).astype(np.float32) for _ in range(2))
    v *= np.exp(rng.uniform(np.log(low), np.log(high), (total, 1, 1))).astype(np.float32)
    pages = -(-total // page)
    slots = rng.permutation(pages)[np.arange(total) // page] * page + np.arange(total) % page
    cache = capi.PagedCache.allocate(kv_type, pages, page, G, D, dev)
    filler = torch.zeros(total, H * D, device=dev)
    capi.paged_kv_write(cache, filler, filler, H, to_dev(k.reshape(total, -1), dev),
                        to_dev(v.reshape(total, -1), dev), None, 0, D, "none", None,
                        i32(slots, dev), total)
    out = empty_f32((new, H * D), dev)
    capi.paged_attention(cache, to_dev(q.reshape(new, -1), dev), out, H, D ** -0.5, 0,
                         i32(slots[::page] // page, dev), pages, i32([total], dev),
                         i32([0, new], dev), 1, new)
    torch.cuda.synchronize()
    ck, cv, ks, vs = (None if x is None else x.cpu()[slots] for x in
                      cells_of(cache, pages, page, G, D))
    if kv_type == "int8":
        cells, scale = stored_host(v, kv_type)
        zero = scale <= 2.0 ** -64
        assert zero.any() == (low < 1e-18)
        cells[zero], scale[zero] = 0, 0
        assert torch.equal(cv, cells) and torch.equal(vs, scale)
    held = [x.double().numpy() * (1 if s is None else s.double().numpy()[..., None])
            for x, s in ((ck, ks), (cv, vs))]
    want, _ = attention_host(q, *held, total - new + np.arange(new), 0, D ** -0.5)
    got = out.cpu().numpy().reshape(want.shape).astype(np.float64)
    assert np.linalg.norm(got - want) <= 2.0 ** -16 * np.linalg.norm(want)


@pytest.mark.parametrize("kv_type,total", [("f16", 6069), ("bf16", 6069), ("int8", 8352)])
@pytest.mark.parametrize("new", [1, 2])
def test_attention_parts_up_to_the_workspace_end(dev, kv_type, total, new):
    """One or two rows at head size 256 whose work is 256 equal runs, 16 of them a head: the
    last part lies at the end of a workspace of exactly the stated size."""
    import torch
    note(f"attention parts to the workspace's end {kv_type} {new} of {total}")
    b = Batch(dev, kv_type, 16, 16, 256, 32, [(new, total)], seed=new)
    stream = own_stream()
    size = capi.paged_attention_workspace_size(b.cache, 16, 1, new)
    capi.workspace_reserve(*size, stream=stream)
    assert capi.workspace_info(stream)[0] >= size[0]
    out = empty_f32((b.T, b.H * b.D), dev)
    torch.cuda.synchronize()
    b.run(out=out, stream=stream)
    stream.synchronize()
    b.check(out)
    assert torch.equal(b.run(), out)
