"""GPU numerics of mle_token_logprobs_f32 against log softmax in 64 bits of the scaled logits.

Tolerances.  A term e^(x - m) is 2^((x - m) log2 e): x - m, log2 e and their product are each
rounded once (2^-24 of |x - m| each, times ln 2 or 1), the power itself to 2^-22, so a term is off
by less than (|x - m| + 1) 2^-22 of itself, the largest ones (x = m) by nothing; sums are of 64
bits.  log S is off by less than the p-weighted mean of that over the other terms,
E = 2^-22 sum_(x < m) p (|x - m| + 1), and log p by E and its own rounding, 2^-24.  The entropy
log S - W / S: W's terms have one rounding more (2^-24), W is kept in 24 bits, and an error of the
terms enters with the weight |log p| + 1 at most: 2^-22 sum_(x < m) p (|x - m| + 1) (|log p| + 2)
+ 2^-23 W / S + 2^-24 H.
"""
import numpy as np
import pytest

from helpers import empty_f32, note, own_stream, to_dev
from llmengine_amd import capi
from llmengine_amd import synthetic as S

pytestmark = pytest.mark.gpu


def scaled(x, temperature):
    if temperature > 0 and temperature != 1:
        return (x * (np.float32(1) / np.float32(temperature))).astype(np.float32)
    return x


def host(row, tokens, top_n, temperature):
    """(logprobs, entropy, ids, top logprobs, their tolerances) of one row, 64 bits."""
    n = row.size
    x = scaled(row, temperature).astype(np.float64)
    k = min(top_n, n)
    if np.isnan(x).any() or not np.isfinite(x.max()):
        lp = np.full(n, -np.log(n))
        ids, entropy, tol_p, tol_h = np.arange(k), np.log(n), 0.0, 2.0 ** -24 * np.log(n)
    else:
        low = x - x.max()
        e = np.exp(low)
        s = e.sum()
        lp, p = low - np.log(s), e / s
        w = np.where(p > 0, -lp, 0.0)
        entropy = (p * w).sum()
        d = np.where(p > 0, -low, 0.0)
        rest = np.where(low < 0, p * (d + 1), 0.0)
        tol_p = 2.0 ** -22 * rest.sum()
        tol_h = (2.0 ** -22 * (rest * (w + 2)).sum() + 2.0 ** -23 * (p * d).sum()
                 + 2.0 ** -24 * entropy)
        ids = np.lexsort((np.arange(n), -x))[:k]
    given = np.array([lp[t] if 0 <= t < n else -np.inf for t in tokens])
    return given, entropy, ids, lp[ids], tol_p, tol_h


def run(x, tokens, top_n, temperature, dev, stream=None, entropy=True):
    import torch
    rows, n = x.shape
    k, m = min(top_n, n), 0 if tokens is None else tokens.shape[1]
    out = [empty_f32((rows, m), dev), empty_f32((rows,), dev),
           torch.full((rows, k), -1, dtype=torch.int32, device=dev), empty_f32((rows, k), dev)]
    d = x if isinstance(x, torch.Tensor) else to_dev(x, dev)
    t = None if tokens is None else to_dev(tokens.astype(np.int32), dev)
    torch.cuda.synchronize()
    capi.token_logprobs(d, rows, n, t, m, top_n, out[0] if m else None,
                        out[1] if entropy else None, out[2] if k else None,
                        out[3] if k else None, temperature, stream=stream)
    torch.cuda.synchronize()
    return [o.cpu().numpy() for o in out]


def near(got, want, tol):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    # A distance may be up to twice the largest fp32 number: past that one plus half its last
    # place, 2^128 (1 - 2^-25), fp32's nearest is an infinity.
    want = np.where(want <= -(2.0 ** 128) * (1 - 2.0 ** -25), -np.inf, want)
    same = got == want  # infinities
    with np.errstate(invalid="ignore"):
        close = np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -24 + 2.0 ** -60
    assert (same | close).all(), (got, want, tol)


def check(x, tokens, top_n, temperature, dev, **kw):
    got = run(x, tokens, top_n, temperature, dev, **kw)
    for r in range(x.shape[0]):
        t = [] if tokens is None else tokens[r]
        given, entropy, ids, top, tol_p, tol_h = host(x[r], t, top_n, temperature)
        near(got[0][r], given, tol_p)
        if kw.get("entropy", True):
            near(got[1][r], entropy, tol_h)
        else:
            assert np.isnan(got[1][r])
        assert np.array_equal(got[2][r], ids), r
        near(got[3][r], top, tol_p)
    return got


@pytest.mark.parametrize("rows,n,given,top_n,temperature", [
    (1, 1, 1, 1, 1.0), (1, 7, 3, 5, 1.0), (1, 5, 2, 10, 1.0), (3, 2048, 1, 40, 0.7),
    (2, 2049, 9, 128, 1.0), (1, 151936, 1, 0, 1.0), (4, 151936, 4, 20, 0.8),
    (2, 100000, 0, 1, 0.0), (2, 32000, 300, 0, 1.5), (5, 63, 1, 0, 1.0), (3, 65, 2, 64, 2.5),
    (300, 5003, 2, 5, 1.0), (700, 12001, 1, 0, 0.6), (2, 600000, 1, 9, 1.0),
    (1, 2500000, 2, 2, 1.0), (1, 3000001, 1, 0, 1.0), (520, 40011, 1, 7, 1.0),
    (60, 400001, 2, 33, 1.0), (530, 3333, 1, 50, 1.1), (9, 33000, 0, 128, 1.0),
    (17, 8191, 1, 64, 1.0)])
def test_logprobs(dev, rows, n, given, top_n, temperature):
    note(f"logprobs rows={rows} n={n} given={given} top_n={top_n} t={temperature}")
    rng = np.random.default_rng(n + rows)
    spread = np.float32(10.0) ** rng.uniform(-1, 1.3, (rows, 1)).astype(np.float32)
    x = (S.activations(500 + n, (rows, n)) * spread).astype(np.float32)
    tokens = rng.integers(0, n, (rows, given)) if given else None
    check(x, tokens, top_n, temperature, dev)


@pytest.mark.parametrize("top_n", [0, 6])
def test_logprobs_special_rows(dev, top_n):
    """Ties, masked logits, rows without a distribution, ids outside the vocabulary."""
    n = 10_000
    x = np.full((9, n), -1.0, np.float32)
    x[0, [4000, 17, 9000]] = 3.0
    x[1, :] = -np.inf
    x[1, 1234] = 2.0                                  # one token is certain
    x[2, 7] = np.nan                                  # uniform from here
    x[3, 99] = np.inf
    x[4, :] = -np.inf                                 # to here
    x[5, 1::2] = 0.5
    x[6, :] = np.finfo(np.float32).min                # masked by the lowest value
    x[6, 3::1000] = -2.0
    x[7, :] = np.finfo(np.float32).min                # nothing but that
    x[8, 0], x[8, 1:] = 3e38, -3e38                   # a distance past fp32
    tokens = np.array([[17, 1234, 0, -1, n, 2 ** 31 - 1, -2 ** 31, 9999]] * 9)
    note(f"logprobs special rows top_n={top_n}")
    got = check(x, tokens, top_n, 1.0, dev)
    assert got[0][1, 1] == 0.0 and got[0][1, 0] == -np.inf and got[1][1] == 0.0
    assert (got[0][:, 3:7] == -np.inf).all()
    for r in (2, 3, 4, 7):
        assert abs(got[1][r] - np.log(n)) <= 2.0 ** -23 * np.log(n)


def test_logprobs_of_likely_tokens(dev):
    """log p near 0 to its own precision: the rest of the row adds 1e-3 to 1e-30 to the sum."""
    n = 4096
    x = np.full((30, n), -200.0, np.float32)
    x[:, 77] = 13.75
    for r in range(30):
        x[r, 5 + 100 * r % n] = 13.75 - 7 - 2.1 * r
    tokens = np.full((30, 1), 77)
    note("logprobs near 0")
    got = check(x, tokens, 3, 1.0, dev)
    assert (got[0] < 0).all() or got[0].max() == 0.0
    want = np.array([host(x[r], [77], 1, 1.0)[0][0] for r in range(30)])
    # 1 + (the rest) has 2^-52 as its last place, on either side.
    assert (np.abs(got[0][:, 0] - want) <= 2.0 ** -16 * np.abs(want) + 2.0 ** -52).all()


@pytest.mark.parametrize("kind,n,top_n", [
    ("sorted", 151936, 40), ("sorted", 5000, 128), ("equal", 151936, 128), ("masked", 151936, 40),
    ("masked", 60000, 3), ("steps", 151936, 100), ("zeros", 9000, 128), ("normal", 1_000_000, 31),
    ("normal", 65, 64)])
def test_logprobs_alternatives(dev, kind, n, top_n):
    """Rows that press on the selection: winners in few groups, ties, masked logits, signed
    zeros; the ids are those of mle_top_tokens_f32."""
    import torch
    rows = 2
    rng = np.random.default_rng(n + top_n)
    x = (S.activations(430, (rows, n)) * np.float32(3)).astype(np.float32)
    if kind == "sorted":
        x = np.sort(x, axis=1)
    elif kind == "equal":
        x[:] = 0.5
    elif kind == "masked":
        keep = rng.integers(0, n, size=(rows, 50))
        m = np.full_like(x, np.finfo(np.float32).min)
        np.put_along_axis(m, keep, np.take_along_axis(x, keep, 1), 1)
        x = m
    elif kind == "steps":
        x = np.round(x).astype(np.float32)
    elif kind == "zeros":
        x = np.where(rng.random((rows, n)) < 0.5, np.float32(0.0), np.float32(-0.0))
    note(f"logprobs alternatives {kind} n={n} top_n={top_n}")
    got = check(x, None, top_n, 0.8, dev)
    ids = torch.empty((rows, min(top_n, n)), dtype=torch.int32, device=dev)
    probs = empty_f32((rows, min(top_n, n)), dev)
    capi.top_tokens(to_dev(x, dev), rows, n, top_n, ids, probs, 0.8)
    torch.cuda.synchronize()
    assert np.array_equal(got[2], ids.cpu().numpy())
    np.testing.assert_allclose(np.exp(got[3].astype(np.float64)), probs.cpu().numpy(), rtol=2e-5,
                               atol=1e-37)


def test_logprobs_parts_streams_and_repeats(dev):
    """Parts left out, unaligned rows, another stream; the same bits on every run."""
    import torch
    rows, n = 40, 7001
    rng = np.random.default_rng(2)
    x = (S.activations(77, (rows, n)) * np.float32(4)).astype(np.float32)
    tokens = rng.integers(0, n, (rows, 3))
    note("logprobs parts and streams")
    first = check(x, tokens, 20, 1.0, dev)
    check(x, None, 20, 1.0, dev, entropy=False)
    check(x, tokens, 0, 1.0, dev, entropy=False)
    check(x, None, 0, 1.0, dev)
    wide = torch.full((rows * n + 3,), float("nan"), device=dev)
    for off in (1, 2, 3):
        d = wide[off:off + rows * n].view(rows, n)
        d.copy_(to_dev(x, dev))
        stream = own_stream() if off == 1 else None
        for a, b in zip(run(d, tokens, 20, 1.0, dev, stream=stream), first):
            assert np.array_equal(a, b)


def test_logprobs_graph_replays(dev):
    """A captured call, replayed on new logits, with eager calls between on its stream."""
    import torch
    rows, n, top = 3, 50257, 10
    stream = own_stream()
    capi.workspace_reserve(*capi.token_logprobs_workspace_size(rows, n, top), stream=stream)
    x = torch.zeros(rows, n, device=dev)
    tokens = torch.zeros(rows, 2, dtype=torch.int32, device=dev)
    outs = [[empty_f32((rows, 2), dev), empty_f32((rows,), dev),
             torch.empty(rows, top, dtype=torch.int32, device=dev), empty_f32((rows, top), dev)]
            for _ in range(2)]

    def call(o):
        capi.token_logprobs(x, rows, n, tokens, 2, top, *o, 0.9, stream=stream)
    torch.cuda.synchronize()
    note("logprobs captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call(outs[0])
    for rep in range(4):
        x.copy_(torch.randn(rows, n, device=dev) * (1 + rep))
        tokens.random_(0, n)
        torch.cuda.synchronize()
        graph.replay()
        call(outs[1])
        torch.cuda.synchronize()
        for a, b in zip(*outs):
            assert torch.equal(a, b), rep
