"""examples/paged_attention_layer.py against the whole block in 64 bits on the host: the
steps of a serving loop through the Q8_0 Linears, the page plan, the rotary cache write and
the attention, with a request that ends and one that takes its pages.

Tolerance: below 64 rows the Linears are within 1e-5 relative L2 of the exact product and the
attention within 2^-16; a f16 cache rounds k and v by 2^-11, a bf16 one by 2^-8 and an 8-bit
one by half a step of 1/127 of the largest of 64 values.  The cached errors reach the output
through logits of a few units, so by a few times their size: 8 times is allowed.
"""
import importlib.util
import os

import numpy as np
import pytest

from helpers import note, rel_l2
from llmengine_amd import synthetic as S

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    path = os.path.join(ROOT, "examples", "paged_attention_layer.py")
    spec = importlib.util.spec_from_file_location("paged_attention_layer", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def dequantized(raw, n, k):
    blocks = raw.reshape(n, k // 32, 34)
    d = blocks[..., :2].copy().view(np.float16).astype(np.float64)
    return (d * blocks[..., 2:].copy().view(np.int8)).reshape(n, k)


@pytest.mark.parametrize("kv_type,rounding", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8),
                                              ("int8", 0.5 / 127 * 2.5)])
@pytest.mark.parametrize("window", [0, 9])
def test_block_against_64_bits(dev, kv_type, rounding, window):
    import torch
    ex = example()
    hidden, H, G, D, page = 256, 4, 2, 64, 16
    lengths = [25, 7, 1, 20]
    pool = ex.PagePool(len(lengths), 4, 8, page, dev)
    layer = ex.AttentionLayer(pool, hidden, H, G, D, kv_type, 64, window=window)
    wqkv = dequantized(layer.raw[0], (H + 2 * G) * D, hidden)
    wout = dequantized(layer.raw[1], hidden, H * D)
    half = D // 2
    history = [[np.zeros((0, G, D))] * 2 for _ in lengths]

    def turned(x, p):
        a = p[:, None, None] * 10000.0 ** (-np.arange(half) / half)
        u, v = x[..., :half], x[..., half:]
        return np.concatenate([u * np.cos(a) - v * np.sin(a), u * np.sin(a) + v * np.cos(a)], -1)

    def check(new, x, y, step):
        torch.cuda.synchronize()
        x, row = x.cpu().numpy().astype(np.float64), 0
        want = np.zeros((len(x), hidden))
        for b, n in enumerate(new):
            if n < 0:
                history[b] = [np.zeros((0, G, D))] * 2
            if n <= 0:
                continue
            qkv = (x[row:row + n] @ wqkv.T).reshape(n, H + 2 * G, D)
            p = len(history[b][0]) + np.arange(n)
            history[b] = [np.concatenate([h, t]) for h, t in zip(
                history[b], (turned(qkv[:, H:H + G], p), qkv[:, H + G:]))]
            q, (k, v) = turned(qkv[:, :H], p), history[b]
            j = np.arange(len(k))
            seen = (j <= p[:, None]) & ((j > p[:, None] - window) if window else True)
            o = np.zeros((n, H, D))
            for h in range(H):
                s = np.where(seen, q[:, h] @ k[:, h // 2].T * D ** -0.5, -np.inf)
                e = np.exp(s - s.max(-1, keepdims=True))
                o[:, h] = e @ v[:, h // 2] / e.sum(-1, keepdims=True)
            want[row:row + n] = o.reshape(n, -1) @ wout.T
            row += n
        err = rel_l2(y.cpu().numpy(), want)
        note(f"block {kv_type} window={window} new={new} rel {err:.2e}")
        assert err <= 2e-5 + 2.0 ** -16 + 8 * rounding

    prompts = [S.activations(30 + i, (n, hidden)) for i, n in enumerate(lengths)]
    last = ex.serve(layer, pool, prompts, 6, finish_at=3, observe=check)
    assert set(last) == {1, 2, 3} and pool.lens.tolist() == [0, 13, 7, 22]
    assert pool.count.item() == 8 - sum(-(-int(n) // page) for n in pool.lens)


def test_example_refuses_when_pages_run_out(dev):
    """A request without pages is refused by the plan, and the loop says so."""
    ex = example()
    pool = ex.PagePool(2, 4, 2, 16, dev)
    layer = ex.AttentionLayer(pool, 256, 4, 2, 64, "f16", 64)
    prompts = [S.activations(40 + i, (n, 256)) for i, n in enumerate((20, 17))]
    with pytest.raises(RuntimeError, match="no pages for request 1"):
        ex.serve(layer, pool, prompts, 2)
