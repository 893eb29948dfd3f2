"""The attention block of a decoder layer over a paged KV cache, as a serving loop runs it.

    python examples/paged_attention_layer.py [--steps 8] [--kv int8]

Requests of different lengths are admitted with their prompts, then decode one token a step
together; one finishes half way and gives its pages to another.  Each step makes one plan and,
per layer, five calls: the q/k/v Linear of Q8_0 weights in 16-row tiles, the rotary embedding
with the cache write, the attention, and the output Linear.  Weights are random; there is no
tokenizer, MLP or norm here, and the block's output is the next step's input.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from llmengine_amd import capi  # noqa: E402
from llmengine_amd import synthetic as S  # noqa: E402


class PagePool:
    """The pages that all layers share the numbers of, and what each request holds of them."""

    def __init__(self, requests, max_pages, pages, page_size, device="cuda"):
        self.requests, self.max_pages, self.pages, self.page_size = (requests, max_pages, pages,
                                                                     page_size)
        self.device = device
        self.table = torch.full((requests, max_pages), -1, dtype=torch.int32, device=device)
        self.free = torch.arange(pages, dtype=torch.int32, device=device)
        self.count = torch.tensor([pages], dtype=torch.int32, device=device)
        self.lens = np.zeros(requests, np.int32)  # the scheduler's copy

    def plan(self, new):
        """Pages for new[b] tokens of each request (negative: it is finished)."""
        new = np.asarray(new, np.int32)
        tokens = int(np.maximum(new, 0).sum())
        B, dev = self.requests, self.device
        step = {n: torch.empty(k, dtype=torch.int32, device=dev)
                for n, k in (("kv_lens", B), ("cu", B + 1), ("positions", tokens),
                             ("slots", tokens), ("granted", B))}
        capi.paged_plan(torch.from_numpy(self.lens).to(dev), torch.from_numpy(new).to(dev), B,
                        self.table, self.max_pages, self.page_size, self.pages, self.free,
                        self.count, self.count, tokens, step["kv_lens"], step["cu"],
                        step["positions"], step["slots"], step["granted"])
        step["tokens"], step["new"] = tokens, new
        return step

    def commit(self, step):
        """The scheduler's lengths after a step: a refused request stays as it was."""
        ok = step["granted"].cpu().numpy() != 0
        self.lens = np.where(step["new"] < 0, 0,
                             self.lens + np.where(ok, np.maximum(step["new"], 0), 0)
                             ).astype(np.int32)
        return ok


class AttentionLayer:
    """x -> output Linear (attention (rotary (q/k/v Linear x)))."""

    def __init__(self, pool, hidden, heads, kv_heads, head_dim, kv_type, positions, seed=1,
                 window=0):
        self.pool, self.hidden, self.window = pool, hidden, window
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.q_size, self.kv_size = heads * head_dim, kv_heads * head_dim
        dev = pool.device
        self.raw = [S.q8_0_weight(seed, self.q_size + 2 * self.kv_size, hidden)[0],
                    S.q8_0_weight(seed + 1, hidden, self.q_size)[0]]
        self.qkv, self.out = (self._tiled(w, n, k) for w, n, k in (
            (self.raw[0], self.q_size + 2 * self.kv_size, hidden),
            (self.raw[1], hidden, self.q_size)))
        self.cache = capi.PagedCache.allocate(kv_type, pool.pages, pool.page_size, kv_heads,
                                              head_dim, dev)
        self.rope = torch.empty(positions, head_dim // 2, 2, device=dev)
        capi.rope_table(self.rope, positions, head_dim)

    def _tiled(self, raw, n, k):
        w = torch.empty(capi.tiled_bytes(n, k), dtype=torch.uint8, device=self.pool.device)
        capi.tile(torch.from_numpy(raw).to(self.pool.device), w, n, k)
        torch.cuda.synchronize()  # the raw copy goes out of scope
        return w

    def __call__(self, x, step):
        T, p = step["tokens"], self.pool
        n = self.q_size + 2 * self.kv_size
        qkv = torch.empty(T, n, device=x.device)
        capi.linear_tiled(x, self.qkv, None, qkv, T, n, self.hidden)
        q, k, v = qkv.split([self.q_size, self.kv_size, self.kv_size], dim=1)
        # q is rotated where it lies and attended in place.
        capi.paged_kv_write(self.cache, q, q, self.heads, k, v, self.rope, self.rope.shape[0],
                            self.head_dim, "halves", step["positions"], step["slots"], T)
        capi.paged_attention(self.cache, q, q, self.heads, self.head_dim ** -0.5, self.window,
                             p.table, p.max_pages, step["kv_lens"], step["cu"], p.requests, T)
        rows = q.contiguous()  # the Linear takes dense rows
        y = torch.empty(T, self.hidden, device=x.device)
        capi.linear_tiled(rows, self.out, None, y, T, self.hidden, self.q_size)
        return y


def serve(layer, pool, prompts, steps, finish_at=None, observe=None):
    """Runs prompts [(tokens, hidden) arrays] and then `steps` decoding steps; request 0 ends
    after `finish_at` of them and the last prompt takes its pages.  Returns the last rows."""
    dev, hidden = pool.device, layer.hidden
    later = prompts[-1] if finish_at is not None else None
    first = prompts[:-1] if later is not None else prompts
    new = [len(p) for p in first] + [0] * (pool.requests - len(first))
    x = torch.from_numpy(np.concatenate(first)).to(dev)
    last = None
    for i in range(steps + 1):
        step = pool.plan(new)
        y = layer(x, step) if step["tokens"] else None
        if observe is not None:
            observe(new, x, y, step)
        ok = pool.commit(step)
        if not ok.all():
            raise RuntimeError(f"step {i}: no pages for request {int(np.argmin(ok))}")
        ends = np.cumsum(np.maximum(step["new"], 0)) - 1
        live = [b for b in range(pool.requests) if new[b] > 0]
        last = {b: y[ends[b]] for b in live}
        if finish_at is not None and i == finish_at:
            new = [-1] + [int(b in live) for b in range(1, pool.requests - 1)] + [len(later)]
            rows = [last[b][None] for b in range(1, pool.requests - 1) if new[b]]
            rows.append(torch.from_numpy(later).to(dev))
        else:
            new = [int(b in live) for b in range(pool.requests)]
            rows = [last[b][None] for b in live]
        x = torch.cat(rows).reshape(-1, hidden).contiguous()
    return last


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--kv", choices=sorted(capi.KV_TYPES), default="f16")
    a = ap.parse_args()
    # The sizes of Qwen2.5-0.5B: 14 heads of 64 over 2 KV heads, 896 wide.
    hidden, heads, kv_heads, dim, page = 896, 14, 2, 64, 16
    lengths = [700, 90, 17, 300]
    pool = PagePool(len(lengths), 64, 90, page)
    layer = AttentionLayer(pool, hidden, heads, kv_heads, dim, a.kv, 1024)
    prompts = [S.activations(10 + i, (n, hidden)) for i, n in enumerate(lengths)]
    last = serve(layer, pool, prompts, a.steps, finish_at=a.steps // 2)
    torch.cuda.synchronize()
    print(f"{a.kv}: {a.steps} steps, {int(pool.count.item())} of {pool.pages} pages free, "
          f"tokens held {pool.lens.tolist()}, "
          f"last rows {[round(float(v.norm()), 3) for v in last.values()]}")


if __name__ == "__main__":
    main()
