"""Greedy decoding in trees of drafted tokens over a paged KV cache.

    python examples/speculative_decoding.py [--tokens 60] [--kv int8] [--depth 6] [--width 3]

Drafts are what followed earlier occurrences of the last token in the request's own text (up to
`width` of them, `depth` tokens each, merged into a tree below the last token).  A step checks
all requests' trees together: one plan; a layer the q/k/v Linear, the cache write with norms of
q and k and the rotary embedding, the attention of the trees, and the output Linear; then the
most likely token behind each node.  The path that these agree with is accepted: its keys and
values move behind the cached ones in all layers, the other nodes' pages go back.  `--depth 0`
decodes token by token.  Weights are random; there is no tokenizer, MLP or norm of the rows.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from paged_attention_layer import AttentionLayer, PagePool  # noqa: E402
from llmengine_amd import capi  # noqa: E402
from llmengine_amd import synthetic as S  # noqa: E402


class NormedLayer(AttentionLayer):
    """The attention block with norms of q and k, whose new tokens may be trees."""

    def __init__(self, pool, *sizes, seed=1, **kw):
        super().__init__(pool, *sizes, seed=seed, **kw)
        self.norms = [torch.from_numpy(1 + S.activations(seed + 2 + i, (self.head_dim,)) / 8)
                      .to(pool.device) for i in range(2)]

    def __call__(self, x, step):
        T, p = step["tokens"], self.pool
        n = self.q_size + 2 * self.kv_size
        qkv = torch.empty(T, n, device=x.device)
        capi.linear_tiled(x, self.qkv, None, qkv, T, n, self.hidden)
        q, k, v = qkv.split([self.q_size, self.kv_size, self.kv_size], dim=1)
        capi.paged_kv_write_normed(self.cache, q, q, self.heads, k, v, *self.norms, 1e-6,
                                   self.rope, self.rope.shape[0], self.head_dim, "halves",
                                   step["node_positions"], step["slots"], T)
        capi.paged_tree_attention(self.cache, q, q, self.heads, self.head_dim ** -0.5,
                                  self.window, p.table, p.max_pages, step["kv_lens"],
                                  step["cu"], p.requests, T, step["masks"], 1,
                                  step["node_positions"], step["trees"])
        y = torch.empty(T, self.hidden, device=x.device)
        capi.linear_tiled(q.contiguous(), self.out, None, y, T, self.hidden, self.q_size)
        return x + y


class Model:
    """Token ids -> logits, with one table for the embedding and the output."""

    def __init__(self, pool, vocab, hidden, heads, kv_heads, head_dim, layers, kv_type,
                 positions, seed=1):
        self.pool, self.vocab, self.hidden = pool, vocab, hidden
        self.table = torch.from_numpy(S.q8_0_weight(seed, vocab, hidden)[0]).to(pool.device)
        self.layers = [NormedLayer(pool, hidden, heads, kv_heads, head_dim, kv_type, positions,
                                   seed=seed + 10 * (i + 1)) for i in range(layers)]
        self.caches = capi.PagedCaches([layer.cache for layer in self.layers])

    def __call__(self, ids, step):
        T, dev = step["tokens"], self.pool.device
        x = torch.empty(T, self.hidden, device=dev)
        capi.embedding(self.table, ids, x, T, self.vocab, self.hidden)
        for layer in self.layers:
            x = layer(x, step)
        logits = torch.empty(T, self.vocab, device=dev)
        capi.linear(x, self.table, None, logits, T, self.vocab, self.hidden)
        return logits


def draft(text, width, depth):
    """[(token, parent)] of a tree below the last token, its root; parents come first."""
    nodes, children = [(text[-1], -1)], {}
    found = [i for i in range(len(text) - 2, -1, -1) if text[i] == text[-1]][:width]
    for i in found:
        at = 0
        for token in text[i + 1:i + 1 + depth]:
            if (at, token) not in children and len(nodes) < 64:
                children[at, token] = len(nodes)
                nodes.append((token, at))
            if (at, token) not in children:
                break
            at = children[at, token]
    return nodes


def run_step(model, pool, trees):
    """One step over trees[b] = (nodes, whether they are a tree): (the step, the most likely
    token behind each node, its log probability)."""
    step = pool.plan([len(nodes) for nodes, _ in trees])
    T, dev = step["tokens"], pool.device
    ids, depth, masks = np.zeros(T, np.int32), np.zeros(T, np.int32), np.zeros(T, np.int64)
    row = 0
    for nodes, is_tree in trees:
        for i, (token, parent) in enumerate(nodes):
            ids[row + i] = token
            depth[row + i] = depth[row + parent] + 1 if parent >= 0 else 0
            if is_tree:
                above = int(masks[row + parent]) if parent >= 0 else 0
                masks[row + i] = np.uint64((above | 1 << i) & (2 ** 64 - 1)).astype(np.int64)
        row += len(nodes)
    base = np.repeat(pool.lens, [len(nodes) for nodes, _ in trees])
    step["node_positions"] = torch.from_numpy((base + depth).astype(np.int32)).to(dev)
    step["masks"] = torch.from_numpy(masks).to(dev)
    step["trees"] = torch.tensor([int(t) for _, t in trees], dtype=torch.int32, device=dev)
    logits = model(torch.from_numpy(ids).to(dev), step)
    top = torch.empty(T, 1, dtype=torch.int32, device=dev)
    logprob = torch.empty(T, 1, device=dev)
    capi.token_logprobs(logits, T, model.vocab, None, 0, 1, None, None, top, logprob)
    if not bool(step["granted"].all()):
        raise RuntimeError("no pages for a request")
    return step, top[:, 0].tolist(), logprob[:, 0].tolist()


def accept(nodes, likely):
    """The rows of the path from the root that the likely tokens agree with, and the token
    behind its end."""
    path = [0]
    for i, (token, parent) in enumerate(nodes):
        if parent == path[-1] and token == likely[parent]:
            path.append(i)
    return path, likely[path[-1]]


def generate(model, pool, prompts, count, width=3, depth=6):
    """`count` tokens behind each prompt: (texts, their log probabilities, steps)."""
    texts, scores, steps = [list(p) for p in prompts], [0.0] * len(prompts), 0
    goal = [len(t) + count for t in texts]
    trees = [([(t, i - 1) for i, t in enumerate(text)], False) for text in texts]
    while any(nodes for nodes, _ in trees):
        step, likely, logprob = run_step(model, pool, trees)
        keep = np.full((len(texts), 64), -1, np.int32)
        counts = np.full(len(texts), -1, np.int32)
        row = 0
        for b, (nodes, is_tree) in enumerate(trees):
            mine, theirs = likely[row:row + len(nodes)], logprob[row:row + len(nodes)]
            row += len(nodes)
            if not nodes:
                continue
            path, last = accept(nodes, mine) if is_tree else ([len(nodes) - 1], mine[-1])
            if is_tree:
                keep[b, :len(path)], counts[b] = path, len(path)
            texts[b] += [nodes[i][0] for i in path[1:]] + [last]
            scores[b] += sum(theirs[i] for i in path)
        lens = torch.empty(len(texts), dtype=torch.int32, device=pool.device)
        capi.paged_kv_keep(model.caches, pool.table, pool.max_pages, step["kv_lens"],
                           step["cu"], step["granted"], pool.requests,
                           torch.from_numpy(keep).to(pool.device), 64,
                           torch.from_numpy(counts).to(pool.device), lens, pool.free,
                           pool.count, pool.count)
        pool.lens = lens.cpu().numpy()
        trees = [(draft(text, width, depth) if len(text) < end else [], True)
                 for text, end in zip(texts, goal)]
        steps += 1
    return texts, scores, steps


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--tokens", type=int, default=60)
    ap.add_argument("--kv", choices=sorted(capi.KV_TYPES), default="f16")
    ap.add_argument("--width", type=int, default=3)
    ap.add_argument("--depth", type=int, default=6)
    a = ap.parse_args()
    pool = PagePool(3, 32, 96, 16)
    model = Model(pool, 2048, 256, 4, 2, 64, 2, a.kv, 512)
    prompts = [S.token_ids(5 + i, n, 2048).tolist() for i, n in enumerate((20, 7, 33))]
    texts, scores, steps = generate(model, pool, prompts, a.tokens, a.width, a.depth)
    made = [len(t) - len(p) for t, p in zip(texts, prompts)]
    print(f"{a.kv}: {made} tokens in {steps} steps, log probabilities "
          f"{[round(s, 2) for s in scores]}, {int(pool.count.item())} of {pool.pages} pages free")


if __name__ == "__main__":
    main()
