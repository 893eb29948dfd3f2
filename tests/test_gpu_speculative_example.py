"""examples/speculative_decoding.py: what its trees accept is what the model finds most likely
when it reads the same text as a run, and drafts take fewer steps than tokens.

Tolerance: the text read as a run has other sums in its Linears (1e-5 below 64 rows) and cells
that may round to the other side, 2^-11 of f16 values, 2^-8 of bf16 ones, and a step of 1/127 of
the largest of 64 8-bit ones; they reach the logits through logits of a few units, so by a few
times their size: 8 times the rounding, of the largest logit, between the likely token's and
the largest.
"""
import importlib.util
import os

import numpy as np
import pytest

from helpers import note
from llmengine_amd import synthetic as S

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    path = os.path.join(ROOT, "examples", "speculative_decoding.py")
    spec = importlib.util.spec_from_file_location("speculative_decoding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("kv_type,rounding", [("f16", 2.0 ** -11), ("bf16", 2.0 ** -8),
                                              ("int8", 1 / 127)])
def test_accepted_text_is_the_models(dev, kv_type, rounding):
    import torch
    ex = example()
    V, count = 512, 24
    # Texts of few tokens, so that drafts are found.
    prompts = [(S.token_ids(5 + i, n, 6)).tolist() for i, n in enumerate((20, 1, 33))]

    def make(requests):
        pool = ex.PagePool(requests, 8, 24, 16, dev)
        return pool, ex.Model(pool, V, 128, 4, 2, 64, 2, kv_type, 128)

    for width, depth in ((3, 5), (1, 0)):
        pool, model = make(3)
        note(f"speculative example {kv_type} width={width} depth={depth}")
        texts, scores, steps = ex.generate(model, pool, prompts, count, width, depth)
        assert all(len(t) >= len(p) + count and t[:len(p)] == p
                   for t, p in zip(texts, prompts))
        # The prompt's step gives a token too; without drafts every other step one each.
        assert steps == count if depth == 0 else steps <= count
        # All but the last token are cached, in fewest pages.
        assert pool.lens.tolist() == [len(t) - 1 for t in texts]
        assert int(pool.count.item()) == 24 - sum(-(-(len(t) - 1) // 16) for t in texts)
        for p, t in zip(prompts, texts):
            alone, judge = make(1)
            step = alone.plan([len(t) - 1])
            i32 = dict(dtype=torch.int32, device=dev)
            step.update(node_positions=step["positions"], trees=torch.zeros(1, **i32),
                        masks=torch.zeros(len(t), dtype=torch.int64, device=dev))
            logits = judge(torch.tensor(t[:-1], **i32), step).double().cpu().numpy()
            for at in range(len(p) - 1, len(t) - 1):
                gap = logits[at].max() - logits[at][t[at + 1]]
                assert gap <= 8 * rounding * np.abs(logits[at]).max(), (at, gap)
        assert np.isfinite(scores).all() and max(scores) <= 0
