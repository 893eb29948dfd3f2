"""Refusals of the calls of speculative decoding (include/mle_paged.h, include/mle_q8_0.h):
every check comes before any HIP call, so none of these needs a GPU."""
import ctypes

import pytest

from llmengine_amd import capi

FAKE = 0x1000   # aligned, never dereferenced
ODD = 0x1002    # misaligned for 4-byte words
INVALID, MISMATCH, UNSUPPORTED = 1, 3, 4


def cache(**kw):
    a = dict(kv_type="f16", num_pages=8, page_size=16, kv_heads=2, head_dim=64, k=FAKE, v=FAKE,
             k_scale=None, v_scale=None)
    a.update(kw)
    return capi.PagedCache(**a)


def write(c=None, **kw):
    a = dict(cache=c or cache(), q=FAKE, q_out=FAKE, heads=4, k=FAKE, v=FAKE, q_norm=FAKE,
             k_norm=FAKE, eps=1e-6, rope=FAKE, rope_positions=10, rope_dim=64,
             rope_mode="halves", positions=FAKE, slots=FAKE, tokens=3, stream=0)
    a.update(kw)
    return capi.paged_kv_write_normed_status(**a)


def attention(c=None, **kw):
    a = dict(cache=c or cache(), q=FAKE, out=FAKE, heads=4, scale=0.125, window=0,
             block_table=FAKE, max_pages=4, kv_lens=FAKE, cu_tokens=FAKE, sequences=2, tokens=3,
             tree_mask=FAKE, mask_words=1, row_positions=FAKE, trees=FAKE, stream=0)
    a.update(kw)
    return capi.paged_tree_attention_status(**a)


def layer(i, **kw):
    return cache(k=(2 * i + 3) * FAKE, v=(2 * i + 4) * FAKE, **kw)


def keep(caches=None, **kw):
    a = dict(caches=capi.PagedCaches(caches if caches is not None else [layer(0), layer(1)]),
             block_table=FAKE, max_pages=4, kv_lens=FAKE, cu_tokens=FAKE, granted=FAKE,
             sequences=2, keep=FAKE, keep_stride=3, keep_counts=FAKE, kept_lens=2 * FAKE,
             free_pages=FAKE, free_count=FAKE, free_count_out=FAKE, stream=0)
    a.update(kw)
    return capi.paged_kv_keep_status(**a)


def logprobs(**kw):
    a = dict(logits=FAKE, rows=2, n=100, tokens=FAKE, tokens_per_row=1, top_n=5, logprobs=FAKE,
             entropy=FAKE, top_ids=FAKE, top_logprobs=FAKE, stream=0)
    a.update(kw)
    return capi.token_logprobs_status(**a)


@pytest.mark.parametrize("bad,code,text", [
    (dict(k=None), INVALID, "cache k pointer"), (dict(kv_type=3), INVALID, "unknown cache type"),
    (dict(head_dim=80), UNSUPPORTED, "head_dim must be"),
    (dict(page_size=24), UNSUPPORTED, "page_size must be"),
    (dict(kv_type="int8"), INVALID, "k_scale pointer"),
    (dict(num_pages=1 << 28), UNSUPPORTED, "31 bits")])
def test_cache_refusals(bad, code, text):
    for call in (write, attention, lambda c: keep([c, c])):
        got, msg = call(cache(**bad))
        assert got == code and text in msg, (got, msg)


def test_null_caches():
    lib = capi.load()
    assert lib.mle_paged_kv_write_normed(None, *[FAKE] * 9, FAKE, FAKE, 1e-6, *[0] * 8) == INVALID
    assert lib.mle_paged_tree_attention(None, *[0] * 5, 1.0, *[0] * 7, FAKE, 1, 0, 0,
                                        0) == INVALID
    assert lib.mle_paged_kv_keep(None, 1, *[FAKE] * 14) == INVALID


@pytest.mark.parametrize("bad,code,text", [
    (dict(q_norm=None), INVALID, "q_norm pointer"), (dict(k_norm=None), INVALID, "k_norm pointer"),
    (dict(q_norm=0x1008), INVALID, "q_norm must be 16-byte"),
    (dict(k_norm=0x1004), INVALID, "k_norm must be 16-byte"),
    (dict(eps=-1e-6), INVALID, "eps"), (dict(eps=float("nan")), INVALID, "eps"),
    (dict(eps=float("inf")), INVALID, "eps"), (dict(q=None), INVALID, "q pointer"),
    (dict(slots=ODD), INVALID, "slots"), (dict(positions=None), INVALID, "positions pointer"),
    (dict(heads=0), INVALID, "heads"), (dict(tokens=-1), INVALID, "tokens"),
    (dict(q_stride=252), INVALID, "q stride"), (dict(v_stride=129), INVALID, "v stride"),
    (dict(rope_dim=72), INVALID, "at most head_dim"), (dict(rope_mode=2), INVALID, "rope_mode"),
    (dict(rope_mode="none"), INVALID, "rope_mode"), (dict(tokens=1 << 28), UNSUPPORTED, "30 bits"),
])
def test_write_refusals(bad, code, text):
    got, msg = write(**bad)
    assert got == code and text in msg and "paged_kv_write_normed" in msg, (got, msg)


@pytest.mark.parametrize("bad,code,text", [
    (dict(tree_mask=None), INVALID, "tree_mask pointer"),
    (dict(tree_mask=0x1004), INVALID, "tree_mask must be 8-byte"),
    (dict(mask_words=0), INVALID, "mask_words"), (dict(mask_words=-3), INVALID, "mask_words"),
    (dict(mask_words=65), UNSUPPORTED, "mask_words"),
    (dict(window=5, row_positions=None), INVALID, "row_positions pointer"),
    (dict(row_positions=ODD), INVALID, "row_positions"), (dict(trees=ODD), INVALID, "trees"),
    (dict(q=None), INVALID, "q pointer"), (dict(kv_lens=None), INVALID, "kv_lens"),
    (dict(heads=5), INVALID, "multiple of kv_heads"), (dict(heads=130), UNSUPPORTED, "at most 64"),
    (dict(sequences=0), INVALID, "sequences"), (dict(window=-1), INVALID, "window"),
    (dict(scale=float("nan")), INVALID, "scale"), (dict(out_stride=257), INVALID, "out stride"),
    (dict(max_pages=1 << 28), UNSUPPORTED, "31 bits"), (dict(tokens=-2), INVALID, "tokens"),
])
def test_attention_refusals(bad, code, text):
    got, msg = attention(**bad)
    assert got == code and text in msg and "paged_tree_attention" in msg, (got, msg)


def test_no_tokens_is_a_no_op():
    assert write(tokens=0)[0] == 0 and attention(tokens=0)[0] == 0
    assert attention(tokens=0, trees=None, row_positions=None)[0] == 0


@pytest.mark.parametrize("name", ["block_table", "kv_lens", "cu_tokens", "granted", "keep",
                                  "keep_counts", "kept_lens", "free_count", "free_count_out"])
def test_keep_pointers(name):
    code, msg = keep(**{name: None})
    assert code == INVALID and name + " pointer" in msg
    code, msg = keep(**{name: ODD})
    assert code == INVALID and name + " must be 4-byte" in msg


@pytest.mark.parametrize("bad,code,text", [
    (dict(free_pages=ODD), INVALID, "free_pages"), (dict(sequences=0), INVALID, "sequences"),
    (dict(max_pages=-1), INVALID, "max_pages"), (dict(keep_stride=0), INVALID, "keep_stride"),
    (dict(kept_lens=FAKE), INVALID, "kept_lens must not overlap kv_lens"),
    (dict(kv_lens=2 * FAKE + 4), INVALID, "kept_lens must not overlap kv_lens"),
    (dict(cu_tokens=2 * FAKE - 8), INVALID, "kept_lens must not overlap cu_tokens"),
    (dict(granted=2 * FAKE), INVALID, "kept_lens must not overlap granted"),
    (dict(keep_counts=2 * FAKE), INVALID, "kept_lens must not overlap keep_counts"),
    (dict(keep=2 * FAKE - 20), INVALID, "kept_lens must not overlap keep"),
    (dict(block_table=2 * FAKE - 28), INVALID, "kept_lens must not overlap block_table"),
    (dict(max_pages=1 << 28), UNSUPPORTED, "31 bits"),
    (dict(sequences=1 << 29), UNSUPPORTED, "31 bits"),
    (dict(sequences=1 << 26, max_pages=1), UNSUPPORTED, "2^32 threads"),
])
def test_keep_refusals(bad, code, text):
    got, msg = keep(**bad)
    assert got == code and text in msg, (got, msg)


# What keep reads and writes, each in a place of its own.
APART = {n: 0x100000 + 0x1000 * i for i, n in enumerate(
    ("kv_lens", "cu_tokens", "granted", "keep_counts", "keep", "block_table", "free_count",
     "kept_lens", "free_pages", "free_count_out"))}


@pytest.mark.parametrize("written,size", [("kept_lens", 8), ("free_pages", 32),
                                          ("free_count_out", 4)])
@pytest.mark.parametrize("other", list(APART))
def test_keep_writes_over_nothing(written, size, other):
    """No array that the call writes may lie over another, in any part of either."""
    if other == written:
        return
    sizes = dict(kv_lens=8, cu_tokens=12, granted=8, keep_counts=8, keep=24, block_table=32,
                 free_count=4, kept_lens=8, free_pages=32, free_count_out=4)
    for off in {0, 4 - size, sizes[other] - 4}:
        if (written, other, off) == ("free_count_out", "free_count", 0):
            continue
        got, msg = keep(**{**APART, written: APART[other] + off})
        assert got == INVALID and written in msg and other in msg, (off, got, msg)
        assert "must not overlap" in msg


def test_keep_count_in_place():
    """The count may take its own place (what is refused then comes later), not another's."""
    same = {**APART, "free_count_out": APART["free_count"]}
    got, msg = keep([layer(0), layer(500)], **{**same, "kept_lens": 3 * FAKE + 8})
    assert got == INVALID and "kept_lens must not overlap cache 0" in msg, (got, msg)
    for other in ("kv_lens", "kept_lens", "free_pages"):
        got, msg = keep(**{**same, other: APART["free_count"]})
        assert got == INVALID and "must not overlap" in msg and "cache" not in msg, (got, msg)


@pytest.mark.parametrize("name", list(APART))
@pytest.mark.parametrize("kv_type", ["f16", "int8"])
def test_keep_arrays_outside_the_caches(name, kv_type):
    """Nor may the caches, which the moves write, lie over an array: their last bytes here."""
    size = dict(f16=2, int8=1)[kv_type] * 8 * 16 * 2 * 64
    at = dict(k=0x400000, v=0x500000)
    if kv_type == "int8":
        at.update(k_scale=0x600000, v_scale=0x700000)
    for part, base in at.items():
        last = base + (8 * 16 * 2 * 4 if "scale" in part else size) - 4
        scales = dict(k_scale=0x800000, v_scale=0x900000) if kv_type == "int8" else {}
        got, msg = keep([layer(500, kv_type=kv_type, **scales), cache(kv_type=kv_type, **at)],
                        **{**APART, name: last})
        assert got == INVALID and name + " must not overlap cache 1" in msg, (part, got, msg)


@pytest.mark.parametrize("other", [dict(num_pages=9), dict(page_size=32), dict(kv_heads=1),
                                   dict(head_dim=128), dict(kv_type="bf16")])
def test_keep_of_unlike_caches(other):
    got, msg = keep([layer(0), layer(1), layer(2, **other)])
    assert got == MISMATCH and "cache 2 differs" in msg, (got, msg)
    got, msg = keep([])
    assert got == INVALID and "layers" in msg


def test_keep_of_a_cache_twice():
    """Two layers of the same memory would move each other's rows."""
    for other in (layer(0), cache(k=99 * FAKE, v=4 * FAKE), cache(k=3 * FAKE, v=99 * FAKE)):
        got, msg = keep([layer(0), layer(1), other])
        assert got == INVALID and "caches 0 and 2 are the same memory" in msg, (got, msg)


def test_keep_of_k_that_is_v():
    """One layer's K that is another's V, or its own, would be moved as both."""
    for caches, which in (
            ([layer(0), layer(1), cache(k=99 * FAKE, v=3 * FAKE)], "0 and 2"),
            ([layer(0), layer(1), cache(k=6 * FAKE, v=99 * FAKE)], "1 and 2"),
            ([layer(0), cache(k=98 * FAKE, v=98 * FAKE)], "1 and 1")):
        got, msg = keep(caches)
        assert got == INVALID and f"caches {which} are the same memory" in msg, (got, msg)
    for scales, which in (((50, 51), "0 and 1"), ((52, 50), "0 and 1"), ((51, 53), "0 and 1"),
                          ((54, 54), "1 and 1")):
        got, msg = keep([layer(0, kv_type="int8", k_scale=50 * FAKE, v_scale=51 * FAKE),
                         layer(1, kv_type="int8", k_scale=scales[0] * FAKE,
                               v_scale=scales[1] * FAKE)])
        assert got == INVALID and f"caches {which} are the same memory" in msg, (got, msg)


@pytest.mark.parametrize("bad,code,text", [
    (dict(logits=None), INVALID, "logits pointer"), (dict(rows=0), INVALID, "rows"),
    (dict(n=0), INVALID, "n must be positive"), (dict(tokens_per_row=-1), INVALID, "tokens_per_row"),
    (dict(top_n=-1), INVALID, "top_n"), (dict(tokens=None), INVALID, "tokens pointer"),
    (dict(logprobs=None), INVALID, "logprobs pointer"), (dict(top_ids=None), INVALID, "top_ids"),
    (dict(top_logprobs=None), INVALID, "top_logprobs"), (dict(rows=70000), UNSUPPORTED, "65535"),
    (dict(top_n=129), UNSUPPORTED, "at most 128"),
    (dict(n=262145, top_n=128), UNSUPPORTED, "at most 262144"),
    (dict(logits=ODD), INVALID, "logits must be"), (dict(tokens=ODD), INVALID, "tokens must be"),
    (dict(entropy=ODD), INVALID, "entropy must be"), (dict(top_ids=ODD), INVALID, "top_ids must"),
    (dict(top_logprobs=ODD), INVALID, "top_logprobs must"),
    (dict(logprobs=ODD), INVALID, "logprobs must be"),
])
def test_logprobs_refusals(bad, code, text):
    got, msg = logprobs(**bad)
    assert got == code and text in msg, (got, msg)


def test_logprobs_of_nothing_is_a_no_op():
    assert logprobs(tokens=None, tokens_per_row=0, logprobs=None, entropy=None, top_n=0,
                    top_ids=None, top_logprobs=None)[0] == 0


def test_logprobs_workspace_size():
    """Grows with the sizes, so that the largest call's holds for smaller ones."""
    last = (0, 0)
    for rows, n, top in ((1, 100, 0), (1, 32000, 0), (130, 32000, 0), (130, 32000, 5),
                         (2048, 32000, 5), (2048, 151936, 128), (65535, 151936, 128)):
        size = capi.token_logprobs_workspace_size(rows, n, top)
        assert size[0] >= last[0] and size[1] >= last[1]
        last = size
    n = ctypes.c_size_t()
    lib = capi.load()
    assert lib.mle_token_logprobs_workspace_size(0, 5, 1, ctypes.byref(n),
                                                 ctypes.byref(n)) == INVALID
    assert lib.mle_token_logprobs_workspace_size(1, 5, 129, ctypes.byref(n),
                                                 ctypes.byref(n)) == UNSUPPORTED
    assert lib.mle_token_logprobs_workspace_size(1, 5, 1, None, ctypes.byref(n)) == INVALID


def test_logprobs_workspace_refusals():
    """As the call's own: a negative top_n is no argument, one too large is not supported."""
    n = ctypes.c_size_t()
    size = capi.load().mle_token_logprobs_workspace_size
    for args, code in (((1, 5, -1), INVALID), ((1, 0, 1), INVALID), ((-1, 5, 1), INVALID),
                       ((65536, 5, 1), UNSUPPORTED), ((1, 5, 129), UNSUPPORTED)):
        assert size(*args, ctypes.byref(n), ctypes.byref(n)) == code, args
        assert "token_logprobs_workspace_size" in capi.last_error()
