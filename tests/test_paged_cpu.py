"""Refusals of the paged KV cache's calls (include/mle_paged.h): every check comes before
any HIP call, so none of these needs a GPU."""
import ctypes

import pytest

from llmengine_amd import capi

FAKE = 0x1000   # aligned, never dereferenced
ODD = 0x1002    # misaligned for 4-byte words
INVALID, UNSUPPORTED = 1, 4


def cache(**kw):
    a = dict(kv_type="f16", num_pages=8, page_size=16, kv_heads=2, head_dim=64, k=FAKE, v=FAKE,
             k_scale=None, v_scale=None)
    a.update(kw)
    return capi.PagedCache(**a)


def plan(**kw):
    a = dict(cached_lens=FAKE, new_lens=FAKE, sequences=2, block_table=FAKE, max_pages=4,
             page_size=16, num_pages=8, free_pages=FAKE, free_count=FAKE, free_count_out=FAKE,
             tokens=3, kv_lens=FAKE, cu_tokens=FAKE, positions=FAKE, slots=FAKE, granted=FAKE,
             stream=0)
    a.update(kw)
    return capi.paged_plan_status(**a)


def write(c=None, **kw):
    a = dict(cache=c or cache(), q=FAKE, q_out=FAKE, heads=4, k=FAKE, v=FAKE, rope=FAKE,
             rope_positions=10, rope_dim=64, rope_mode="halves", positions=FAKE, slots=FAKE,
             tokens=3, stream=0)
    a.update(kw)
    return capi.paged_kv_write_status(**a)


def attention(c=None, **kw):
    a = dict(cache=c or cache(), q=FAKE, out=FAKE, heads=4, scale=0.125, window=0,
             block_table=FAKE, max_pages=4, kv_lens=FAKE, cu_tokens=FAKE, sequences=2, tokens=3,
             stream=0)
    a.update(kw)
    return capi.paged_attention_status(**a)


CACHE_ERRORS = [
    (dict(k=None), INVALID, "cache k pointer"), (dict(v=None), INVALID, "cache v pointer"),
    (dict(k=0x1008), INVALID, "cache k must be 16-byte"),
    (dict(v=0x1004), INVALID, "cache v must be 16-byte"),
    (dict(kv_type=3), INVALID, "unknown cache type"),
    (dict(kv_type=-1), INVALID, "unknown cache type"),
    (dict(num_pages=0), INVALID, "num_pages must be positive"),
    (dict(page_size=-16), INVALID, "page_size must be positive"),
    (dict(kv_heads=0), INVALID, "kv_heads must be positive"),
    (dict(head_dim=80), UNSUPPORTED, "head_dim must be"),
    (dict(head_dim=0), UNSUPPORTED, "head_dim must be"),
    (dict(page_size=24), UNSUPPORTED, "page_size must be"),
    (dict(page_size=2048), UNSUPPORTED, "page_size must be"),
    (dict(num_pages=1 << 28), UNSUPPORTED, "31 bits"),
    (dict(kv_type="int8"), INVALID, "k_scale pointer"),
    (dict(kv_type="int8", k_scale=FAKE), INVALID, "v_scale pointer"),
    (dict(kv_type="int8", k_scale=0x1004, v_scale=FAKE), INVALID, "k_scale must be 16-byte"),
]


@pytest.mark.parametrize("bad,code,text", CACHE_ERRORS)
def test_cache_refusals(bad, code, text):
    for call in (write, attention):
        got, msg = call(cache(**bad))
        assert got == code and text in msg, (got, msg)


def test_null_cache():
    lib = capi.load()
    n = ctypes.c_size_t()
    assert lib.mle_paged_kv_write(None, *[0] * 17) == INVALID
    assert lib.mle_paged_attention(None, *[0] * 5, 1.0, *[0] * 8) == INVALID
    assert lib.mle_paged_attention_workspace_size(None, 1, 1, 1, ctypes.byref(n),
                                                  ctypes.byref(n)) == INVALID


@pytest.mark.parametrize("name", ["cached_lens", "new_lens", "block_table", "free_pages",
                                  "free_count", "free_count_out", "kv_lens", "cu_tokens",
                                  "positions", "slots", "granted"])
def test_plan_pointers(name):
    code, msg = plan(**{name: None})
    assert code == INVALID and name + " pointer" in msg
    code, msg = plan(**{name: ODD})
    assert code == INVALID and name + " must be 4-byte" in msg


@pytest.mark.parametrize("bad,code,text", [
    (dict(sequences=0), INVALID, "sequences"), (dict(max_pages=0), INVALID, "max_pages"),
    (dict(page_size=0), INVALID, "page_size"), (dict(num_pages=-1), INVALID, "num_pages"),
    (dict(tokens=-1), INVALID, "tokens"), (dict(tokens=1 << 30), UNSUPPORTED, "30 bits"),
    (dict(sequences=1 << 20, max_pages=1 << 12), UNSUPPORTED, "31 bits"),
    (dict(num_pages=1 << 27, page_size=16), UNSUPPORTED, "31 bits"),
])
def test_plan_sizes(bad, code, text):
    got, msg = plan(**bad)
    assert got == code and text in msg


@pytest.mark.parametrize("bad,code,text", [
    (dict(table=None), INVALID, "table pointer"), (dict(table=0x1008), INVALID, "16-byte"),
    (dict(positions=0), INVALID, "positions"), (dict(rope_dim=0), INVALID, "rope_dim"),
    (dict(rope_dim=7), INVALID, "even"), (dict(theta=0.0), INVALID, "theta"),
    (dict(theta=float("inf")), INVALID, "theta"), (dict(theta=float("nan")), INVALID, "theta"),
    (dict(freq_factors=ODD), INVALID, "freq_factors"),
])
def test_rope_table_refusals(bad, code, text):
    a = dict(table=FAKE, positions=4, rope_dim=64, stream=0)
    a.update(bad)
    got, msg = capi.rope_table_status(**a)
    assert got == code and text in msg


@pytest.mark.parametrize("bad,code,text", [
    (dict(q=None), INVALID, "q pointer"), (dict(q_out=None), INVALID, "q_out pointer"),
    (dict(k=None), INVALID, "k pointer"), (dict(v=None), INVALID, "v pointer"),
    (dict(slots=None), INVALID, "slots pointer"), (dict(slots=ODD), INVALID, "slots"),
    (dict(positions=None), INVALID, "positions pointer"),
    (dict(positions=ODD), INVALID, "positions must be"), (dict(q=0x1008), INVALID, "16-byte"),
    (dict(rope=0x1008), INVALID, "rope must be"), (dict(heads=0), INVALID, "heads"),
    (dict(tokens=-1), INVALID, "tokens"), (dict(tokens=1 << 30), UNSUPPORTED, "30 bits"),
    (dict(q_stride=252), INVALID, "q stride"), (dict(q_stride=258), INVALID, "q stride"),
    (dict(q_out_stride=128), INVALID, "q_out stride"), (dict(k_stride=124), INVALID, "k stride"),
    (dict(v_stride=129), INVALID, "v stride"), (dict(rope_positions=0), INVALID, "rope_pos"),
    (dict(rope_dim=0), INVALID, "rope_dim"), (dict(rope_dim=12), INVALID, "multiple of 8"),
    (dict(rope_dim=72), INVALID, "at most head_dim"), (dict(rope_mode=2), INVALID, "rope_mode"),
    (dict(tokens=1 << 28), UNSUPPORTED, "30 bits"),
])
def test_write_refusals(bad, code, text):
    got, msg = write(**bad)
    assert got == code and text in msg, (got, msg)


@pytest.mark.parametrize("bad,code,text", [
    (dict(q=None), INVALID, "q pointer"), (dict(out=None), INVALID, "out pointer"),
    (dict(block_table=None), INVALID, "block_table"), (dict(kv_lens=None), INVALID, "kv_lens"),
    (dict(cu_tokens=None), INVALID, "cu_tokens"), (dict(cu_tokens=ODD), INVALID, "cu_tokens"),
    (dict(block_table=ODD), INVALID, "block_table"), (dict(kv_lens=ODD), INVALID, "kv_lens"),
    (dict(out=0x1004), INVALID, "16-byte"), (dict(heads=0), INVALID, "heads"),
    (dict(heads=5), INVALID, "multiple of kv_heads"), (dict(heads=130), UNSUPPORTED, "at most 64"),
    (dict(sequences=0), INVALID, "sequences"), (dict(max_pages=0), INVALID, "max_pages"),
    (dict(max_pages=1 << 28), UNSUPPORTED, "31 bits"), (dict(window=-1), INVALID, "window"),
    (dict(scale=float("nan")), INVALID, "scale"), (dict(scale=float("inf")), INVALID, "scale"),
    (dict(q_stride=250), INVALID, "q stride"), (dict(out_stride=257), INVALID, "out stride"),
    (dict(tokens=-2), INVALID, "tokens"),
    (dict(heads=128, tokens=1 << 25), UNSUPPORTED, "31 bits"),
])
def test_attention_refusals(bad, code, text):
    got, msg = attention(**bad)
    assert got == code and text in msg, (got, msg)


def test_no_tokens_is_a_no_op():
    assert write(tokens=0)[0] == 0 and attention(tokens=0)[0] == 0


def test_workspace_size():
    """Grows with the call, and is refused for what the call refuses."""
    last = (0, 0)
    for tokens in (1, 64, 4096):
        size = capi.paged_attention_workspace_size(cache(), 4, 64, tokens)
        assert size[0] >= last[0] and size[1] >= last[1]
        last = size
    for kw in (dict(heads=5), dict(sequences=0), dict(tokens=-1)):
        a = dict(heads=4, sequences=2, tokens=3)
        a.update(kw)
        with pytest.raises(capi.Q8_0Error):
            capi.paged_attention_workspace_size(cache(), **a)


def test_rotation_table_without_a_mode():
    """rope_mode "none" says that nothing turns: with a table it is refused, not taken for pairs."""
    got, msg = write(rope_mode="none")
    assert got == INVALID and "rope_mode" in msg, (got, msg)
    assert write(rope=None, rope_mode="none", tokens=0)[0] == 0


@pytest.mark.parametrize("head_dim,heads,kv_heads,tokens", [
    (64, 4, 2, (1 << 32) // (8 * 6)), (96, 2, 1, (1 << 32) // (16 * 3) + 1),
    (128, 8, 8, (1 << 32) // (16 * 20) + 1), (256, 8, 8, 1 << 23), (256, 1, 1, 1 << 26)])
def test_write_of_more_threads_than_a_launch_has(head_dim, heads, kv_heads, tokens):
    row, kv_row = heads * head_dim, kv_heads * head_dim
    got, msg = write(cache(head_dim=head_dim, kv_heads=kv_heads), heads=heads, tokens=tokens,
                     q_stride=row, q_out_stride=row, k_stride=kv_row, v_stride=kv_row)
    assert got == UNSUPPORTED and "2^32 threads" in msg, (got, msg)


@pytest.mark.parametrize("positions,rope_dim", [(1 << 27, 64), (1 << 30, 1 << 20),
                                                (0x7fffffff, 0x7ffffffe)])
def test_rope_table_of_more_threads_than_a_launch_has(positions, rope_dim):
    got, msg = capi.rope_table_status(FAKE, positions, rope_dim, stream=0)
    assert got == UNSUPPORTED and "2^32" in msg, (got, msg)


def test_no_asm_writes_m0_unseen():
    """An asm statement cannot name m0 as overwritten, so none may write it: it gets m0 as an
    operand, which the compiler sets."""
    import glob
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    files = glob.glob(os.path.join(root, "llmengine_amd", "csrc", "**", "*.h*"), recursive=True)
    assert len(files) > 10
    for path in files:
        with open(path) as f:
            code = re.sub(r"//[^\n]*", "", f.read())
        for text in re.findall(r"\basm\b[^;]*;", code):
            assert not re.search(r"[\"\s]s_\w+ m0\b", text), (path, text)


def test_places_of_joined_parts():
    """The threads that join a tile's parts read inside them: built from the kernel's header."""
    import os
    import subprocess
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "bin",
                       "test_paged_parts")
    if not os.path.exists(exe):
        pytest.fail(f"{exe} not built: run `python -m llmengine_amd.build`")
    p = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                       timeout=60)
    assert p.returncode == 0, p.stdout
