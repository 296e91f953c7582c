"""What the operators of a batched decode step refuse (include/mllm.h:
mllm_rope_kv_paged, mllm_attn_paged, mllm_sample), on the CPU: every check
comes before the GPU is touched."""
import ctypes as C

import pytest

from mllm import abi

BUF = (C.c_uint8 * 4096)()
B = C.addressof(BUF) + (-C.addressof(BUF) % 16)
INVALID, UNSUPPORTED = 1, 4


def pages(**kw):
    d = dict(k=B, v=B, storage=1, n_kv_heads=2, head_dim=64, pages=8, page_size=16, page_stride=0, head_stride=0,
             row_stride=0, table=B, sequences=4, table_cols=4)
    d.update(kw)
    return abi.MllmKvPages(*[d[n] for n, _ in abi.MllmKvPages._fields_])


BAD_PAGES = [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(table=None), INVALID),
    (dict(storage=3), UNSUPPORTED), (dict(storage=-1), UNSUPPORTED), (dict(head_dim=48), UNSUPPORTED),
    (dict(head_dim=288), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED), (dict(n_kv_heads=0), INVALID),
    (dict(pages=0), INVALID), (dict(page_size=0), INVALID), (dict(page_size=-16), INVALID),
    (dict(sequences=0), INVALID), (dict(table_cols=0), INVALID), (dict(page_size=1 << 20, table_cols=1 << 12), INVALID),
    (dict(k=B + 8), INVALID), (dict(v=B + 4), INVALID),
    (dict(page_stride=4096), INVALID),  # the other strides are 0
    (dict(page_stride=4096, head_stride=1024, row_stride=60), INVALID),  # rows overlap
    (dict(page_stride=4096, head_stride=1024, row_stride=68), INVALID),  # 136 bytes
    (dict(page_stride=-4096, head_stride=1024, row_stride=64), INVALID),
]


def rope(kv, tokens=3, heads=4, qkv=B, seq=B, pos=B, freq=B, rot=64, inter=0, gq=None, gk=None, q=B):
    return abi.lib().mllm_rope_kv_paged(kv, tokens, heads, qkv, seq, pos, freq, rot, inter, gq, gk, 1e-6, q, None)


def attn(kv, rows=3, heads=4, q=B, seq=B, ln=B, max_len=64, out=B, ws=B, nbytes=1 << 40):
    return abi.lib().mllm_attn_paged(kv, rows, heads, q, seq, ln, max_len, 0.125, out, ws, nbytes, None)


@pytest.mark.parametrize("over,code", BAD_PAGES, ids=[str(o) for o, _ in BAD_PAGES])
def test_pages_refused_by_both(over, code):
    assert rope(pages(**over)) == code
    assert abi.lib().mllm_last_error()
    assert attn(pages(**over)) == code
    assert abi.lib().mllm_attn_paged_workspace(pages(**over), 3, 4, 64) == 0


@pytest.mark.parametrize("over", [
    dict(tokens=0), dict(tokens=-1), dict(heads=0), dict(heads=3), dict(qkv=None), dict(pos=None), dict(q=None),
    dict(freq=None), dict(rot=63), dict(rot=-2), dict(rot=66), dict(qkv=B + 4), dict(q=B + 8),
    dict(seq=None, tokens=5), dict(tokens=1 << 30, heads=1 << 10)])
def test_rope_refusals(over):
    assert rope(pages(), **over) == INVALID


def test_rope_null_pages():
    assert rope(None) == INVALID and attn(None) == INVALID


@pytest.mark.parametrize("over", [
    dict(rows=0), dict(rows=-4), dict(heads=0), dict(heads=5), dict(q=None), dict(q=B + 4), dict(ln=None), dict(out=None),
    dict(max_len=-1), dict(max_len=65), dict(seq=None, rows=5), dict(rows=1 << 30, heads=1 << 10), dict(rows=1 << 23)])
def test_attn_refusals(over):
    assert attn(pages(), **over) == INVALID


def test_attn_workspace_is_checked():
    kv = pages(table_cols=64)
    need = abi.lib().mllm_attn_paged_workspace(kv, 3, 4, 1024)
    assert need > 0
    assert attn(kv, max_len=1024, ws=None) == INVALID
    assert attn(kv, max_len=1024, nbytes=need - 1) == INVALID
    assert attn(kv, max_len=1024, ws=B + 4, nbytes=need) == INVALID
    assert str(need).encode() in (attn(kv, max_len=1024, nbytes=0), abi.lib().mllm_last_error())[1]


@pytest.mark.parametrize("over,code", [
    (dict(rows=0), INVALID), (dict(vocab=0), INVALID), (dict(rows=1 << 22), INVALID), (dict(vocab=524289), UNSUPPORTED), (dict(logits=None), INVALID),
    (dict(u=None), INVALID), (dict(ids=None), INVALID)])
def test_sample_refusals(over, code):
    a = dict(rows=2, vocab=100, logits=B, u=B, ids=B)
    a.update(over)
    rc = abi.lib().mllm_sample(a["rows"], a["vocab"], a["logits"], None, None, None, None, a["u"], a["ids"], None, None)
    assert rc == code and abi.lib().mllm_last_error()


@pytest.mark.parametrize("size,cols", [(1 << 20, 2047), (1 << 20, 1025), ((1 << 30) + 1, 1), (1, (1 << 31) - 1)])
def test_positions_past_2_to_the_30_are_refused(size, cols):
    """Positions are stepped past in 32 bits: near 2^31 the steps would wrap."""
    kv = pages(page_size=size, table_cols=cols)
    assert rope(kv) == INVALID and attn(kv, max_len=size * cols) == INVALID
    assert abi.lib().mllm_attn_paged_workspace(kv, 3, 4, size * cols) == 0
    assert b"2^30" in abi.lib().mllm_last_error()


def test_the_largest_rows_and_heads_are_refused():
    """2^62 workgroups: their threads wrap 64 bits."""
    n = (1 << 31) - 1
    kv = pages(n_kv_heads=n, head_dim=32, sequences=n)
    assert abi.lib().mllm_attn_paged_workspace(kv, n, n, 64) == 0
    assert attn(kv, rows=n, heads=n) == INVALID and b"exceed a launch" in abi.lib().mllm_last_error()
    assert rope(kv, tokens=n, heads=n) == INVALID


def test_a_workspace_for_the_largest_call_serves_smaller_ones():
    """With an empty workspace the call says what it needs: never more than the
    function gave for as many rows and as long a cache, or more."""
    kv = pages(page_size=256, table_cols=1024)
    size = abi.lib().mllm_attn_paged_workspace
    at = [(r, n) for r in (1, 2, 3, 5, 16, 60, 130, 700, 2100) for n in (0, 256, 257, 1000, 4000, 6100, 9000, 70000, 262144)]
    needed = {}
    for r, n in at:
        rc, msg = attn(kv, rows=r, max_len=n, seq=B, out=None, nbytes=0), abi.lib().mllm_last_error().decode()
        assert rc == INVALID  # the workspace, or out
        needed[r, n] = int(msg.split(" bytes, ")[1].split()[0]) if "needed" in msg else 0
    assert sum(v > 0 for v in needed.values()) > 20
    for r, n in at:
        assert size(kv, r, 4, n) >= max(v for (a, b), v in needed.items() if a <= r and b <= n), (r, n)
