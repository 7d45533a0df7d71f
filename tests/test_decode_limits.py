"""The decode step's size limits and further refusals, which are decided on the
host: nothing here touches a GPU."""
import ctypes

import pytest

import s2x
from test_decode_args import INVALID, ODD, OK, UNSUPPORTED, WORKSPACE, P, attn, cache, qk, slots


def test_q4_workspace_past_the_int8_gemm():
    """Weights whose scales lie past the int8 GEMM's 31-bit offsets, or whose
    rows of y do, are read as they lie for any number of rows: no workspace."""
    size = s2x.lib.s2x_mul_mat_q4_0_workspace_size
    for m in (257, 1 << 20):
        assert size(1 << 19, 1 << 17, m) == 0  # K * N = 2^36
        assert size(1 << 18, 1 << 17, m) == 0  # 2^35
        assert size((1 << 18) - 32, 1 << 17, m) >= ((1 << 18) - 32) << 17
        assert size(1 << 18, (1 << 17) - 128, m) >= (1 << 18) * ((1 << 17) - 128)
        assert size(1 << 18, (1 << 17) - 127, m) == 0  # (columns count to whole 128)
        assert size(32, 1 << 22, m) == 0
        assert size(32, (1 << 22) - 1, m) >= 32 << 22


def attn_rows(**kw):
    a = dict(q=P, ld_q=4 * 128, n_row=3, tok_start=P, cache=cache(), table=P, ld_table=8, kv_len=P, n_seq=2, max_len=128,
             n_q_head=4, scale=0.1, window=0, out=P, out_type=s2x.TYPE_F16, ld_out=4 * 128, lse=None, ws=P, ws_bytes=0,
             stream=None)
    a.update(kw)
    a["cache"] = ctypes.byref(a["cache"]) if a["cache"] is not None else None
    return s2x.lib.s2x_attn_paged_rows(*a.values())


@pytest.mark.parametrize("change,status", [
    (dict(n_row=-1), INVALID), (dict(tok_start=None), INVALID), (dict(tok_start=ctypes.c_void_p((1 << 20) + 2)), INVALID),
    (dict(n_row=0, n_seq=-1), INVALID), (dict(cache=None), INVALID), (dict(cache=cache(d_head=100)), UNSUPPORTED),
    (dict(n_q_head=3), INVALID), (dict(ld_q=504), INVALID), (dict(ld_out=516), INVALID), (dict(q=None), INVALID),
    (dict(out=ODD), INVALID), (dict(kv_len=None), INVALID), (dict(table=None), INVALID),
    (dict(out_type=s2x.TYPE_BF16), UNSUPPORTED), (dict(window=-1), INVALID),
    (dict(max_len=1 << 17), WORKSPACE), (dict(max_len=1 << 17, ws=None), INVALID)])
def test_attn_rows_refusals(change, status):
    assert attn_rows(**change) == status, s2x.lib.s2x_last_error()


def test_attn_rows_without_rows():
    assert attn_rows(n_row=0, q=None, out=None, tok_start=None, kv_len=None) == OK
    assert attn_rows(n_seq=0, q=None, out=None, tok_start=None, kv_len=None) == OK


@pytest.mark.parametrize("change", [
    dict(pos=4 << 20), dict(slots=(4 << 20) + 72), dict(len_out=(4 << 20) - 8), dict(used=6 << 20),
    dict(start=(8 << 20) + 8), dict(pos=(5 << 20) + 12)])
def test_slots_outputs_apart(change):
    """The table (80 bytes from 4 << 20 on) is read while the others are
    written; no two outputs share a byte."""
    assert slots(**change) == INVALID, s2x.lib.s2x_last_error()


def test_attn_limits():
    """Sequences x key heads, a key head once for each 16 query heads on it; the
    largest lengths and head counts; refused shapes want no workspace."""
    size = s2x.lib.s2x_attn_paged_workspace_size
    assert size(1, 1 << 30, 1024, 1, 64) > 0 and size(1, (1 << 30) + 1, 1024, 1, 64) == 0
    assert size(1, 5000, 1024, 1, 64) > 0 and size(1, 5000, 1025, 1, 64) == 0
    # 18 query heads a key head count as two, 16 as one; the null pointer is refused behind the shape
    for n_q, n_kv, most in ((1008, 56, (1 << 22) // 112), (896, 56, 65535), (1024, 64, 65535), (1024, 1, 65535),
                            (128, 128, (1 << 22) // 128)):
        kw = dict(n_q_head=n_q, ld_q=n_q * 128, ld_out=n_q * 128, q=None)
        c = lambda: cache(n_head=n_kv, ld_page=n_kv * 16 * 128)
        assert attn(n_seq=most, cache=c(), **kw) == INVALID, (n_q, n_kv)
        assert attn(n_seq=most + 1, cache=c(), **kw) == UNSUPPORTED, (n_q, n_kv)
    assert attn(n_seq=0, max_len=1 << 30) == OK
    big = dict(ld_q=1026 * 128, ld_out=1026 * 128)
    assert attn(n_seq=0, n_q_head=1024, **big) == OK and attn(n_seq=0, n_q_head=1026, **big) == UNSUPPORTED
    assert attn(ld_table=1 << 31) == INVALID


def test_qk_limits():
    wide = dict(n_tok=0, ld_x=1100 * 128, ld_q=1100 * 128)
    assert qk(n_q_head=1024, **wide) == OK and qk(n_q_head=1025, **wide) == UNSUPPORTED
    most = dict(n_tok=0, ld_x=(2 + 2 * 1025) * 128)
    assert qk(cache=cache(n_head=1024, ld_page=1024 * 16 * 128), **most) == OK
    assert qk(cache=cache(n_head=1025, ld_page=1025 * 16 * 128), **most) == UNSUPPORTED
    assert qk(cache=cache(n_pages=2 ** 31 - 1), n_tok=0) == OK


@pytest.mark.parametrize("change", [dict(n_free=2 ** 31), dict(ld_table=2 ** 31), dict(n_pages=2 ** 31),
                                    dict(max_tok=2 ** 31 - 1), dict(n_seq=8193)])
def test_slots_limits(change):
    assert slots(**change) == UNSUPPORTED, s2x.lib.s2x_last_error()
