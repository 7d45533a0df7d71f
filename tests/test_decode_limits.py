"""The decode step's size limits and further refusals, which are decided on the
host: nothing here touches a GPU."""
import ctypes

import pytest

import s2x
from test_decode_args import INVALID, ODD, OK, UNSUPPORTED, WORKSPACE, P, cache, slots


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
