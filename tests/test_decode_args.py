"""Refusals of the decode step's entry points: argument checks run before any
HIP call, so none of this touches a GPU."""
import ctypes

import pytest

import s2x

P = ctypes.c_void_p(1 << 20)  # an aligned address that no check follows
ODD = ctypes.c_void_p((1 << 20) + 8)
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


def cache(**kw):
    c = dict(k=1 << 20, v=1 << 20, type=s2x.TYPE_F16, page_size=16, n_pages=10, n_head=2, d_head=128,
             ld_page=2 * 16 * 128, ld_head=16 * 128, ld_tok=128)
    c.update(kw)
    return s2x.KVCache(**c)


BAD_CACHES = [
    (dict(type=s2x.TYPE_F32), UNSUPPORTED), (dict(type=7), UNSUPPORTED), (dict(page_size=24), UNSUPPORTED),
    (dict(page_size=0), UNSUPPORTED), (dict(page_size=-16), UNSUPPORTED), (dict(page_size=1 << 17), UNSUPPORTED),
    (dict(n_pages=0), INVALID), (dict(n_pages=1 << 31), INVALID), (dict(n_head=0), INVALID),
    (dict(n_head=2000), UNSUPPORTED), (dict(d_head=0), INVALID), (dict(d_head=100), UNSUPPORTED),
    (dict(d_head=264), UNSUPPORTED), (dict(ld_tok=0), INVALID), (dict(ld_tok=120), INVALID),
    (dict(ld_tok=132), INVALID), (dict(ld_head=16 * 128 - 8), INVALID), (dict(ld_page=2 * 16 * 128 - 8), INVALID),
    (dict(ld_head=-8), INVALID), (dict(ld_page=1 << 31), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(k=(1 << 20) + 8), INVALID),
    (dict(ld_head=128, ld_tok=128), INVALID),  # a token's heads over the next tokens
]


def qk(**kw):
    a = dict(x=P, x_type=0, ld_x=6 * 128, n_tok=4, n_q_head=2, q_norm=P, k_norm=P, eps=1e-6, freq=P, d_rot=128, style=0,
             pos=P, slots=P, q=P, ld_q=2 * 128, cache=cache(), stream=None)
    a.update(kw)
    c = a["cache"]
    a["cache"] = ctypes.byref(c) if c is not None else None
    return s2x.lib.s2x_qk_norm_rope_kv(*a.values())


def attn(**kw):
    a = dict(q=P, ld_q=4 * 128, cache=cache(), table=P, ld_table=8, kv_len=P, n_seq=1, max_len=128, n_q_head=4,
             scale=0.1, window=0, out=P, out_type=s2x.TYPE_F16, ld_out=4 * 128, lse=None, ws=P, ws_bytes=0,
             stream=None)
    a.update(kw)
    c = a["cache"]
    a["cache"] = ctypes.byref(c) if c is not None else None
    return s2x.lib.s2x_attn_paged(*a.values())


def slots(**kw):
    a = dict(kv_len=1 << 20, n_new=2 << 20, n_seq=4, free=3 << 20, n_free=9, page=16, n_pages=30, table=4 << 20,
             ld_table=5, max_tok=4, len_out=5 << 20, start=6 << 20, pos=7 << 20, slots=8 << 20, used=9 << 20,
             stream=None)
    a.update(kw)
    return s2x.lib.s2x_kv_slots(*a.values())


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_cache_refusals(change, status):
    c = cache(**change)
    for f in (qk, attn):
        assert f(cache=c) == status, s2x.lib.s2x_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(cache=None), INVALID), (dict(x_type=3), INVALID), (dict(style=2), INVALID), (dict(n_tok=-1), INVALID),
    (dict(n_tok=(1 << 23) + 1), UNSUPPORTED), (dict(n_q_head=0), INVALID), (dict(d_rot=130), INVALID),
    (dict(d_rot=3), INVALID), (dict(d_rot=-2), INVALID), (dict(ld_x=6 * 128 - 8), INVALID),
    (dict(ld_x=6 * 128 + 4), INVALID), (dict(ld_q=2 * 128 - 8), INVALID), (dict(ld_q=2 * 128 + 2), INVALID),
    (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(slots=None), INVALID), (dict(pos=None), INVALID),
    (dict(freq=None), INVALID), (dict(x=ODD), INVALID), (dict(q=ODD), INVALID)])
def test_qk_refusals(change, status):
    assert qk(**change) == status, s2x.lib.s2x_last_error()


def test_no_rows_is_no_work():
    assert qk(n_tok=0, x=None, q=None, slots=None, pos=None, freq=None) == OK
    assert attn(n_seq=0, q=None, out=None, kv_len=None) == OK


@pytest.mark.parametrize("change,status", [
    (dict(cache=None), INVALID), (dict(n_seq=-1), INVALID), (dict(n_seq=65536), UNSUPPORTED),
    (dict(max_len=-1), INVALID), (dict(max_len=(1 << 30) + 1), UNSUPPORTED), (dict(n_q_head=3), INVALID),
    (dict(n_q_head=0), INVALID), (dict(out_type=s2x.TYPE_BF16), UNSUPPORTED), (dict(out_type=9), UNSUPPORTED),
    (dict(window=-1), INVALID), (dict(ld_table=-1), INVALID), (dict(ld_q=504), INVALID), (dict(ld_out=516), INVALID),
    (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(kv_len=None), INVALID), (dict(table=None), INVALID),
    (dict(q=ODD), INVALID), (dict(out=ODD), INVALID),
    (dict(n_seq=65535, n_q_head=128, ld_q=1 << 14, ld_out=1 << 14,
          cache=cache(n_head=128, ld_page=128 * 16 * 128)), UNSUPPORTED)])
def test_attn_refusals(change, status):
    assert attn(**change) == status, s2x.lib.s2x_last_error()


def test_attn_workspace_refusals():
    size = s2x.lib.s2x_attn_paged_workspace_size
    assert size(-1, 100, 4, 2, 128) == 0 and size(1, 100, 3, 2, 128) == 0 and size(1, 100, 4, 2, 100) == 0
    assert size(100, 100, 4, 2, 128) == 0  # one chunk a sequence
    assert size(65535, 1 << 30, 64, 64, 128) < 1 << 42
    need = size(1, 1 << 17, 4, 2, 128)
    assert 0 < need < 1 << 30
    assert attn(max_len=1 << 17, ws_bytes=need - 1) == WORKSPACE
    assert attn(max_len=1 << 17, ws=None, ws_bytes=need) == INVALID
    assert attn(max_len=1 << 17, ws=ODD, ws_bytes=need) == INVALID


@pytest.mark.parametrize("change,status", [
    (dict(n_seq=-1), INVALID), (dict(n_seq=8193), UNSUPPORTED), (dict(page=20), UNSUPPORTED),
    (dict(page=0), UNSUPPORTED), (dict(n_free=-1), INVALID), (dict(max_tok=-1), INVALID),
    (dict(max_tok=2 ** 31 - 1), UNSUPPORTED), (dict(n_pages=2 ** 31), UNSUPPORTED), (dict(kv_len=None), INVALID),
    (dict(n_new=None), INVALID), (dict(free=None), INVALID), (dict(table=None), INVALID), (dict(len_out=None), INVALID),
    (dict(start=None), INVALID), (dict(pos=None), INVALID), (dict(slots=None), INVALID), (dict(used=None), INVALID),
    (dict(slots=(8 << 20) + 4), INVALID), (dict(len_out=1 << 20), INVALID), (dict(start=(2 << 20) - 4), INVALID),
    (dict(table=(3 << 20) - 40), INVALID), (dict(used=(1 << 20) + 8), INVALID)])
def test_slots_refusals(change, status):
    assert slots(**change) == status, s2x.lib.s2x_last_error()


def test_q4_refusals():
    lib = s2x.lib
    out = ctypes.c_void_p()
    o = ctypes.byref(out)
    assert lib.s2x_weight_q4_0_bytes(33, 4) == 0 and lib.s2x_weight_q4_0_bytes(32, 0) == 0
    assert lib.s2x_weight_q4_0_bytes((1 << 20) + 32, 4) == 0 and lib.s2x_weight_q4_0_bytes(32, (1 << 24) + 1) == 0
    assert lib.s2x_weight_q4_0_bytes(1 << 20, 1 << 17) == 0 and lib.s2x_weight_q4_0_bytes(1 << 19, 1 << 17) > 0
    assert lib.s2x_weight_q4_0_bytes(4096, 4096) == 4096 * 4096 // 32 * 18
    assert lib.s2x_weight_q4_0_create(P, 0, 100, 4, None, o) == INVALID
    assert lib.s2x_weight_q4_0_create(None, 1, 128, 4, None, o) == INVALID
    assert lib.s2x_weight_q4_0_create(P, 0, 128, 4, None, None) == INVALID
    assert lib.s2x_weight_q4_0_create_in(P, 128, 4, ODD, None, o) == INVALID
    assert lib.s2x_weight_q4_0_create_in(P, 128, 0, P, None, o) == INVALID
    assert out.value is None
    lib.s2x_weight_q4_0_destroy(None)
    assert lib.s2x_weight_q4_0_k(None) == 0 and lib.s2x_weight_q4_0_n(None) == 0
    assert lib.s2x_mul_mat_q4_0_q8_1(None, P, P, 1, P, 4, None, None, 0, None) == INVALID
    assert lib.s2x_mul_mat_q4_0_workspace_size(1152, 64, 256) == 0
    assert lib.s2x_mul_mat_q4_0_workspace_size(1152, 64, 257) >= 1152 * 64
    assert lib.s2x_mul_mat_q4_0_workspace_size(1150, 64, 257) == 0
