"""Refusals and limits of the beam search's entry points (the residual RMS norm
with Q8_1, the beam selection, the cache's pages, the attention over a prefix):
argument checks run before any HIP call, so none of this touches a GPU."""
import ctypes

import pytest

import s2x
from test_decode_args import BAD_CACHES, cache

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4
A = [i << 24 for i in range(1, 30)]  # aligned addresses far apart that no check follows
F32, F16, BF16 = s2x.TYPE_F32, s2x.TYPE_F16, s2x.TYPE_BF16


def call(name, args, kw):
    unknown = set(kw) - set(args)
    assert not unknown, unknown
    args = {**args, **kw}
    return getattr(s2x.lib, name)(*args.values())


def rms(**kw):
    return call("s2x_add_rmsnorm_quantize_q8_1", dict(
        x=A[0], x_type=F16, ld_x=100, resid=A[1], resid_type=F32, ld_resid=100, H=100, M=3, w=A[2], eps=1e-6, h_out=A[3],
        ld_h=100, K_pad=128, qs=A[4], ds=A[5], y=A[6], y_type=F32, ld_y=100, stream=None), kw)


@pytest.mark.parametrize("change,status", [
    (dict(x_type=3), INVALID), (dict(resid_type=-1), INVALID), (dict(y_type=7), INVALID),
    (dict(resid_type=BF16), UNSUPPORTED), (dict(x_type=F32, resid_type=F16), UNSUPPORTED),
    (dict(H=0), INVALID), (dict(H=-3), INVALID), (dict(M=-1), INVALID), (dict(M=(1 << 30) + 1), UNSUPPORTED),
    (dict(H=32769, ld_x=40000, ld_resid=40000, ld_h=40000, ld_y=40000, K_pad=32800), UNSUPPORTED),
    (dict(qs=None), INVALID), (dict(ds=None), INVALID), (dict(qs=None, ds=None, y=None), INVALID),
    (dict(K_pad=96), INVALID), (dict(K_pad=160), INVALID), (dict(K_pad=100), INVALID),
    (dict(ld_x=99), INVALID), (dict(ld_resid=99), INVALID), (dict(ld_h=99), INVALID), (dict(ld_y=99), INVALID),
    (dict(ld_x=(1 << 32) + 1), UNSUPPORTED), (dict(x=None), INVALID), (dict(x=A[0] + 1), INVALID),
    (dict(resid=A[1] + 2), INVALID), (dict(w=A[2] + 2), INVALID), (dict(h_out=A[3] + 2), INVALID),
    (dict(y=A[6] + 2), INVALID), (dict(qs=A[4] + 8), INVALID), (dict(ds=A[5] + 2), INVALID),
    (dict(y=A[1]), INVALID), (dict(y=A[3] + 1196), INVALID), (dict(h_out=A[0]), INVALID), (dict(h_out=A[2]), INVALID),
    (dict(h_out=A[1], ld_h=104), INVALID), (dict(h_out=A[1] + 400), INVALID), (dict(qs=A[1] + 16), INVALID),
    (dict(ds=A[4] + 256), INVALID)])
def test_rms_refusals(change, status):
    assert rms(**change) == status, s2x.lib.s2x_last_error()


def test_rms_without_rows():
    assert rms(M=0, x=None, qs=None, ds=None, y=None) == OK


def beam(**kw):
    return call("s2x_beam_select", dict(
        logits=A[0], type=F32, ld=1000, n_req=3, n_beam=4, n_vocab=1000, scores=A[1], done=A[2], done_token=2, n_out=8,
        parent=A[3], token=A[4], score=A[5], ws=A[6], ws_bytes=1 << 20, stream=None), kw)


@pytest.mark.parametrize("change,status", [
    (dict(type=3), INVALID), (dict(ld=999), INVALID), (dict(ld=(1 << 32) + 1), INVALID), (dict(n_req=-1), INVALID),
    (dict(n_beam=0), INVALID), (dict(n_beam=65), UNSUPPORTED), (dict(n_vocab=0), INVALID),
    (dict(n_vocab=(1 << 24) + 1, ld=1 << 25), UNSUPPORTED), (dict(n_out=0), INVALID), (dict(n_out=65), UNSUPPORTED),
    (dict(n_req=16384), UNSUPPORTED), (dict(n_req=65536, n_beam=1), UNSUPPORTED), (dict(logits=None), INVALID),
    (dict(scores=None), INVALID), (dict(parent=None), INVALID), (dict(token=None), INVALID), (dict(score=None), INVALID),
    (dict(ws=None), INVALID), (dict(ws=A[6] + 128), INVALID), (dict(ws_bytes=100), WORKSPACE),
    (dict(logits=A[0] + 2), INVALID), (dict(type=F16, logits=A[0] + 1), INVALID), (dict(token=A[4] + 2), INVALID),
    (dict(token=A[3] + 92), INVALID), (dict(score=A[1]), INVALID), (dict(ws=A[0]), INVALID), (dict(parent=A[2] + 8), INVALID)])
def test_beam_refusals(change, status):
    assert beam(**change) == status, s2x.lib.s2x_last_error()


def test_beam_sizes():
    size = s2x.lib.s2x_beam_select_workspace_size
    assert beam(n_req=0, logits=None, parent=None, ws=None) == OK
    assert 0 < size(1, 4, 32000, 4) < 1 << 16
    assert 0 < size(1, 64, 1 << 24, 64) < 1 << 31
    assert size(65535, 1, 1, 1) > 0
    assert size(65536, 1, 1, 1) == 0 and size(1, 65, 10, 1) == 0 and size(1, 1, 0, 1) == 0 and size(1, 1, 1, 65) == 0
    need = size(3, 4, 1000, 8)
    assert beam(ws_bytes=need - 1) == WORKSPACE


PAGES = dict(ws=A[20], ws_bytes=1 << 20, stream=None)


def fork(**kw):
    return call("s2x_kv_fork", dict(
        parent=A[0], n_out=5, kv_len=A[1], table=A[2], n_seq=4, ld_table=10, page=16, n_pages=100, pinned=A[3],
        table_out=A[4], ld_out=12, len_out=A[5], src=A[6], dst=A[7], tok=A[8], free=A[9], count=A[10], **PAGES), kw)


def compact(**kw):
    return call("s2x_kv_compact", dict(
        kv_len=A[1], table=A[2], n_seq=4, ld_table=10, page=16, n_pages=100, table_out=A[4], ld_out=12, src=A[6], dst=A[7],
        count=A[10], **PAGES), kw)


COMMON = [
    (dict(n_seq=-1), INVALID), (dict(n_seq=8193), UNSUPPORTED), (dict(page=20), UNSUPPORTED), (dict(page=0), UNSUPPORTED),
    (dict(page=1 << 17), UNSUPPORTED), (dict(n_pages=-1), INVALID),
    (dict(n_pages=(1 << 24) + 1), UNSUPPORTED), (dict(ld_table=-1), INVALID), (dict(ld_out=9), INVALID),
    (dict(ld_table=1 << 31, ld_out=1 << 31), UNSUPPORTED), (dict(kv_len=None), INVALID), (dict(table=None), INVALID),
    (dict(table_out=None), INVALID), (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(count=None), INVALID),
    (dict(count=A[10] + 4), INVALID), (dict(table=A[2] + 2), INVALID), (dict(ws=None), INVALID),
    (dict(ws=A[20] + 16), INVALID), (dict(ws_bytes=64), WORKSPACE), (dict(table_out=A[2]), INVALID),
    (dict(table_out=A[2] + 156), INVALID), (dict(dst=A[6]), INVALID), (dict(count=A[4] + 8), INVALID),
    (dict(ws=A[2]), INVALID)]


@pytest.mark.parametrize("change,status", COMMON)
def test_pages_refusals(change, status):
    assert fork(**change) == status, s2x.lib.s2x_last_error()
    assert compact(**change) == status, s2x.lib.s2x_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(n_out=-1), INVALID), (dict(n_out=8193), UNSUPPORTED), (dict(parent=None), INVALID), (dict(len_out=None), INVALID),
    (dict(tok=None), INVALID), (dict(free=None), INVALID), (dict(len_out=A[1]), INVALID), (dict(free=A[3]), INVALID),
    (dict(tok=A[7] + 16), INVALID), (dict(free=A[0] - 396), INVALID)])
def test_fork_refusals(change, status):
    assert fork(**change) == status, s2x.lib.s2x_last_error()


def test_pages_workspace():
    size = s2x.lib.s2x_kv_pages_workspace_size
    assert size(0) > 0 and size(-5) == 0 and size((1 << 24) + 1) == 0 and size(1) > 0 and size(1 << 24) < 1 << 28
    assert fork(ws_bytes=size(100) - 1) == WORKSPACE


def copy(cs=None, **kw):
    cs = [cache(), cache(k=A[12], v=A[13])] if cs is None else cs
    arr = (s2x.KVCache * max(1, len(cs)))(*cs)
    return call("s2x_kv_copy_pages", dict(caches=arr, n_cache=len(cs), src=A[0], dst=A[1], n_tok=None, n=4, n_dev=None,
                                          stream=None), kw)


@pytest.mark.parametrize("change,status", [
    (dict(n_cache=-1), INVALID), (dict(n=-1), INVALID), (dict(n=(1 << 24) + 1), UNSUPPORTED), (dict(caches=None), INVALID),
    (dict(src=None), INVALID), (dict(dst=None), INVALID), (dict(n_tok=A[2] + 2), INVALID), (dict(n_dev=A[2] + 4), INVALID)])
def test_copy_refusals(change, status):
    assert copy(**change) == status, s2x.lib.s2x_last_error()


def test_copy_caches():
    for change, status in BAD_CACHES:
        assert copy([cache(**change)]) == status
        assert copy([cache(), cache(**change)]) == status
    wide = dict(n_head=4, d_head=64, ld_page=4 * 16 * 64, ld_head=16 * 64, ld_tok=64)
    for change in (dict(type=s2x.TYPE_BF16), dict(n_pages=11), dict(ld_page=2 * 16 * 128 + 8), wide,
                   dict(page_size=8)):
        assert copy([cache(), cache(**change)]) == INVALID
    assert copy(n=0, src=None, dst=None) == OK and copy([], n_cache=0, caches=None) == OK


def prefix(**kw):
    a = dict(q=A[0], ld_q=512, n_row=6, tok_start=None, cache=cache(), table=A[1], ld_table=8, kv_len=A[2], n_seq=6,
             start=A[3], plen=A[4], n_group=2, max_group=3, max_prefix=100, max_own=50, n_q_head=4, scale=0.1, out=A[5],
             out_type=F16, ld_out=512, lse=None, ws=A[6], ws_bytes=1 << 24, stream=None)
    kw = dict(kw)
    c = kw.pop("cache", a["cache"])
    a["cache"] = ctypes.byref(c) if c is not None else None
    return call("s2x_attn_paged_prefix", a, kw)


@pytest.mark.parametrize("change,status", [
    (dict(cache=None), INVALID), (dict(n_group=-1), INVALID), (dict(max_group=-1), INVALID), (dict(max_prefix=-1), INVALID),
    (dict(max_own=-1), INVALID), (dict(n_group=65536), UNSUPPORTED), (dict(n_group=300, max_group=300), UNSUPPORTED),
    (dict(max_prefix=(1 << 30) + 1), UNSUPPORTED), (dict(max_own=(1 << 30) + 1), UNSUPPORTED), (dict(n_q_head=3), INVALID),
    (dict(n_seq=65536), UNSUPPORTED), (dict(n_seq=40000, n_q_head=1024), UNSUPPORTED),
    (dict(n_q_head=0), INVALID), (dict(n_q_head=1026), UNSUPPORTED), (dict(n_seq=-1), INVALID), (dict(n_row=-1), INVALID),
    (dict(out_type=BF16), UNSUPPORTED), (dict(out_type=9), UNSUPPORTED), (dict(ld_table=-1), INVALID),
    (dict(ld_q=504), INVALID), (dict(ld_q=516), INVALID), (dict(ld_out=504), INVALID), (dict(q=None), INVALID),
    (dict(out=None), INVALID), (dict(kv_len=None), INVALID), (dict(table=None), INVALID), (dict(start=None), INVALID),
    (dict(plen=None), INVALID), (dict(q=A[0] + 8), INVALID), (dict(out=A[5] + 8), INVALID), (dict(start=A[3] + 2), INVALID),
    (dict(tok_start=A[7] + 2), INVALID), (dict(lse=A[7] + 2), INVALID), (dict(ws=None), INVALID),
    (dict(ws=A[6] + 16), INVALID), (dict(ws_bytes=100), WORKSPACE)])
def test_prefix_refusals(change, status):
    assert prefix(**change) == status, s2x.lib.s2x_last_error()


def test_prefix_sizes():
    size = s2x.lib.s2x_attn_paged_prefix_workspace_size
    for change, status in BAD_CACHES:
        assert prefix(cache=cache(**change)) == status
    for none in (dict(n_seq=0), dict(n_row=0), dict(n_group=0), dict(max_group=0)):
        assert prefix(q=None, out=None, ws=None, **none) == OK
    assert size(0, 3, 100, 50, 4, 2, 128) == 0 and size(2, 0, 100, 50, 4, 2, 128) == 0
    assert size(2, 3, 100, 50, 3, 2, 128) == 0 and size(2, 3, 100, 50, 4, 2, 100) == 0
    need = size(2, 3, 100, 50, 4, 2, 128)
    assert 0 < need < 1 << 20 and prefix(ws_bytes=need - 1) == WORKSPACE
    assert size(1, 64, 1 << 17, 1000, 32, 8, 128) < 1 << 30
    # 2^21 sequences x key heads, 18 query heads on one counting twice
    assert size(1, 32768, 100, 50, 64, 64, 64) > 0 and size(1, 32769, 100, 50, 64, 64, 64) == 0
    assert size(1, 16384, 100, 50, 1024, 64, 64) > 0 and size(1, 18724, 100, 50, 1008, 56, 64) > 0
    assert size(1, 18725, 100, 50, 1008, 56, 64) == 0


def test_rms_columns_of_one_buffer():
    """Rows between one another's: one element too near is an overlap (that none is
    shows where there is a GPU)."""
    one = dict(x_type=F32, ld_x=400, ld_resid=400, ld_h=400, ld_y=400, qs=None, ds=None, x=A[0], resid=A[0] + 400,
               h_out=A[0] + 800, y=A[0] + 1200)
    for name, offset in (("resid", 404), ("h_out", 796), ("y", 1196), ("y", 1204), ("h_out", 1600 - 4), ("y", 2 * 1600 + 4)):
        bad = {**one, name: A[0] + offset}
        if name == "resid":
            bad["h_out"] = A[0] + 800
        assert rms(**bad) == INVALID, (name, offset)
    assert rms(**{**one, "ld_y": 404}) == INVALID
