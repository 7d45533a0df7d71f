"""The decode step on the GPU, each operator through the C-ABI against a plain
form in 64 bits, then the step as a whole, eager and captured.

Tolerances count roundings: u = 2^-24 for f32, half a step of the output's type
for the last rounding."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import (CODES, HALF_STEP, TYPES, Cache, attn_ref, heads_ref, q4_0_blocks, q8_0_blocks, q8_1_planes,
                         slots_ref)
from gpu_util import assert_same, dev, empty, host, ptr, say, stream

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAN = float("nan")


def within(got, ref, tol, what):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~(np.abs(got - ref) <= tol)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        say(f"{what}: {bad.sum()} of {bad.size} off; first {i}: got {got[i]!r} ref {ref[i]!r} "
            f"tol {np.broadcast_to(tol, ref.shape)[i]!r}")
    assert not bad.any(), what


# ---------------------------------------------------------------------------
# slots
# ---------------------------------------------------------------------------
def run_slots(kv_len, n_new, free, page, n_pages, table, max_tok, st=None):
    n = len(kv_len)
    t = [dev(np.asarray(a, np.int32)) for a in (kv_len, n_new, free)]
    tab = dev(table.astype(np.int32))
    out = [torch.full((size,), -77, dtype=dt, device="cuda:0")
           for size, dt in ((n, torch.int32), (n + 1, torch.int32), (max_tok, torch.int32), (max_tok, torch.int64),
                            (2, torch.int64))]
    s2x.call("s2x_kv_slots", ptr(t[0]), ptr(t[1]), n, ptr(t[2]), len(free), page, n_pages, ptr(tab), table.shape[1],
             max_tok, *[ptr(o) for o in out], st or stream())
    return [host(tab)] + [host(o) for o in out]


def check_slots(kv_len, n_new, free, page, n_pages, table, max_tok, what):
    say(f"slots: {what}")
    got = run_slots(kv_len, n_new, free, page, n_pages, table, max_tok)
    ref = slots_ref(kv_len, n_new, free, page, n_pages, table, max_tok)
    for name, g, r in zip(("table", "len", "start", "pos", "slots", "used"), got, ref):
        assert_same(g, r, f"{what} {name}")


def slots_case(rng, n_seq, len_max, new_max, page, short=0, lost=0):
    """A consistent batch; `short` pages missing from the free list, `lost`
    rows too few."""
    kv_len = rng.integers(0, len_max + 1, n_seq).astype(np.int32)
    n_new = rng.integers(0, new_max + 1, n_seq).astype(np.int32)
    if n_seq > 3:
        kv_len[1], n_new[2], n_new[3] = 0, 0, page
    have = -(-kv_len // page)
    want = -(-(kv_len + n_new) // page)
    n_pages = int(want.sum()) + 5
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n_seq, int(want.max(initial=0)) + 2), -1, np.int32)
    at = 0
    for b in range(n_seq):
        table[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    need = int((want - have).sum())
    return kv_len, n_new, ids[at:at + max(0, need - short)], page, n_pages, table, max(0, int(n_new.sum()) + 9 - lost)


@pytest.mark.parametrize("n_seq,len_max,new_max,page", [
    (1, 0, 1, 16), (1, 40, 1, 1), (5, 33, 1, 16), (64, 300, 1, 32), (65, 500, 40, 16), (3, 5000, 3000, 64),
    (1023, 50, 3, 8), (1025, 20, 9, 16), (8192, 30, 2, 16), (2, 70000, 1, 65536)])
def test_slots(n_seq, len_max, new_max, page):
    rng = np.random.default_rng(n_seq * 7 + page)
    check_slots(*slots_case(rng, n_seq, len_max, new_max, page), f"{n_seq} seq, page {page}")


def test_slots_shortages():
    """Too few free pages, too few rows, a table too narrow, ids outside the
    cache, negative lengths."""
    rng = np.random.default_rng(3)
    check_slots(*slots_case(rng, 20, 100, 50, 16, short=7), "7 pages short")
    check_slots(*slots_case(rng, 20, 100, 50, 16, short=10 ** 6), "no free pages")
    check_slots(*slots_case(rng, 20, 100, 50, 16, lost=40), "31 rows short")
    check_slots(*slots_case(rng, 20, 100, 50, 16, lost=10 ** 6), "no rows")
    c = list(slots_case(rng, 20, 100, 50, 16))
    c[5] = c[5][:, :4].copy()
    check_slots(*c, "narrow table")
    c = list(slots_case(rng, 20, 100, 50, 16))
    c[4] = 40  # ids from 40 up are none
    check_slots(*c, "ids outside")
    c = list(slots_case(rng, 20, 100, 50, 16))
    c[0][4], c[1][5], c[1][6] = -5, -2 ** 31, 0
    check_slots(*c, "negative lengths")
    # no sequences at all
    got = run_slots([], [], [], 16, 4, np.zeros((0, 3), np.int32), 5)
    assert got[2].tolist() == [0] and got[3].tolist() == [0] * 5 and got[4].tolist() == [-1] * 5
    assert got[5].tolist() == [0, 0]


def test_slots_huge_lengths():
    """Sums past 31 bits: starts stop at the rows there are, pages at the free
    list; nothing is written past the table."""
    table = np.full((3, 2), -1, np.int32)
    kv_len, n_new = [2 ** 31 - 1, 5, 0], [2 ** 31 - 1, 2 ** 31 - 1, 3]
    got = run_slots(kv_len, n_new, [1, 0], 65536, 2, table, 100)
    assert got[1].tolist() == [2 ** 31 - 1, 2 ** 31 - 1, 3]
    assert got[2].tolist() == [0, 100, 100, 100]
    assert (got[4] == -1).all() and (got[3] == 2 ** 31 - 1).all()  # sequence 0's: behind its row, past 31 bits
    assert got[5].tolist() == [32768 + 32768 + 1, 2 * (2 ** 31 - 1) + 3]
    # sequence 1 holds entry 0; its first new page is past the free list, the rows of the table stay -1
    assert got[0].tolist() == [[-1, -1], [-1, -1], [-1, -1]]


# ---------------------------------------------------------------------------
# norms, rotation, cache write
# ---------------------------------------------------------------------------
def qk_case(seed, t, hq, hkv, d, d_rot, style, norm, x_kind, kind, page, by, gap=0, far=5000, pad=0, qpad=0):
    rng = np.random.default_rng(seed)
    ld = (hq + 2 * hkv) * d + pad
    x = torch.from_numpy((rng.standard_normal((t, ld)) * 2).astype(np.float32)).to(TYPES[x_kind])
    wq, wk = (rng.normal(1, 0.2, (2, d)).astype(np.float32) if norm else (None, None))
    freq = 10000.0 ** (-np.arange(0, d_rot, 2) / max(d_rot, 1))
    pos = rng.integers(0, far, t).astype(np.int32)
    n_pages = t // page + 2
    slots = rng.permutation(n_pages * page)[:t].astype(np.int64)
    if t > 2:
        slots[t // 2] = -1
        slots[t - 1] = n_pages * page  # one past the cache
    cache = Cache(n_pages, hkv, page, d, kind, by, gap)
    before = [m.clone() for m in cache.mem]
    q = torch.full((t, hq * d + qpad), NAN, dtype=TYPES[kind], device="cuda:0")
    xd, eps = x.to("cuda:0"), 1e-6
    args = [None if a is None else dev(a) for a in (wq, wk, freq, pos, slots)]
    s2x.call("s2x_qk_norm_rope_kv", ptr(xd), CODES[x_kind], ld, t, hq, ptr(args[0]), ptr(args[1]), eps, ptr(args[2]),
             d_rot, s2x.ROPE_HALVES if style == "half" else s2x.ROPE_PAIRS, ptr(args[3]), ptr(args[4]), ptr(q),
             hq * d + qpad, cache.ref(), stream())
    torch.cuda.synchronize()
    heads = heads_ref(x.float().numpy()[:, :(hq + 2 * hkv) * d], hq, hkv, d, wq, wk, eps, freq, d_rot, style, pos)
    u = HALF_STEP[kind]
    # of 32 f32 roundings at most a value's own size each: 14 / 2 in the sum
    # of squares, 6 in 1/sqrt and the two products, 2 + 4 in angle, cos and
    # sin, 3 in the rotation; then one to the output's type (2^-25: half the
    # smallest step of f16)
    tols = [u * np.abs(r) + 32 * U * s + 2.0 ** -25 for r, s in heads]
    within(q[:, :hq * d].double().cpu().numpy().reshape(t, hq, d), heads[0][0], tols[0], "q")
    assert torch.isnan(q[:, hq * d:]).all()
    # the cache: the rows of valid slots, every other element as it was
    ok = (slots >= 0) & (slots < n_pages * page)
    want = [b.clone() for b in before]
    for c, m, i in ((cache.k, cache.mem[0], 1), (cache.v, cache.mem[1], 2)):
        got = c[slots[ok] // page, :, slots[ok] % page].double().cpu().numpy()
        within(got, heads[i][0][ok], tols[i][ok], "kv"[i - 1])
        w = want[i - 1]
        view = w[..., :d] if by == "head" else w[..., :d].transpose(1, 2)
        view[slots[ok] // page, :, slots[ok] % page] = c[slots[ok] // page, :, slots[ok] % page]
        assert torch.equal(w.view(torch.int16), m.view(torch.int16)), "the rest of the cache"
    return q, cache


@pytest.mark.parametrize("t,hq,hkv,d,d_rot,style,norm,x_kind,kind,page,by", [
    (1, 16, 16, 72, 72, "half", True, "f32", "f16", 16, "head"),
    (5, 4, 4, 72, 36, "half", True, "f32", "f16", 16, "token"),      # pairs end inside a lane
    (7, 3, 1, 72, 36, "pairs", True, "f16", "bf16", 8, "head"),
    (33, 8, 2, 128, 128, "half", True, "bf16", "bf16", 64, "head"),
    (17, 6, 3, 128, 64, "pairs", False, "bf16", "f16", 1, "token"),
    (9, 5, 5, 64, 64, "pairs", True, "f32", "bf16", 32, "head"),
    (40, 2, 1, 256, 256, "half", True, "f16", "f16", 16, "token"),
    (11, 2, 2, 256, 250, "half", True, "f32", "f16", 16, "head"),    # 32 + 1 lanes a head
    (6, 7, 1, 8, 8, "half", True, "f32", "f16", 4, "head"),
    (6, 1, 1, 8, 2, "pairs", True, "f32", "bf16", 4, "head"),
    (13, 3, 3, 80, 0, "half", True, "f32", "f16", 16, "head"),       # no rotation
    (1500, 3, 1, 96, 96, "half", True, "f32", "f16", 128, "token"),  # several tokens a workgroup
    (1027, 1, 1, 192, 10, "pairs", False, "bf16", "bf16", 16, "head"),
    (1026, 2, 1, 64, 0, "half", True, "f16", "bf16", 16, "head")])
def test_qk_norm_rope(t, hq, hkv, d, d_rot, style, norm, x_kind, kind, page, by):
    say(f"qk: {t} rows {hq}/{hkv} x {d} rot {d_rot} {style} {x_kind}->{kind}")
    qk_case(t + d, t, hq, hkv, d, d_rot, style, norm, x_kind, kind, page, by)


@pytest.mark.parametrize("t,hq,hkv,d,d_rot,style,norm,x_kind,kind,page,by", [
    (4097, 1, 1, 96, 48, "half", True, "f32", "bf16", 16, "head"),   # workgroups of one and two waves
    (4096, 9, 3, 128, 128, "pairs", True, "bf16", "f16", 64, "token"),
    (4099, 2, 1, 72, 36, "half", False, "f16", "bf16", 16, "head"),
    (4097, 1, 2, 256, 256, "half", True, "f16", "f16", 8, "head"),
    (4097, 1, 1, 64, 0, "half", True, "f32", "f16", 16, "head")])
def test_qk_few_heads_many_rows(t, hq, hkv, d, d_rot, style, norm, x_kind, kind, page, by):
    say(f"qk: {t} rows {hq}/{hkv} x {d} rot {d_rot} {style} {x_kind}->{kind}")
    qk_case(t + d, t, hq, hkv, d, d_rot, style, norm, x_kind, kind, page, by)


def test_qk_strides_and_far_positions():
    qk_case(1, 37, 4, 2, 128, 128, "half", True, "f32", "f16", 16, "head", gap=8, pad=24, qpad=40)
    qk_case(2, 37, 4, 2, 72, 72, "pairs", True, "bf16", "bf16", 16, "token", gap=16, pad=8, qpad=8)
    qk_case(3, 64, 2, 2, 64, 64, "half", True, "f32", "f16", 16, "head", far=2 ** 31 - 1)


def test_qk_special_values():
    """A head of zeros stays zeros, an infinity or a NaN reaches its own head
    alone, f16 overflow is an infinity."""
    t, hq, hkv, d = 4, 2, 1, 64
    x = np.ones((t, (hq + 2 * hkv) * d), np.float32)
    x[0, :d] = 0.0
    x[1, 5] = np.nan
    x[2, 3 * d + 1] = 1e9  # a value head: 1e9 is past f16
    cache = Cache(1, hkv, 16, d, "f16")
    q = empty((t, hq * d), torch.float16)
    xd, w, freq = dev(x), dev(np.ones(d, np.float32)), dev(np.zeros(d // 2))
    pos, slots = dev(np.zeros(t, np.int32)), dev(np.arange(t, dtype=np.int64))
    s2x.call("s2x_qk_norm_rope_kv", ptr(xd), 0, x.shape[1], t, hq, ptr(w), ptr(w), 1e-6, ptr(freq), d, 0, ptr(pos),
             ptr(slots), ptr(q), hq * d, cache.ref(), stream())
    g = host(q.float())
    assert (g[0, :d] == 0).all() and (g[0, d:] == 1).all()
    assert np.isnan(g[1, :d]).all() and (g[1, d:] == 1).all() and (g[2:] == 1).all()
    v = host(cache.v.float())[0, 0, :t]
    assert np.isinf(v[2, 1]) and (np.delete(v.ravel(), 2 * d + 1) == 1).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attn_inputs(rng, lens, hq, hkv, d, kind, page, by, gap=0, spread=1.5):
    n = len(lens)
    held = [-(-max(0, int(x)) // page) for x in lens]
    n_pages = sum(held) + 1
    cache = Cache(n_pages, hkv, page, d, kind, by, gap)  # NaN wherever no token is
    table = np.full((n, max(held + [1]) + 1), -1, np.int32)
    ids, at = rng.permutation(n_pages), 0
    for s, h in enumerate(held):
        table[s, :h] = ids[at:at + h]
        at += h
        for t0 in range(0, max(0, int(lens[s])), page):
            c = min(page, int(lens[s]) - t0)
            for m in (cache.k, cache.v):
                m[int(table[s, t0 // page]), :, :c] = torch.from_numpy(
                    rng.standard_normal((hkv, c, d)).astype(np.float32)).to("cuda:0")
    q = torch.from_numpy((rng.standard_normal((n, hq, d)) * spread).astype(np.float32)).to(TYPES[kind])
    return q, cache, table


def run_attn(q, cache, table, lens, max_len, scale, window, out_kind, qpad=0, opad=0, lse=True, st=None, ws=None):
    n, hq, d = q.shape
    qd = torch.full((n, hq * d + qpad), NAN, dtype=q.dtype, device="cuda:0")
    qd[:, :hq * d] = q.reshape(n, -1).to("cuda:0")
    out = torch.full((n, hq * d + opad), NAN, dtype=TYPES[out_kind], device="cuda:0")
    ls = torch.full((n, hq), NAN, device="cuda:0") if lse else None
    td, ld = dev(table), dev(np.asarray(lens, np.int32))
    size = s2x.lib.s2x_attn_paged_workspace_size(n, max_len, hq, cache.n_head, d)
    if ws is None:
        ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda:0")  # NaNs
    torch.cuda.synchronize()
    s2x.call("s2x_attn_paged", ptr(qd), hq * d + qpad, cache.ref(), ptr(td), table.shape[1], ptr(ld), n, max_len, hq,
             scale, window, ptr(out), CODES[out_kind], hq * d + opad, ptr(ls), ptr(ws), size, st or stream())
    torch.cuda.synchronize()
    assert torch.isnan(out[:, hq * d:]).all()
    return out[:, :hq * d].double().cpu().numpy().reshape(n, hq, d), None if ls is None else host(ls)


def check_attn(q, cache, table, lens, max_len, scale, window, out_kind, **kw):
    got, lse = run_attn(q, cache, table, lens, max_len, scale, window, out_kind, **kw)
    ref, size, rlse, top, seen = attn_ref(q.float().numpy(), cache, table, lens, max_len, scale, window)
    d = q.shape[2]
    # a score is off by its d products' roundings, the scale's and the
    # exponent's, exp by 2 ulp, a probability by that and by its two (three)
    # terms of the cache's type, the two sums by a rounding a key at most
    score = (d + 6) * U * top
    prob = {"f16": 2.0 ** -21, "bf16": 2.0 ** -15 if out_kind != "f32" else 2.0 ** -22}[cache.kind]
    n = seen[:, None]
    rel = 2 * score + 4 * U + prob + 2 * (n + 8) * U
    within(got, ref, rel[:, :, None] * size + HALF_STEP[out_kind] * np.abs(ref) + 2.0 ** -25, "out")
    if lse is not None:
        empty_ = np.isinf(rlse)
        assert (lse[empty_] == -np.inf).all()
        within(np.where(empty_, 0, lse), np.where(empty_, 0, rlse),
               score + (n + 8) * U + 4 * U * np.abs(np.where(empty_, 0, rlse)), "lse")


@pytest.mark.parametrize("lens,hq,hkv,d,kind,out_kind,page,by", [
    ([1], 1, 1, 64, "f16", "f16", 16, "head"),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 4, 2, 128, "f16", "f32", 16, "head"),
    ([0], 4, 2, 128, "bf16", "bf16", 16, "token"),
    ([300, 7, 0, 129], 16, 16, 72, "f16", "f32", 16, "head"),
    ([300, 7, 0, 129], 16, 16, 72, "bf16", "f32", 1, "token"),
    ([127, 128, 129, 255, 256, 257], 8, 1, 128, "bf16", "bf16", 64, "head"),
    ([513, 64, 65], 48, 2, 64, "f16", "f16", 32, "token"),      # 24 query heads on one key head
    ([200, 90], 34, 2, 80, "f16", "f16", 8, "head"),            # 17 on one
    ([1000], 3, 1, 256, "f16", "f32", 16, "head"),
    ([999, 1], 5, 5, 192, "bf16", "bf16", 128, "token"),
    ([77, 1234], 6, 2, 96, "f16", "f16", 4, "head"),
    ([100, 50], 2, 1, 8, "f16", "f32", 16, "head"),
    ([61, 50], 2, 1, 40, "bf16", "f32", 2, "token"),
    ([5000, 3, 2600], 16, 2, 128, "f16", "f16", 16, "head"),
    ([2000], 4, 4, 128, "bf16", "f32", 2048, "token"),
    ([300, 31], 32, 2, 256, "f16", "f16", 16, "head"),           # the most LDS a workgroup takes
    ([1200], 16, 1, 248, "bf16", "f32", 32, "token"),
    ([90, 250], 20, 1, 208, "f16", "f32", 16, "head"),
    ([1021] * 16, 8, 8, 64, "f16", "f16", 16, "head"),           # one launch past 320 tokens
    ([3, 0, 12] * 30, 5, 5, 256, "bf16", "f32", 16, "head"),     # many short ones
    (list(range(300, 380)), 4, 4, 72, "f16", "f16", 16, "head"),
    ([7000], 1, 1, 72, "f16", "f32", 16, "token"),               # more than 32 chunks
    (list(range(0, 740, 20)), 2, 1, 64, "bf16", "bf16", 16, "head")])
def test_attn_paged(lens, hq, hkv, d, kind, out_kind, page, by):
    say(f"attn: lens {lens} {hq}/{hkv} x {d} {kind}->{out_kind} page {page} {by}")
    rng = np.random.default_rng(sum(lens) + d)
    q, cache, table = attn_inputs(rng, lens, hq, hkv, d, kind, page, by)
    check_attn(q, cache, table, lens, max(max(lens), 1), d ** -0.5, 0, out_kind)


@pytest.mark.parametrize("window", [1, 2, 31, 100, 128, 5000])
def test_attn_window(window):
    rng = np.random.default_rng(window)
    lens = [0, 1, 90, 128, 1000, 2049]
    q, cache, table = attn_inputs(rng, lens, 6, 2, 128, "f16", 16, "head")
    check_attn(q, cache, table, lens, 2049, 128 ** -0.5, window, "f32")


@pytest.mark.parametrize("n,length,window,hq,hkv", [
    (2, 9000, 300, 4, 2), (2, 9000, 2000, 4, 2), (1, 40000, 5000, 2, 1), (40, 1500, 700, 4, 4), (130, 1030, 1000, 1, 1),
    (6, 3000, 2990, 8, 8)])
def test_attn_window_of_long_sequences(n, length, window, hq, hkv):
    """Chunks laid for the window, in the workspace sized without it; tokens
    before the window in pages that are gone from the table."""
    rng = np.random.default_rng(window)
    lens = [length - 7 * i for i in range(n)]
    q, cache, table = attn_inputs(rng, lens, hq, hkv, 64, "f16", 16, "head")
    for i, x in enumerate(lens):
        table[i, :max(0, (x - window) // 16)] = -1
    check_attn(q, cache, table, lens, length, 0.125, window, "f32")


def test_attn_bounds_and_strides():
    """Lengths past max_len and past the table's row, page ids outside the
    cache, negative lengths, gaps between rows, a batch with no pages."""
    rng = np.random.default_rng(11)
    lens = [700, 400, 300, 650]
    q, cache, table = attn_inputs(rng, lens, 8, 4, 72, "f16", 16, "token", gap=8)
    check_attn(q, cache, table, lens, 512, 0.1, 0, "f16", qpad=8, opad=16)  # (three sequences past max_len)
    table = np.ascontiguousarray(table[:, :20])
    check_attn(q, cache, table, lens, 700, 0.1, 0, "f32", opad=8)
    bad = table.copy()
    bad[0, 3], bad[1, 5:8], bad[2] = -1, cache.n_pages, 2 ** 31 - 1
    bad[3, 0] = -2 ** 31
    check_attn(q, cache, bad, lens, 700, 0.1, 0, "f32", lse=True)
    check_attn(q, cache, bad, lens, 700, 0.1, 40, "f32", lse=False)
    check_attn(q, cache, table, [-1, -2 ** 31, 5, 2 ** 31 - 1], 700, 0.1, 0, "f16")
    check_attn(q, cache, table, [0, 0, 0, 0], 0, 0.1, 0, "f16")


def test_attn_score_range():
    """Scores far apart (the running maximum moves by hundreds), one key that
    takes everything, equal scores, and infinite and NaN keys in other
    sequences' pages."""
    rng = np.random.default_rng(5)
    lens = [600, 600, 600]
    q, cache, table = attn_inputs(rng, lens, 4, 1, 128, "bf16", 16, "head")
    q = q * 20
    check_attn(q, cache, table, lens, 600, 1.0, 0, "f32")
    check_attn(q, cache, table, lens, 600, -1.0, 0, "f32")
    check_attn(q, cache, table, lens, 600, 0.0, 0, "f32")
    cache.k[int(table[1, 3]), 0, 5] = float("inf")
    cache.v[int(table[1, 2]), 0, 5] = NAN
    got, lse = run_attn(q, cache, table, lens, 600, 0.05, 0, "f32")
    ref = attn_ref(q.float().numpy()[[0, 2]], cache, table[[0, 2]], [600, 600], 600, 0.05, 0)
    within(got[[0, 2]], ref[0], 1e-3 * ref[1], "neighbours of a NaN")
    assert np.isnan(got[1]).any(axis=1).all()  # its own rows say so


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attn_infinite_value(kind):
    """An infinite value that is seen makes its own element infinite or a NaN, for
    the heads on its key head; every other element keeps its bits.  One that a
    window leaves out changes nothing.  (The first term of a probability is
    positive: inf; or 0, where it underflows: NaN.  The second is the first's
    rounding error: positive, and the sum is inf; negative, inf - inf; 0, inf +
    0 * inf.  Never finite, never -inf.)"""
    rng = np.random.default_rng(7)
    lens = [90, 700]  # one chunk and several
    q, cache, table = attn_inputs(rng, lens, 4, 2, 72, kind, 16, "head")
    before, lse0 = run_attn(q, cache, table, lens, 700, 0.1, 0, "f32")
    apart, _ = run_attn(q, cache, table, lens, 700, 0.1, 40, "f32")
    for s in (0, 1):
        cache.v[int(table[s, 1]), 1, 3, 37] = float("inf")  # token 19
    got, lse = run_attn(q, cache, table, lens, 700, 0.1, 0, "f32")
    hit = np.zeros(got.shape, bool)
    hit[:, 2:, 37] = True
    assert (np.isnan(got[hit]) | (got[hit] == np.inf)).all() and (got[~hit] == before[~hit]).all() and (lse == lse0).all()
    assert (run_attn(q, cache, table, lens, 700, 0.1, 40, "f32")[0] == apart).all()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_attn_small_values(kind):
    """Values below the types' normal range count: keys and values around
    2^-20 (subnormal in f16), scores made of them."""
    rng = np.random.default_rng(6)
    lens = [150, 33]
    q, cache, table = attn_inputs(rng, lens, 4, 2, 64, kind, 16, "head")
    cache.k.mul_(2.0 ** -19)
    cache.v.mul_(2.0 ** -20)
    got, _ = run_attn(q, cache, table, lens, 150, 2.0 ** 17, 0, "f32")
    ref, size, _, top, seen = attn_ref(q.float().numpy(), cache, table, lens, 150, 2.0 ** 17, 0)
    # as in check_attn, without its allowance for the smallest output step
    prob = {"f16": 2.0 ** -21, "bf16": 2.0 ** -22}[kind]
    rel = 2 * (64 + 6) * U * top + 4 * U + prob + 2 * (seen[:, None] + 8) * U
    within(got, ref, rel[:, :, None] * size + U * np.abs(ref), kind)


def test_attn_offsets_past_32_bits():
    """A cache of more than 2^32 elements, the last pages in use."""
    d, page, hkv = 128, 16, 8
    n_pages = (1 << 32) // (page * hkv * d) + 100
    rng = np.random.default_rng(8)
    say(f"attn: {n_pages} pages, {2 * n_pages * page * hkv * d * 2 >> 30} GiB")
    cache = Cache(n_pages, hkv, page, d, "f16")
    lens = [33, 16 * 40]
    table = np.stack([np.arange(n_pages - 100, n_pages - 60), np.arange(n_pages - 40, n_pages)]).astype(np.int32)
    table[0, 0] = 1
    small = Cache(100, hkv, page, d, "f16", fill=lambda s: torch.from_numpy(
        rng.standard_normal(s).astype(np.float32)).to("cuda:0"))
    cache.k[-100:], cache.v[-100:] = small.k, small.v
    cache.k[1], cache.v[1] = small.k[0], small.v[0]
    q = torch.from_numpy(rng.standard_normal((2, 16, d)).astype(np.float32)).half()
    got, _ = run_attn(q, cache, table, lens, 640, 0.09, 0, "f32")
    low = np.maximum(table - (n_pages - 100), 0)
    want, _ = run_attn(q, small, low, lens, 640, 0.09, 0, "f32")
    assert_same(got, want, "the same pages low and high")
    # and the write into the last slots
    x = torch.randn(3, (2 + 2 * hkv) * d, device="cuda:0")
    slots = torch.tensor([n_pages * page - 1, 0, (n_pages - 1) * page], device="cuda:0")
    pos, out = torch.zeros(3, dtype=torch.int32, device="cuda:0"), empty((3, 2 * d), torch.float16)
    s2x.call("s2x_qk_norm_rope_kv", ptr(x), 0, x.shape[1], 3, 2, None, None, 0.0, None, 0, 0, ptr(pos), ptr(slots),
             ptr(out), 2 * d, cache.ref(), stream())
    assert torch.equal(cache.k[-1, :, -1], x[0, 2 * d:(2 + hkv) * d].view(hkv, d).half())
    assert torch.equal(cache.v[-1, :, 0], x[2, (2 + hkv) * d:].view(hkv, d).half())


def test_attn_repeats_and_streams():
    """The same call twice, with workspaces that held other values, on another
    stream, and two calls at once on two streams: the same bits."""
    rng = np.random.default_rng(21)
    lens = [3000, 40, 1, 2999]
    q, cache, table = attn_inputs(rng, lens, 8, 2, 128, "f16", 16, "head")
    a, la = run_attn(q, cache, table, lens, 3000, 0.09, 0, "f16")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    b, lb = run_attn(q, cache, table, lens, 3000, 0.09, 0, "f16", st=ctypes.c_void_p(s1.cuda_stream))
    assert_same(b, a, "other stream")
    assert_same(lb, la, "other stream lse")
    n, hq, d = q.shape
    qd, td, ld = q.reshape(n, -1).to("cuda:0"), dev(table), dev(np.asarray(lens, np.int32))
    size = s2x.lib.s2x_attn_paged_workspace_size(n, 3000, hq, 2, d)
    outs = []
    torch.cuda.synchronize()
    for i in range(8):
        out, ws = empty((n, hq * d), torch.float16), empty((max(size, 1),), torch.uint8)
        outs.append((out, ws))
    torch.cuda.synchronize()
    for i, (out, ws) in enumerate(outs):
        s2x.call("s2x_attn_paged", ptr(qd), hq * d, cache.ref(), ptr(td), table.shape[1], ptr(ld), n, 3000, hq, 0.09, 0,
                 ptr(out), CODES["f16"], hq * d, None, ptr(ws), size,
                 ctypes.c_void_p((s1, s2)[i % 2].cuda_stream))
    torch.cuda.synchronize()
    for out, _ in outs:
        assert_same(out.double().cpu().numpy().reshape(n, hq, d), a, "two streams at once")


# ---------------------------------------------------------------------------
# Q4_0 products
# ---------------------------------------------------------------------------
class Q4:
    def __init__(self, q, d, how="host"):
        self.n, self.k = q.shape
        self.h = ctypes.c_void_p()
        raw = q4_0_blocks(q, d)
        if how == "host":
            s2x.call("s2x_weight_q4_0_create", raw.ctypes.data, 1, self.k, self.n, stream(), ctypes.byref(self.h))
        elif how == "device":
            s2x.call("s2x_weight_q4_0_create", ptr(dev(raw)), 0, self.k, self.n, stream(), ctypes.byref(self.h))
        else:
            self.buf = empty((s2x.lib.s2x_weight_q4_0_bytes(self.k, self.n),), torch.uint8)
            self.raw = dev(raw)
            s2x.call("s2x_weight_q4_0_create_in", ptr(self.raw), self.k, self.n, ptr(self.buf), stream(),
                     ctypes.byref(self.h))

    def __del__(self):
        s2x.lib.s2x_weight_q4_0_destroy(self.h)


def q4_weight(rng, n, k):
    q = rng.integers(0, 16, (n, k)).astype(np.uint8)
    d = rng.normal(0, 0.01, (n, k // 32)).astype(np.float16)
    return q, d


def run_q4(w, qx, ds, m, epi=None, ldy=None, st=None):
    ldy = ldy or w.n
    y = torch.full((m, ldy), NAN, device="cuda:0")
    size = s2x.lib.s2x_mul_mat_q4_0_workspace_size(w.k, w.n, m)
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda:0") if size else None
    s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, ptr(qx), ptr(ds), m, ptr(y), ldy,
             None if epi is None else ctypes.byref(epi), ptr(ws), size, st or stream())
    g = host(y)
    assert np.isnan(g[:, w.n:]).all()
    return g[:, :w.n]


def q4_terms(q, dw, qx, dx):
    """The product in f64 and the sum of its terms' sizes."""
    n, k = q.shape
    w = ((q.astype(np.float64) - 8).reshape(n, k // 32, 32) * dw.astype(np.float64)[:, :, None]).reshape(n, k)
    x = (qx.astype(np.float64).reshape(len(qx), k // 32, 32) * dx.astype(np.float64)[:, :, None]).reshape(len(qx), k)
    # sizes block by block: the block dots are exact
    i = np.einsum("mbk,nbk->mnb", x.reshape(len(qx), k // 32, 32), w.reshape(n, k // 32, 32))
    return x @ w.T, np.abs(i).sum(2)


@pytest.mark.parametrize("m,k,n,how", [
    (1, 32, 1, "host"), (1, 64, 17, "device"), (1, 1152, 3456, "in"), (2, 96, 15, "host"), (3, 4320, 100, "host"),
    (7, 160, 33, "in"), (8, 1152, 64, "host"), (15, 288, 48, "host"), (16, 1024, 130, "device"),
    (17, 416, 19, "host"), (31, 2048, 16, "host"), (33, 4320, 65, "in"), (48, 992, 31, "host"),
    (64, 1152, 129, "host"), (100, 4096, 70, "host"), (208, 320, 270, "device"), (256, 96, 5200, "host"), (33, 4128, 3000, "device"),
    (17, 1024, 9000, "host"), (4, 512, 5000, "device"), (50, 256, 9000, "device"), (1, 8192, 40, "host"), (64, 32, 3, "host"), (2, 128, 70000, "device"), (5, 11040, 21, "host")])
def test_q4_few_rows(m, k, n, how):
    rng = np.random.default_rng(m * 31 + k + n)
    say(f"q4: {m} x {k} x {n} ({how})")
    q, dw = q4_weight(rng, n, k)
    qx, ds, dx = q8_1_planes(rng, m, k)
    w = Q4(q, dw, how)
    assert s2x.lib.s2x_weight_q4_0_k(w.h) == k and s2x.lib.s2x_weight_q4_0_n(w.h) == n
    qd, dd = dev(qx), dev(ds)
    ref, size = q4_terms(q, dw, qx, dx)
    # a block's term is rounded twice and added once, the ranges of K are
    # joined by at most 16 additions
    tol = (k // 32 + 20) * U * size + 1e-30
    y = run_q4(w, qd, dd, m)
    within(y, ref, tol, "y")
    # one row alone: the same bits
    r = m // 2
    assert_same(run_q4(w, qd[r:r + 1].contiguous(), dd[r:r + 1].contiguous(), 1)[0], y[r], "row alone")
    bias, resid = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n + 3)).astype(np.float32)
    bd, rd = dev(bias), dev(resid)
    e = s2x.Epilogue(kind=s2x.EPI_BIAS, bias=bd.data_ptr())
    yb = run_q4(w, qd, dd, m, e, ldy=n + 5)
    assert_same(yb, y + bias, "bias")
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_RESID, bias=bd.data_ptr(), resid=rd.data_ptr(), ld_resid=n + 3)
    assert_same(run_q4(w, qd, dd, m, e), (y + bias) + resid[:, :n], "residual")
    e.resid_rows = 1
    assert_same(run_q4(w, qd, dd, m, e), (y + bias) + resid[:1, :n], "residual of one row")
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_GELU, bias=bd.data_ptr())
    g = run_q4(w, qd, dd, m, e)
    v = (y + bias).astype(np.float64)
    want = v / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    # (the exponent's 4 roundings grow with it, at most 87)
    within(g, want, (16 + 8 * np.abs(v) * (1 + 0.05 * v * v)) * U * np.abs(want) + 1e-35, "gelu")


@pytest.mark.parametrize("m,k,n", [(257, 1152, 200), (257, 4320, 96), (300, 64, 1000), (270, 32, 1),
                                   (257, 416, 129)])
def test_q4_many_rows(m, k, n):
    """Past the few-rows limit: the bits of the Q8_0 product of the same
    weight."""
    rng = np.random.default_rng(m + k)
    q, dw = q4_weight(rng, n, k)
    qx, ds, _ = q8_1_planes(rng, m, k)
    w, qd, dd = Q4(q, dw), dev(qx), dev(ds)
    bias = dev(rng.standard_normal(n).astype(np.float32))
    h = ctypes.c_void_p()
    raw8 = q8_0_blocks(q, dw)
    s2x.call("s2x_weight_create", raw8.ctypes.data, 1, k, n, stream(), ctypes.byref(h))
    for kind in (s2x.EPI_NONE, s2x.EPI_BIAS_GELU):
        e = s2x.Epilogue(kind=kind, bias=bias.data_ptr())
        y8 = empty((m, n), torch.float32)
        s2x.call("s2x_mul_mat_q8_0_q8_1", h, ptr(qd), ptr(dd), m, ptr(y8), n, ctypes.byref(e), stream())
        assert_same(run_q4(w, qd, dd, m, e), host(y8), f"m={m} kind {kind}")
    s2x.lib.s2x_weight_destroy(h)


@pytest.mark.parametrize("m,k,n", [(2, 128, 20), (7, 256, 20), (40, 1024, 6000)])
def test_q4_extremes(m, k, n):
    """Largest quants against largest nibbles (|I| = 32 * 8 * 128), zero and
    negative scales, residual in place, no rows."""
    q = np.zeros((n, k), np.uint8)  # -8
    q[1] = 15
    dw = np.ones((n, k // 32), np.float16)
    dw[2], dw[3] = 0, -1
    qx = np.full((m, k), -128, np.int8)
    qx[1] = 127
    dx = np.ones((m, k // 32), np.float16)
    ds = dx.view(np.uint16).astype(np.uint32)
    w, qd, dd = Q4(q, dw), dev(qx), dev(ds)
    y = run_q4(w, qd, dd, m)
    ref, _ = q4_terms(q, dw, qx, dx)
    assert_same(y, ref.astype(np.float32), "exact in f32")
    yr = dev(np.arange(m * n, dtype=np.float32).reshape(m, n))
    zero = dev(np.zeros(n, np.float32))
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_RESID, bias=zero.data_ptr(), resid=yr.data_ptr(), ld_resid=n)
    s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, ptr(qd), ptr(dd), m, ptr(yr), n, ctypes.byref(e), None, 0, stream())
    assert_same(host(yr), y + np.arange(m * n, dtype=np.float32).reshape(m, n), "in place")
    s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, None, None, 0, ptr(yr), n, None, None, 0, stream())


@pytest.mark.parametrize("m,k,n", [(9, 256, 40), (40, 1024, 6000)])
def test_q4_scales_out_of_the_normal_range(m, k, n):
    """Subnormal f16 scales on both sides count; a row whose scales are NaN or
    infinite, a column whose scale is, leave the others alone."""
    rng = np.random.default_rng(12)
    q, dw = q4_weight(rng, n, k)
    qx, ds, dx = q8_1_planes(rng, m, k)
    dw[:] = (rng.integers(1, 900, dw.shape) * 2.0 ** -24).astype(np.float16)
    dx[:4] = (rng.integers(1, 900, dx[:4].shape) * 2.0 ** -24).astype(np.float16)
    ref, size = q4_terms(q, dw, qx, dx)
    word = lambda d: dev(np.ascontiguousarray(d).view(np.uint16).astype(np.uint32))
    qd = dev(qx)
    w = Q4(q, dw)
    y = run_q4(w, qd, word(dx), m)
    within(y, ref, (k // 32 + 20) * U * size, "subnormal scales")
    bad = dx.copy()
    bad[2, 1], bad[5, 0] = np.nan, np.inf
    keep = [i for i in range(m) if i not in (2, 5)]
    z = run_q4(w, qd, word(bad), m)
    assert_same(z[keep], y[keep], "rows beside NaN and inf")
    assert np.isnan(z[2]).all() and not np.isfinite(z[5]).any()
    dw2 = dw.copy()
    dw2[7, 3] = np.inf
    z = run_q4(Q4(q, dw2), qd, word(dx), m)
    cols = [c for c in range(n) if c != 7]
    assert_same(z[:, cols], y[:, cols], "columns beside inf")
    assert not np.isfinite(z[:, 7]).any()


def test_q4_two_streams_at_once():
    """Calls on two streams, one weight, buffers of their own; past the
    few-rows limit each with its workspace."""
    rng = np.random.default_rng(13)
    k, n = 1024, 1300
    w = Q4(*q4_weight(rng, n, k))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for m in (3, 20, 130, 270):
        sets = []
        for i in range(6):
            qx, ds, _ = q8_1_planes(rng, m, k)
            size = s2x.lib.s2x_mul_mat_q4_0_workspace_size(k, n, m)
            sets.append((dev(qx), dev(ds), empty((m, n), torch.float32), empty((max(size, 1),), torch.uint8), size))
        torch.cuda.synchronize()
        for i, (qx, ds, y, ws, size) in enumerate(sets):
            s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, ptr(qx), ptr(ds), m, ptr(y), n, None, ptr(ws), size,
                     ctypes.c_void_p(streams[i % 2].cuda_stream))
        torch.cuda.synchronize()
        for qx, ds, y, _, _ in sets:
            assert_same(host(y), run_q4(w, qx, ds, m), f"m={m}")


# ---------------------------------------------------------------------------
# the step as a whole
# ---------------------------------------------------------------------------
class Step:
    """One layer's attention for B sequences' new tokens: slots, the QKV
    product, norms + rotation + cache, attention, the quantizer and the output
    product, over buffers that stay."""

    def __init__(self, n_seq, hq, hkv, d, hidden, page, max_len, kind="f16"):
        rng = np.random.default_rng(77)
        self.n_seq, self.hq, self.hkv, self.d, self.hidden, self.page, self.max_len = (n_seq, hq, hkv, d, hidden, page,
                                                                                       max_len)
        self.wide = (hq + 2 * hkv) * d
        self.qkv, self.o = (Q4(*q4_weight(rng, n, k)) for n, k in ((self.wide, hidden), (hidden, hq * d)))
        per = -(-max_len // page)
        self.cache = Cache(n_seq * per, hkv, page, d, kind)
        self.free = dev(rng.permutation(n_seq * per).astype(np.int32))
        self.table = torch.full((n_seq, per), -1, dtype=torch.int32, device="cuda:0")
        self.wq, self.wk = (dev(rng.normal(1, 0.1, d).astype(np.float32)) for _ in range(2))
        self.freq = dev(10000.0 ** (-np.arange(0, d, 2) / d))
        i32, i64 = torch.int32, torch.int64
        self.x = torch.zeros(n_seq, hidden, device="cuda:0")
        self.len, self.new = (torch.zeros(n_seq, dtype=i32, device="cuda:0") for _ in range(2))
        self.len_out, self.start, self.pos = (empty((n_seq + i,), i32) for i in (0, 1, 0))
        self.slots, self.used = empty((n_seq,), i64), empty((2,), i64)
        self.y, self.q = empty((n_seq, self.wide), torch.float32), empty((n_seq, hq * d), TYPES[kind])
        self.ctx, self.out = empty((n_seq, hq * d), torch.float32), empty((n_seq, hidden), torch.float32)
        self.planes = [(empty((n_seq, k), torch.int8), empty((n_seq, k // 32), i32)) for k in (hidden, hq * d)]
        size = s2x.lib.s2x_attn_paged_workspace_size(n_seq, max_len, hq, hkv, d)
        self.ws, self.ws_size = empty((max(size, 1),), torch.uint8), size

    def run(self):
        st, n = stream(), self.n_seq
        (q0, d0), (q1, d1) = self.planes
        h = self.hq * self.d
        s2x.call("s2x_kv_slots", ptr(self.len), ptr(self.new), n, ptr(self.free), self.free.numel(), self.page,
                 self.cache.n_pages, ptr(self.table), self.table.shape[1], n, ptr(self.len_out), ptr(self.start),
                 ptr(self.pos), ptr(self.slots), ptr(self.used), st)
        s2x.call("s2x_quantize_q8_1", ptr(self.x), self.hidden, n, self.hidden, self.hidden, ptr(q0), ptr(d0), st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.qkv.h, ptr(q0), ptr(d0), n, ptr(self.y), self.wide, None, None, 0, st)
        s2x.call("s2x_qk_norm_rope_kv", ptr(self.y), 0, self.wide, n, self.hq, ptr(self.wq), ptr(self.wk), 1e-6,
                 ptr(self.freq), self.d, 0, ptr(self.pos), ptr(self.slots), ptr(self.q), h, self.cache.ref(), st)
        s2x.call("s2x_attn_paged", ptr(self.q), h, self.cache.ref(), ptr(self.table), self.table.shape[1],
                 ptr(self.len_out), n, self.max_len, self.hq, self.d ** -0.5, 0, ptr(self.ctx), 0, h, None,
                 ptr(self.ws), self.ws_size, st)
        s2x.call("s2x_quantize_q8_1", ptr(self.ctx), h, n, h, h, ptr(q1), ptr(d1), st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.o.h, ptr(q1), ptr(d1), n, ptr(self.out), self.hidden, None, None, 0, st)

    def advance(self):
        """The host's side of a step: lengths on, taken pages off."""
        taken = int(self.used[0])
        self.free = torch.cat([self.free[taken:], self.free[:taken]])
        self.len.copy_(self.len_out)


def test_step_from_empty_caches():
    """Forty steps of three sequences, one of them idle every third step: the
    new tokens' places, keys and context against 64 bits."""
    s = Step(3, 8, 2, 64, 288, 16, 64)
    rng = np.random.default_rng(4)
    lens = np.zeros(3, np.int64)
    for i in range(40):
        new = np.array([1, 1, 0 if i % 3 == 2 else 1])
        s.x.copy_(dev(rng.standard_normal((3, 288)).astype(np.float32)))
        s.new.copy_(dev(new.astype(np.int32)))
        before = s.cache.k.clone()
        s.run()
        torch.cuda.synchronize()
        rows = np.flatnonzero(new)  # row t of the step is the t-th active sequence
        # (the idle sequence brings no row: the batch is packed)
        pos, slots, table = host(s.pos), host(s.slots), host(s.table)
        assert pos[:len(rows)].tolist() == lens[rows].tolist() and (slots[len(rows):] == -1).all()
        for t, b in enumerate(rows):
            assert slots[t] == table[b, lens[b] // 16] * 16 + lens[b] % 16
        y = host(s.y)
        _, (k, ks), (v, _) = heads_ref(y, 8, 2, 64, host(s.wq), host(s.wk), 1e-6, host(s.freq), 64, "half", pos)
        for t in range(len(rows)):
            got = s.cache.k[slots[t] // 16, :, slots[t] % 16].double().cpu().numpy()
            within(got, k[t], 2.0 ** -11 * np.abs(k[t]) + 32 * U * ks[t] + 2.0 ** -25, f"step {i} key {t}")
        changed = (s.cache.k.view(torch.int16) != before.view(torch.int16)).any(-1).any(1).sum()
        assert int(changed) == len(rows)
        lens = lens + new
        # context: the query rows belong to the sequences in order only when
        # all are active; then every row is checked
        if len(rows) == 3:
            ref, size, _, top, _ = attn_ref(host(s.q.float()).reshape(3, 8, 64), s.cache, table, lens, 64, 0.125, 0)
            tol = (2 * 70 * U * top + 2.0 ** -20 + 2 * (lens.max() + 8) * U)[:, :, None] * size
            within(host(s.ctx).reshape(3, 8, 64), ref, tol, f"step {i} context")
        s.advance()
    assert host(s.len).tolist() == lens.tolist()


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_step_captured(kind):
    """The step in a graph, replayed over new inputs and lengths with eager
    work between the replays: every replay's outputs and cache equal those of
    eager calls on buffers of their own."""
    a, b = (Step(5, 8, 2, 128, 1152, 16, 400, kind) for _ in range(2))
    for s in (a, b):
        s.cache.mem[0].zero_()
        s.cache.mem[1].zero_()
        s.new.fill_(1)
    free = a.free.clone()  # the graph holds this address: pages are moved within it
    a.free = b.free = free
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a.run()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.run()
    a.table.fill_(-1)
    a.cache.mem[0].zero_()
    a.cache.mem[1].zero_()
    rng = np.random.default_rng(9)
    lens = np.array([0, 15, 16, 200, 350])
    per = -(-lens // 16)
    table = np.full((5, 25), -1, np.int32)
    order, at = rng.permutation(125).astype(np.int32), 0
    for i in range(5):
        table[i, :per[i]] = order[at:at + per[i]]
        at += per[i]
    free.copy_(dev(np.concatenate([order[at:], order[:at]])))
    for s in (a, b):
        s.len.copy_(dev(lens.astype(np.int32)))
        s.table.copy_(dev(table))
    for m0, m1 in zip(a.cache.mem, b.cache.mem):
        m0.copy_(torch.randn(m0.shape, device="cuda:0"))
        m1.copy_(m0)
    for i in range(6):
        x = dev(rng.standard_normal((5, 1152)).astype(np.float32))
        for s in (a, b):
            s.x.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        b.run()
        torch.cuda.synchronize()
        for name in ("out", "ctx", "q", "y", "pos", "slots", "table", "len_out", "used"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (i, name)
        for m0, m1 in zip(a.cache.mem, b.cache.mem):
            assert torch.equal(m0, m1), i
        taken = int(a.used[0])
        free.copy_(torch.roll(free, -taken))
        for s in (a, b):
            s.len.copy_(s.len_out)
        torch.randn(1000, 1000, device="cuda:0").sum()  # eager work between replays
