"""Calls of the decode step that its documentation allows and that lie apart
from the ordinary ones: sizes past a kernel's reach, epilogues past the few-rows
limit, idle sequences, shortages."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import CODES, HALF_STEP, TYPES, Cache, attn_ref, q8_1_planes, slots_ref
from gpu_util import assert_same, dev, empty, host, ptr, say, stream
from test_gpu_decode import (NAN, U, Q4, Step, attn_inputs, check_slots, q4_terms, q4_weight, run_attn, run_q4,
                             run_slots, slots_case, within)

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# Q4_0 products past the int8 GEMM's reach
# ---------------------------------------------------------------------------
def test_q4_rows_of_y_far_apart():
    """257 rows of y 2^22 floats apart: the values of f64, each row with the bits
    it has alone, nothing between the rows."""
    rng = np.random.default_rng(31)
    m, k, n, ldy = 257, 416, 200, 1 << 22
    q, dw = q4_weight(rng, n, k)
    qx, ds, dx = q8_1_planes(rng, m, k)
    w, qd, dd = Q4(q, dw), dev(qx), dev(ds)
    y = torch.full((m, ldy), NAN, device="cuda:0")
    size = s2x.lib.s2x_mul_mat_q4_0_workspace_size(k, n, m)
    ws = empty((max(size, 1),), torch.uint8)
    say(f"q4: {m} x {k} x {n}, ldy 2^22")
    s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, ptr(qd), ptr(dd), m, ptr(y), ldy, None, ptr(ws), size, stream())
    got = host(y[:, :n])
    ref, terms = q4_terms(q, dw, qx, dx)
    within(got, ref, (k // 32 + 20) * U * terms + 1e-30, "y")
    for r in (0, 128, 256):
        assert_same(run_q4(w, qd[r:r + 1].contiguous(), dd[r:r + 1].contiguous(), 1)[0], got[r], f"row {r} alone")
    assert bool(torch.isnan(y[:, n:]).all())


def test_q4_widest_weights():
    """More than 2^22 columns at 257 rows, no workspace: the last columns
    against f64, one row against the call of that row."""
    m, k, n = 257, 32, (1 << 22) + 3
    g = torch.Generator(device="cuda:0")
    g.manual_seed(5)
    raw = torch.randint(0, 256, (n, 18), generator=g, device="cuda:0", dtype=torch.int16).to(torch.uint8)
    dw = (torch.rand(n, generator=g, device="cuda:0") * 0.02).half()
    raw[:, :2] = dw.view(torch.uint8).view(n, 2)
    h = ctypes.c_void_p()
    s2x.call("s2x_weight_q4_0_create", ptr(raw), 0, k, n, stream(), ctypes.byref(h))
    rng = np.random.default_rng(6)
    qx, ds, dx = q8_1_planes(rng, m, k)
    qd, dd, y = dev(qx), dev(ds), empty((m, n), torch.float32)
    say(f"q4: {m} x {k} x {n}")
    s2x.call("s2x_mul_mat_q4_0_q8_1", h, ptr(qd), ptr(dd), m, ptr(y), n, None, None, 0, stream())
    one = empty((1, n), torch.float32)
    s2x.call("s2x_mul_mat_q4_0_q8_1", h, ptr(qd[200:201].contiguous()), ptr(dd[200:201].contiguous()), 1, ptr(one), n,
             None, None, 0, stream())
    assert torch.equal(y[200], one[0])
    last = host(raw[-100:])
    q = np.concatenate([last[:, 2:] & 15, last[:, 2:] >> 4], 1)
    ref, terms = q4_terms(q, host(dw[-100:])[:, None], qx, dx)
    within(host(y[:, -100:]), ref, 21 * U * terms + 1e-30, "last columns")
    s2x.lib.s2x_weight_q4_0_destroy(h)


def test_q4_residual_past_two_gib():
    """A residual of 3 GB that wraps, over more rows than one launch takes: the
    row of the residual is the row of the whole call."""
    rng = np.random.default_rng(32)
    m, k, n, rows, ld = 2100, 64, 40, 1500, 1 << 19
    q, dw = q4_weight(rng, n, k)
    qx, ds, dx = q8_1_planes(rng, m, k)
    w, qd, dd = Q4(q, dw), dev(qx), dev(ds)
    bias, resid = rng.standard_normal(n).astype(np.float32), rng.standard_normal((rows, n)).astype(np.float32)
    bd, rd = dev(bias), torch.full((rows, ld), NAN, device="cuda:0")
    rd[:, :n] = dev(resid)
    say(f"q4: {m} x {k} x {n}, residual of {rows} rows 2^19 apart")
    parts = np.concatenate([run_q4(w, qd[a:a + 256].contiguous(), dd[a:a + 256].contiguous(), len(qx[a:a + 256]))
                            for a in range(0, m, 256)])
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_RESID, bias=bd.data_ptr(), resid=rd.data_ptr(), ld_resid=ld, resid_rows=rows)
    assert_same(run_q4(w, qd, dd, m, e), (parts + bias) + resid[np.arange(m) % rows], "y")


# ---------------------------------------------------------------------------
# attention over packed rows
# ---------------------------------------------------------------------------
def run_rows(q, starts, cache, table, lens, max_len, scale, window, out_kind, lse=True):
    """q (rows, hq, d) packed; rows of out and lse start as NaNs."""
    n_row, hq, d = q.shape
    n = len(lens)
    out = torch.full((n_row, hq, d), NAN, dtype=TYPES[out_kind], device="cuda:0")
    ls = torch.full((n_row, hq), NAN, device="cuda:0") if lse else None
    qd, td, ld, sd = q.to("cuda:0"), dev(table), dev(np.asarray(lens, np.int32)), dev(np.asarray(starts, np.int32))
    assert len(starts) == n + 1
    size = s2x.lib.s2x_attn_paged_workspace_size(n, max_len, hq, cache.n_head, d)
    ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda:0")
    s2x.call("s2x_attn_paged_rows", ptr(qd), hq * d, n_row, ptr(sd), cache.ref(), ptr(td), table.shape[1], ptr(ld), n,
             max_len, hq, scale, window, ptr(out), CODES[out_kind], hq * d, ptr(ls), ptr(ws), size, stream())
    torch.cuda.synchronize()
    return out.double().cpu().numpy(), None if ls is None else host(ls)


@pytest.mark.parametrize("lens,news,hq,hkv,d,kind,out_kind,window,pad", [
    ([40, 7, 12], [1, 0, 1], 4, 2, 64, "f16", "f16", 0, 1),
    ([0, 7, 0, 300], [0, 0, 0, 0], 4, 2, 64, "f16", "f32", 0, 3),
    ([300, 0, 129, 5, 200], [0, 0, 1, 5, 90], 16, 16, 72, "f16", "f32", 0, 0),
    ([3000, 17, 2999, 64], [1, 17, 0, 1], 8, 2, 128, "bf16", "bf16", 0, 2),      # several chunks
    ([9000, 4000], [0, 33], 4, 1, 128, "f16", "f32", 700, 5),
    ([513, 64, 65, 1], [2, 0, 1, 0], 34, 2, 80, "bf16", "f32", 0, 0),
    ([1021] * 16, [1, 0] * 8, 8, 8, 64, "f16", "f16", 100, 8)])
def test_attn_rows(lens, news, hq, hkv, d, kind, out_kind, window, pad):
    """Packed rows: each sequence's last row has the bits that its query has
    where row s is sequence s's; all other rows stay."""
    say(f"attn rows: lens {lens} new {news} {hq}/{hkv} x {d} {kind}->{out_kind}")
    rng = np.random.default_rng(sum(lens) + 3)
    _, cache, table = attn_inputs(rng, lens, hq, hkv, d, kind, 16, "head")
    starts = np.concatenate([[0], np.cumsum(news)])
    n_row = int(starts[-1]) + pad
    q = torch.from_numpy(rng.standard_normal((n_row, hq, d)).astype(np.float32)).to(TYPES[kind])
    got, lse = run_rows(q, starts, cache, table, lens, max(lens), d ** -0.5, window, out_kind)
    last = np.maximum(starts[1:] - 1, 0)
    want, wlse = run_attn(q[last], cache, table, lens, max(lens), d ** -0.5, window, out_kind)
    brings = np.flatnonzero(news)
    assert_same(got[last[brings]], want[brings], "out")
    assert_same(lse[last[brings]], wlse[brings], "lse")
    others = np.setdiff1d(np.arange(n_row), last[brings])
    assert np.isnan(got[others]).all() and np.isnan(lse[others]).all()
    again, _ = run_rows(q, starts, cache, table, lens, max(lens), d ** -0.5, window, out_kind, lse=False)
    assert_same(again[last[brings]], want[brings], "without lse")


@pytest.mark.parametrize("length", [200, 5000])
def test_attn_rows_bad_starts(length):
    """Starts that are no rows of q (negative, falling, past its end): those
    sequences are left out, the others are not."""
    rng = np.random.default_rng(length)
    lens = [length, 30, 20, length, 8, 9]
    _, cache, table = attn_inputs(rng, lens, 4, 2, 64, "f16", 16, "head")
    q = torch.from_numpy(rng.standard_normal((6, 4, 64)).astype(np.float32)).half()
    starts = [-2 ** 31, -3, 2, 1, 5, 7, 2 ** 31 - 1]  # (only sequence 3, row 4, is whole and inside)
    got, lse = run_rows(q, starts, cache, table, lens, length, 0.125, 0, "f32")
    want, _ = run_attn(q[[4] * 6], cache, table, lens, length, 0.125, 0, "f32")
    assert_same(got[4], want[3], "row 4")
    assert np.isnan(np.delete(got, 4, 0)).all() and np.isnan(np.delete(lse, 4, 0)).all()
    starts = [0, 1, 1, 2, 2 ** 31 - 1, -1, 4]
    got, _ = run_rows(q, starts, cache, table, lens, length, 0.125, 0, "f32")
    want, _ = run_attn(q[[0, 0, 1, 1, 1, 1]], cache, table, lens, length, 0.125, 0, "f32")
    assert_same(got[:2], want[[0, 2]], "rows 0 and 1")
    assert np.isnan(got[2:]).all()


class PackedStep(Step):
    """The step as documented, for batches in which a sequence may be idle."""

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
        s2x.call("s2x_attn_paged_rows", ptr(self.q), h, n, ptr(self.start), self.cache.ref(), ptr(self.table),
                 self.table.shape[1], ptr(self.len_out), n, self.max_len, self.hq, self.d ** -0.5, 0, ptr(self.ctx), 0, h,
                 None, ptr(self.ws), self.ws_size, st)
        s2x.call("s2x_quantize_q8_1", ptr(self.ctx), h, n, h, h, ptr(q1), ptr(d1), st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.o.h, ptr(q1), ptr(d1), n, ptr(self.out), self.hidden, None, None, 0, st)


def check_context(s, lens, new, kind, what):
    """The context of every sequence that brought a token, against 64 bits; rows
    behind the last token as they were."""
    rows = np.flatnonzero(new)
    hq, d = s.hq, s.d
    q = np.zeros((s.n_seq, hq, d), np.float32)
    q[rows] = host(s.q.float()).reshape(-1, hq, d)[:len(rows)]
    ref, size, _, top, _ = attn_ref(q, s.cache, host(s.table), lens, s.max_len, d ** -0.5, 0)
    # a score's d products and two scalings, a probability's terms of the
    # cache's type, the two sums
    tol = (2 * (d + 6) * U * top + {"f16": 2.0 ** -20, "bf16": 2.0 ** -21}[kind] + 2 * (lens.max() + 8) * U)[:, :, None] * size
    ctx = host(s.ctx).reshape(-1, hq, d)
    within(ctx[:len(rows)], ref[rows], tol[rows], what)
    assert (ctx[len(rows):] == 7.0).all(), what


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_step_with_idle_sequences(kind):
    """Thirty steps of four sequences, each idle now and then, all of them
    once: every active sequence's context is that of its own query."""
    s = PackedStep(4, 8, 2, 64, 288, 16, 64, kind)
    rng = np.random.default_rng(14)
    lens = np.zeros(4, np.int64)
    for i in range(30):
        new = np.zeros(4, int) if i == 11 else (rng.random(4) < 0.6).astype(int)
        s.x.copy_(dev(rng.standard_normal((4, 288)).astype(np.float32)))
        s.new.copy_(dev(new.astype(np.int32)))
        s.ctx.fill_(7.0)
        s.run()
        lens = lens + new
        check_context(s, lens, new, kind, f"step {i}, new {new}")
        s.advance()
    assert host(s.len).tolist() == lens.tolist()


def test_captured_step_with_idle_sequences():
    """The same step in a graph: which sequences are idle is read anew at each
    replay."""
    s = PackedStep(5, 8, 2, 128, 1152, 16, 400)
    rng = np.random.default_rng(15)
    for m in s.cache.mem:
        m.zero_()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        s.run()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    s.table.fill_(-1)
    lens, free = np.zeros(5, np.int64), s.free
    for i in range(25):
        new = (rng.random(5) < 0.7).astype(int)
        s.x.copy_(dev(rng.standard_normal((5, 1152)).astype(np.float32)))
        s.new.copy_(dev(new.astype(np.int32)))
        s.ctx.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        lens = lens + new
        check_context(s, lens, new, "f16", f"replay {i}, new {new}")
        free.copy_(torch.roll(free, -int(s.used[0])))
        s.len.copy_(s.len_out)
        torch.randn(1000, 1000, device="cuda:0").sum()  # eager work between replays


# ---------------------------------------------------------------------------
# bits of the probabilities
# ---------------------------------------------------------------------------
def split_bf16(x, terms):
    """x (f64) as a sum of bf16 terms, each the nearest to what is left."""
    left, total = x.copy(), np.zeros_like(x)
    for _ in range(terms):
        t = torch.from_numpy(left.astype(np.float32)).bfloat16().double().numpy()
        total, left = total + t, left - t
    return total


@pytest.mark.parametrize("out_kind", ["bf16", "f32"])
@pytest.mark.parametrize("max_len", [3, 4000])
def test_attn_bf16_probabilities(out_kind, max_len):
    """A bf16 cache holds its probabilities in 24 bits whatever the output's
    type: three keys, two of score 0 with the first two bf16 terms of e as
    values, one of score ln e with -1, so that the sum is what two terms leave of
    e.  U of `size`, the sum of the terms' sizes: e is off by 2 of exp2 and 1.2 of
    its argument, half of the size; five sums of at most the size's half, 2 each
    where the matrix pipe cuts off.  10 in all, then the output's rounding."""
    rng = np.random.default_rng(41)
    n, d = 64, 64
    x = torch.from_numpy(rng.uniform(0.1, 0.6, n).astype(np.float32)).bfloat16().double().numpy()
    e = np.exp(-x)
    hi = split_bf16(e, 1)
    lo = split_bf16(e - hi, 1)
    cache = Cache(n, 1, 16, d, "bf16", fill=lambda s: torch.zeros(s, device="cuda:0"))
    sign = np.where(np.arange(d) % 3 == 1, -1.0, 1.0)
    cache.k[:, 0, 2, 0] = torch.from_numpy(-x).to("cuda:0", torch.bfloat16)
    for t, v in enumerate((hi, lo, -np.ones(n))):
        cache.v[:, 0, t] = torch.from_numpy(v[:, None] * sign).to("cuda:0", torch.bfloat16)
    q = torch.zeros(n, 1, d, dtype=torch.bfloat16)
    q[:, 0, 0] = 1
    table = np.zeros((n, max_len // 16 + 1), np.int32)
    table[:, 0] = np.arange(n)
    ref, size = (hi + lo - e) / (2 + e), (hi + np.abs(lo) + e) / (2 + e)
    tol = 10 * U * size + HALF_STEP[out_kind] * np.abs(ref) + 4 * U * np.abs(ref)
    assert (np.abs((hi + lo - split_bf16(e, 2)) / (2 + e) - ref) > tol).sum() >= 10  # two terms would not do
    got, _ = run_attn(q, cache, table, [3] * n, max_len, 1.0, 0, out_kind)
    within(got[:, 0], ref[:, None] * sign, tol[:, None] + np.zeros(d), f"{out_kind} max_len {max_len}")


# ---------------------------------------------------------------------------
# slots
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("n_seq,new,cached,ld", [
    (1000, 2 ** 31 - 1, 0, 2), (1, 2 ** 31 - 1, 5, 3), (1000, 2 ** 20, 1, 2), (8192, 2 ** 17, 0, 1), (1500, 2 ** 20, 3, 0)])
def test_slots_lengths_past_the_table(n_seq, new, cached, ld):
    """More new pages than the table or the free list hold, up to 2^31 of one token: the
    rows' entries within the table, and no time for those behind it (a thread a
    page would be 2 million rounds of a search)."""
    rng = np.random.default_rng(n_seq)
    table = np.full((n_seq, ld), -1, np.int32)
    if ld:
        table[:, :min(cached, ld)] = 7
    free = rng.permutation(3 * n_seq + 10)
    a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    run_slots([1], [1], [0], 1, 1, np.zeros((1, 1)), 1)
    torch.cuda.synchronize()
    say(f"slots: {n_seq} of {new} new tokens, table of {ld}")
    a.record()
    got = run_slots([cached] * n_seq, [new] * n_seq, free, 1, 3 * n_seq + 10, table, 50)
    b.record()
    torch.cuda.synchronize()
    assert a.elapsed_time(b) < 100, "milliseconds"
    want = table.copy()
    for s in range(n_seq):
        for i in range(cached, ld):
            f = s * new + i - cached
            if f < 2 ** 31 - 1:
                want[s, i] = free[f] if f < len(free) else -1
    assert_same(got[0], want, "table")
    assert got[1].tolist() == [min(cached + new, 2 ** 31 - 1)] * n_seq and got[5].tolist() == [n_seq * new] * 2
    assert got[2].tolist() == [0] + [50] * n_seq and got[3].tolist() == list(range(cached, cached + 50))
    slots = [int(want[0, i]) if i < ld else -1 for i in range(cached, cached + 50)]
    assert got[4].tolist() == slots


@pytest.mark.parametrize("short,lost", [(7, 0), (10 ** 6, 0), (0, 40), (9, 30)])
def test_slots_shortage_and_again(short, lost):
    """A call with too few pages or rows, then the same lengths again with
    enough, over the tables that the first one left: all outputs of a call that
    had enough from the start."""
    rng = np.random.default_rng(short % 97 + lost)
    kv_len, n_new, free, page, n_pages, table, rows = slots_case(rng, 20, 100, 50, 16)
    few = free[:max(0, len(free) - short)]
    first = run_slots(kv_len, n_new, few, page, n_pages, table, rows - 9 - lost if lost else rows)
    used = first[5].tolist()
    assert (used[0] > len(few)) == (short > 0) and used[1] == rows - 9
    again = run_slots(kv_len, n_new, free, page, n_pages, first[0], rows)
    whole = run_slots(kv_len, n_new, free, page, n_pages, table, rows)
    ref = slots_ref(kv_len, n_new, free, page, n_pages, table, rows)
    for name, a, w, r in zip(("table", "len", "start", "pos", "slots", "used"), again, whole, ref):
        assert_same(a, w, name)
        assert_same(a, r, name)
    assert (again[4][:used[1]] >= 0).all()


def test_slots_shortage_carried_on():
    """Carried on all the same, a missing page stays missing: its tokens have no
    slot, the pages behind it are given as ever."""
    table = np.array([[3, -1, -1], [5, -1, -1]], np.int32)
    got = run_slots([16, 16], [1, 1], [9], 16, 20, table, 2)  # one page for two
    assert got[0].tolist() == [[3, 9, -1], [5, -1, -1]] and got[4].tolist() == [9 * 16, -1]
    assert got[5].tolist() == [2, 2]
    check_slots(got[1], [1, 1], [8, 7], 16, 20, got[0], 2, "the next step")
    got = run_slots(got[1], [1, 16], [8, 7], 16, 20, got[0], 17)
    assert got[0].tolist() == [[3, 9, -1], [5, -1, 8]]
    assert got[4].tolist() == [9 * 16 + 1] + [-1] * 15 + [8 * 16]


# ---------------------------------------------------------------------------
# Q4_0 products past the few-rows limit
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("m,k,n", [(257, 1152, 200), (300, 416, 1027), (1000, 96, 129), (263, 4320, 33)])
def test_q4_many_rows_epilogues(m, k, n):
    """The expanded weight's product against f64 and every epilogue on its bits:
    bias, GELU, residual (strided, wrapped, in place), rows of y with a gap."""
    rng = np.random.default_rng(m + n)
    say(f"q4: {m} x {k} x {n}")
    q, dw = q4_weight(rng, n, k)
    qx, ds, dx = q8_1_planes(rng, m, k)
    w, qd, dd = Q4(q, dw), dev(qx), dev(ds)
    ref, terms = q4_terms(q, dw, qx, dx)
    y = run_q4(w, qd, dd, m, ldy=n + 7)
    # a block's term is rounded twice and added once
    within(y, ref, (k // 32 + 4) * U * terms + 1e-30, "y")
    bias, resid = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n + 3)).astype(np.float32)
    bd, rd = dev(bias), dev(resid)
    e = s2x.Epilogue(kind=s2x.EPI_BIAS, bias=bd.data_ptr())
    assert_same(run_q4(w, qd, dd, m, e, ldy=n + 1), y + bias, "bias")
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_RESID, bias=bd.data_ptr(), resid=rd.data_ptr(), ld_resid=n + 3)
    assert_same(run_q4(w, qd, dd, m, e, ldy=n + 5), (y + bias) + resid[:, :n], "residual")
    for rows in (1, 100):
        e.resid_rows = rows
        assert_same(run_q4(w, qd, dd, m, e), (y + bias) + resid[np.arange(m) % rows, :n], f"residual of {rows} rows")
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_GELU, bias=bd.data_ptr())
    g = run_q4(w, qd, dd, m, e, ldy=n + 2)
    v = (y + bias).astype(np.float64)
    want = v / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    # (the exponent's 4 roundings grow with it)
    within(g, want, (16 + 8 * np.abs(v) * (1 + 0.05 * v * v)) * U * np.abs(want) + 1e-35, "gelu")
    yr = dev(np.ascontiguousarray(resid[:, :n]))
    e = s2x.Epilogue(kind=s2x.EPI_BIAS_RESID, bias=bd.data_ptr(), resid=yr.data_ptr(), ld_resid=n)
    size = s2x.lib.s2x_mul_mat_q4_0_workspace_size(k, n, m)
    ws = empty((size,), torch.uint8)
    s2x.call("s2x_mul_mat_q4_0_q8_1", w.h, ptr(qd), ptr(dd), m, ptr(yr), n, ctypes.byref(e), ptr(ws), size, stream())
    assert_same(host(yr), (y + bias) + resid[:, :n], "in place")


@pytest.mark.parametrize("from_host", [False, True])
def test_q4_weight_without_memory(from_host):
    """A weight that does not fit says so, and the calls after it are as ever: the
    refused allocation's error is not reported by the next launch."""
    k, n = 1 << 15, 1 << 18  # 4.8 GB of blocks, as much of planes
    rng = np.random.default_rng(3)
    small = Q4(*q4_weight(rng, 40, 64))
    qx, ds, _ = q8_1_planes(rng, 3, 64)
    qd, dd = dev(qx), dev(ds)
    before = run_q4(small, qd, dd, 3)
    raw = torch.empty(n * k // 32 * 18, dtype=torch.uint8, device="cpu" if from_host else "cuda:0")
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    say(f"free {free >> 20} MiB, all but 1 GiB taken")
    rest = torch.empty(free - (1 << 30), dtype=torch.uint8, device="cuda:0")
    h, y = ctypes.c_void_p(), empty((3, 40), torch.float32)
    status = s2x.lib.s2x_weight_q4_0_create(ptr(raw), int(from_host), k, n, stream(), ctypes.byref(h))
    after = s2x.lib.s2x_mul_mat_q4_0_q8_1(small.h, ptr(qd), ptr(dd), 3, ptr(y), 40, None, None, 0, stream())
    del rest
    torch.cuda.empty_cache()
    assert status == 5 and h.value is None, (status, s2x.lib.s2x_last_error())
    assert after == 0, s2x.lib.s2x_last_error()
    assert_same(host(y), before, "the next product")
