"""Calls of the decode step that its documentation allows and that lie apart
from the ordinary ones: sizes past a kernel's reach, epilogues past the few-rows
limit, idle sequences, shortages."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import q8_1_planes
from gpu_util import assert_same, dev, empty, host, ptr, say, stream
from test_gpu_decode import NAN, U, Q4, q4_terms, q4_weight, run_q4, within

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
