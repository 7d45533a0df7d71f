"""The beam search's operators on the GPU, each through the C-ABI against a plain
form in 64 bits.

Tolerances count roundings: u = 2^-24 for f32, half a step of the output's type
for the last rounding."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import CODES, HALF_STEP, TYPES, Cache, attn_ref
from gpu_util import assert_same, dev, empty, host, ptr, say, stream
from search_util import beam_scores, compact_ref, fork_ref
from test_gpu_decode import NAN, U, within

pytestmark = pytest.mark.gpu
INF = float("inf")


def nans(*shape, dtype=torch.float32):
    return torch.full(shape, NAN, dtype=dtype, device="cuda:0")


# ---------------------------------------------------------------------------
# residual, RMS norm, Q8_1
# ---------------------------------------------------------------------------
def run_rms(x, r, w, h_kind=None, out="q8", y_kind="f32", pads=(0, 0, 0, 0), eps=1e-6, in_place=None):
    """x (M, H), r or None: torch tensors on the host.  Returns h, y, (qs, ds)."""
    m, h = x.shape
    k_pad = -(-h // 32) * 32

    def rows(t, pad):
        if t is None:
            return None
        full = nans(m, h + pad, dtype=t.dtype)
        full[:, :h] = t.to("cuda:0")
        return full
    xd, rd = rows(x, pads[0]), rows(r, pads[1])
    kind = {v: k for k, v in TYPES.items()}
    rk = h_kind or (kind[r.dtype] if r is not None else "f32")
    ho = xd if in_place == "x" else rd if in_place == "r" else nans(m, h + pads[2], dtype=TYPES[rk])
    y = nans(m, h + pads[3], dtype=TYPES[y_kind]) if "y" in out else None
    qs = torch.full((m, k_pad), 77, dtype=torch.int8, device="cuda:0") if "q8" in out else None
    ds = torch.full((m, k_pad // 32), 77, dtype=torch.int32, device="cuda:0") if "q8" in out else None
    wd = None if w is None else dev(w)
    s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(xd), CODES[kind[x.dtype]], xd.shape[1], ptr(rd), CODES[rk],
             0 if rd is None else rd.shape[1], h, m, ptr(wd), eps, ptr(ho), ho.shape[1], k_pad, ptr(qs), ptr(ds), ptr(y),
             CODES[y_kind], 0 if y is None else y.shape[1], stream())
    torch.cuda.synchronize()
    if not in_place:
        assert torch.isnan(ho[:, h:]).all()
    if y is not None:
        assert torch.isnan(y[:, h:]).all()
        y = y[:, :h]
    return ho[:, :h], y, qs, ds


def check_rms(x, r, w, y_kind="f32", **kw):
    m, h = x.shape
    ho, y, qs, ds = run_rms(x, r, w, out="q8 y", y_kind=y_kind, **kw)
    s = x.float() if r is None else x.float() + r.float()
    assert torch.equal(ho.cpu(), s.to(ho.dtype)), "h"
    s = s.double().numpy()
    ref = s / np.sqrt((s * s).mean(1, keepdims=True) + float(np.float32(kw.get("eps", 1e-6)))) * (1.0 if w is None else w.astype(np.float64))
    # inv is rounded once (its f64 steps add less than 2^-40), then two products; where
    # those are subnormal a rounding is 2^-150 whatever the value, the first one's
    # then times w: (1 + |w|) 2^-150
    small = (1 + (1.0 if w is None else np.abs(w.astype(np.float64)))) * 2.0 ** -150
    within(y.double().cpu().numpy(), ref, (3.001 * U + HALF_STEP[y_kind]) * np.abs(ref) + small +
           (2.0 ** -25 if y_kind == "f16" else 0), "y")
    if y_kind != "f32":
        _, y, q2, d2 = run_rms(x, r, w, out="q8 y", **kw)
        assert torch.equal(q2, qs) and torch.equal(d2, ds)
    k_pad = qs.shape[1]
    q1, d1 = torch.empty_like(qs), torch.empty_like(ds)
    yc = y.contiguous()
    s2x.call("s2x_quantize_q8_1", ptr(yc), h, m, h, k_pad, ptr(q1), ptr(d1), stream())
    assert_same(host(qs), host(q1), "quants")
    assert_same(host(ds), host(d1), "scales")
    # either output alone has the same bits
    _, y2, _, _ = run_rms(x, r, w, out="y", **kw)
    assert torch.equal(y2, y)
    _, _, q2, d2 = run_rms(x, r, w, out="q8", **kw)
    assert torch.equal(q2, qs) and torch.equal(d2, ds)


def rms_case(seed, m, h, x_kind, r_kind):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.standard_normal((m, h)).astype(np.float32)).to(TYPES[x_kind])
    r = None if r_kind is None else torch.from_numpy(
        (rng.standard_normal((m, h)) * np.exp(rng.standard_normal(h))).astype(np.float32)).to(TYPES[r_kind])
    return x, r, rng.normal(1, 0.3, h).astype(np.float32)


@pytest.mark.parametrize("m,h,x_kind,r_kind,y_kind", [
    (1, 1152, "f32", "f32", "f32"), (1, 1, "f32", "f32", "f32"), (3, 7, "f16", "f16", "f16"), (2, 31, "bf16", "f32", "bf16"),
    (5, 32, "f32", None, "f16"), (5, 33, "bf16", "bf16", "f32"), (130, 4304, "f32", "f32", "bf16"),
    (9, 511, "f16", "f32", "f32"), (9, 512, "bf16", "bf16", "bf16"), (9, 513, "f32", "f32", "f32"),
    (7, 1023, "f16", None, "f16"), (7, 1025, "bf16", "f32", "f16"), (4, 2047, "f32", "f32", "f32"),
    (4, 2049, "bf16", "bf16", "bf16"), (4, 4096, "f16", "f16", "f32"), (3, 4097, "f32", None, "f32"),
    (3, 8192, "bf16", "f32", "f32"), (3, 8200, "f16", "f32", "f16"), (2, 16384, "f32", "f32", "bf16"),
    (2, 16390, "bf16", "bf16", "f32"), (2, 32768, "f16", "f16", "f16"), (2, 32767, "f32", "f32", "f32"),
    (5000, 300, "bf16", "bf16", "f32"), (2500, 1100, "f32", "f32", "f32")])
def test_rms(m, h, x_kind, r_kind, y_kind):
    say(f"rms: {m} x {h} {x_kind} + {r_kind} -> {y_kind}")
    check_rms(*rms_case(m + h, m, h, x_kind, r_kind), y_kind=y_kind)


def test_rms_strides_and_in_place():
    for x_kind, r_kind, pads in (("f32", "f32", (3, 5, 1, 7)), ("f16", "f16", (1, 3, 5, 9)), ("bf16", "f32", (8, 4, 0, 24))):
        x, r, w = rms_case(5, 11, 1157, x_kind, r_kind)
        check_rms(x, r, w, pads=pads)
        check_rms(x, r, None, pads=pads)
        check_rms(x, r, w, pads=(pads[0], pads[1], pads[1], 0), in_place="r")
        if x_kind == r_kind:
            check_rms(x, r, w, pads=(pads[0], pads[1], pads[0], 0), in_place="x")


def test_rms_special_values():
    """Zero rows, rows whose squares leave f32's range, subnormal rows, a large eps;
    NaNs and infinities stay in their rows, and Q8_1 takes them as its own entry does."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((9, 700)).astype(np.float32)
    x[1] = 0
    x[2] *= 1e30
    x[3] *= 1e-30
    x[4] *= 1e-42
    r = torch.zeros(9, 700)
    w = rng.normal(1, 0.2, 700).astype(np.float32)
    check_rms(torch.from_numpy(x), r, w)
    check_rms(torch.from_numpy(x), r, w, eps=100.0)
    x[2, :] = rng.standard_normal(700)
    x[5, 3], x[6, 9], x[7, 650] = np.nan, np.inf, -np.inf
    xt = torch.from_numpy(x)
    ho, y, qs, ds = run_rms(xt, r, w, out="q8 y")
    good = [0, 2, 3, 8]
    _, y2, q2, d2 = run_rms(xt[good], r[good], w, out="q8 y")
    assert torch.equal(y[good], y2) and torch.equal(qs[good], q2) and torch.equal(ds[good], d2)
    assert torch.isnan(y[5]).all() and torch.isnan(y[6, 9]) and torch.isnan(y[7, 650])
    assert (y[6, :9] == 0).all() and (y[7, :650] == 0).all()
    q1, d1 = torch.empty_like(qs), torch.empty_like(ds)
    s2x.call("s2x_quantize_q8_1", ptr(y.contiguous()), 700, 9, 700, 704, ptr(q1), ptr(d1), stream())
    assert torch.equal(qs, q1) and torch.equal(ds, d1)


# ---------------------------------------------------------------------------
# beam selection
# ---------------------------------------------------------------------------
def run_beam(logits, scores, n_out, done=None, done_token=1, pad=0, ws=None, st=None):
    """logits (n_req, n_beam, vocab) torch on the host."""
    n, beams, vocab = logits.shape
    x = nans(n * beams, vocab + pad, dtype=logits.dtype)
    x[:, :vocab] = logits.reshape(n * beams, vocab).to("cuda:0")
    sd, dd = dev(scores.astype(np.float32)), None if done is None else dev(done.astype(np.uint8))
    parent, token = (torch.full((n, n_out), -77, dtype=torch.int32, device="cuda:0") for _ in range(2))
    score = nans(n, n_out)
    size = s2x.lib.s2x_beam_select_workspace_size(n, beams, vocab, n_out)
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda:0") if ws is None else ws
    kind = {v: k for k, v in TYPES.items()}[logits.dtype]
    torch.cuda.synchronize()
    s2x.call("s2x_beam_select", ptr(x), CODES[kind], vocab + pad, n, beams, vocab, ptr(sd), ptr(dd), done_token, n_out,
             ptr(parent), ptr(token), ptr(score), ptr(ws), size, st or stream())
    return host(parent), host(token), host(score)


def check_beam(logits, scores, n_out, done=None, done_token=1, **kw):
    """Every place holds a candidate whose score is that place's, no candidate
    twice, and the very candidate wherever its neighbours are further off than
    the sum's error: of a lane's sum 128 additions at most, the exponentials 2 ulp,
    their arguments' 3 roundings of at most ln(vocab) on average."""
    parent, token, score = run_beam(logits, scores, n_out, done, done_token, **kw)
    n, beams, vocab = logits.shape
    x = logits.float().numpy()
    tol = (128 + 4 + 3 * np.log(vocab) + 40) * U
    for r in range(n):
        s = beam_scores(x[r], scores[r], None if done is None else done[r], done_token)
        flat = np.argsort(-s, axis=None, kind="stable")[:n_out + 1]
        best = s.flatten()[flat]
        got_s = np.full(n_out, -np.inf)
        for i in range(n_out):
            if i >= len(best) or best[i] == -np.inf:
                assert parent[r, i] == -1 and token[r, i] == -1 and score[r, i] == -np.inf, (r, i)
                continue
            b, t = parent[r, i] - r * beams, token[r, i]
            assert 0 <= b < beams and 0 <= t < vocab, (r, i, b, t)
            got_s[i] = s[b, t]
            want = best[i]
            assert abs(got_s[i] - want) <= 2 * tol, (r, i, got_s[i], want)
            assert abs(score[r, i] - want) <= 2 * tol + 2 * U * abs(want), (r, i, score[r, i], want)
            apart = [abs(want - best[j]) for j in (i - 1, i + 1) if 0 <= j < len(best)]
            # (equal ones of one beam, too: their order is the tokens')
            same = [flat[j] // vocab == flat[i] // vocab and best[j] == want for j in (i - 1, i + 1) if 0 <= j < len(best)]
            if all(a > 4 * tol or e for a, e in zip(apart, same)):
                assert (b, t) == divmod(int(flat[i]), vocab), (r, i)
        seen = [(int(p), int(t)) for p, t in zip(parent[r], token[r]) if p >= 0]
        assert len(set(seen)) == len(seen), r
        assert (np.diff(score[r][np.isfinite(score[r])]) <= 0).all(), r


def beam_case(seed, n, beams, vocab, kind, spread=2.0):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy((rng.standard_normal((n, beams, vocab)) * spread).astype(np.float32)).to(TYPES[kind])
    return x, -rng.uniform(2, 30, (n, beams)).astype(np.float32)


@pytest.mark.parametrize("n,beams,vocab,kind,n_out", [
    (1, 1, 1, "f32", 1), (1, 1, 1, "f16", 5), (2, 3, 7, "bf16", 4), (1, 4, 100, "f32", 64), (3, 4, 1000, "f32", 4),
    (2, 5, 2047, "f16", 10), (2, 5, 2049, "bf16", 10), (1, 64, 5000, "f32", 64), (1, 64, 3001, "bf16", 64),
    (1, 4, 32000, "f32", 4), (13, 5, 50021, "f16", 10), (2, 8, 256000, "bf16", 16), (60, 3, 8193, "f32", 6),
    (300, 2, 4099, "bf16", 3), (1, 1, 300001, "f16", 64), (1, 2, 1000003, "f32", 33), (700, 4, 257, "f16", 8)])
def test_beam(n, beams, vocab, kind, n_out):
    say(f"beam: {n} x {beams} x {vocab} {kind} -> {n_out}")
    check_beam(*beam_case(vocab + n, n, beams, vocab, kind), n_out, pad=3 if vocab % 2 else 0)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_beam_masks(kind):
    """Tokens of -inf, of the type's lowest value, whole rows of either; beams that
    have ended, beams with no finite score, rows with NaN or +inf."""
    x, s = beam_case(4, 6, 4, 3001, kind)
    low = torch.finfo(TYPES[kind]).min
    x[:, :, ::3] = -INF
    x[0, 1, 5:] = -INF          # two tokens left
    x[0, 2] = -INF              # nothing follows
    x[1, 0] = low               # all alike
    x[1, 1, 7:] = low
    x[1, 2, 100], x[1, 3, 2999] = NAN, INF
    x[2, :] = -INF
    x[2, 0, 17] = 3.0           # one candidate in all
    s[3, 1:] = -INF             # a search's first step
    s[4, 0], s[4, 1], s[4, 2] = NAN, INF, -INF
    done = np.zeros((6, 4), np.uint8)
    done[4, 2:] = 1             # (2: ended, but its score is none)
    done[5] = [1, 1, 0, 255]
    x[5, 0] = NAN               # an ended beam's logits are not read
    for n_out in (1, 4, 8, 40):
        check_beam(x, s, n_out, done, done_token=2)
        check_beam(x, s, n_out, None)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [50, 5000, 140000])
def test_beam_ties(kind, vocab):
    """Equal logits everywhere, equal beams, two values only: the lower beam, then the
    lower token."""
    x = torch.full((2, 3, vocab), 1.5).to(TYPES[kind])
    x[1, :, vocab // 3::7] = 2.5
    s = np.full((2, 3), -4.0, np.float32)
    for n_out in (3, 64):
        parent, token, score = run_beam(x, s, n_out)
        k = min(n_out, vocab)
        want = [(0, t) for t in range(vocab)][:n_out] + [(1, t) for t in range(max(0, n_out - vocab))]
        assert [(int(a), int(b)) for a, b in zip(parent[0], token[0])] == want, k
        high = list(range(vocab // 3, vocab, 7))
        low = sorted(set(range(vocab)) - set(high))
        want = ([(3 + b, t) for b in range(3) for t in high] + [(3 + b, t) for b in range(3) for t in low])[:n_out]
        assert [(int(a), int(b)) for a, b in zip(parent[1], token[1])] == want
    # zeros of either sign are one value
    x = torch.zeros(1, 2, vocab).to(TYPES[kind])
    x[0, :, ::2] = -0.0
    parent, token, _ = run_beam(x, s[:1, :2], 20)
    assert parent[0].tolist() == [0] * 20 and token[0].tolist() == list(range(20))


def test_beam_crowded_lanes():
    """The largest values side by side, at a workgroup's stride, ascending and
    descending rows: the lists' largest lengths."""
    rng = np.random.default_rng(3)
    vocab = 70001
    x = rng.standard_normal((4, 2, vocab)).astype(np.float32)
    x[0, :, 5000:9000] += 50
    for j in range(8):
        x[1, :, 8 * 3 + j::2048] += 50 + j
    x[2] = np.sort(x[2], axis=1)
    x[3] = -np.sort(-x[3], axis=1)
    for kind in ("f32", "f16"):
        check_beam(torch.from_numpy(x).to(TYPES[kind]), np.full((4, 2), -1.0, np.float32) * [[1.0, 1.25]], 64)


def test_beam_score_range():
    """Sharp and flat distributions, far apart scores, logits near the types' ends."""
    for kind, spread in (("f32", 30.0), ("f32", 1e-4), ("bf16", 1e30), ("f32", 1e37), ("f16", 15000.0)):
        x, s = beam_case(8, 3, 4, 9001, kind, spread)
        x[~torch.isfinite(x)] = 0
        check_beam(x, s, 8)
        check_beam(x, s * 100, 8)


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def ints(a):
    return dev(np.ascontiguousarray(a, dtype=np.int32))


def pages_ws(n_pages):
    size = s2x.lib.s2x_kv_pages_workspace_size(n_pages)
    return torch.full((size,), 0xff, dtype=torch.uint8, device="cuda:0"), size


def run_fork(parent, kv_len, table, page, n_pages, pinned=None, ld_out=None, st=None):
    n, (m, ld) = len(parent), table.shape
    ld_out = ld if ld_out is None else ld_out
    t = [ints(parent), ints(kv_len), ints(table)]
    pin = None if pinned is None else dev(pinned.astype(np.uint8))
    out = [torch.full(s, -77, dtype=d, device="cuda:0")
           for s, d in (((n, ld_out), torch.int32), ((n,), torch.int32), ((n,), torch.int32), ((n,), torch.int32),
                        ((n,), torch.int32), ((n_pages,), torch.int32), ((2,), torch.int64))]
    ws, size = pages_ws(n_pages)
    s2x.call("s2x_kv_fork", ptr(t[0]), n, ptr(t[1]), ptr(t[2]), m, ld, page, n_pages, ptr(pin), ptr(out[0]), ld_out,
             *[ptr(o) for o in out[1:]], ptr(ws), size, st or stream())
    return [host(o) for o in out]


def check_fork(parent, kv_len, table, page, n_pages, pinned=None, ld_out=None, what=""):
    got = run_fork(parent, kv_len, table, page, n_pages, pinned, ld_out)
    ref = fork_ref(parent, kv_len, table, page, n_pages, pinned, table.shape[1] if ld_out is None else ld_out)
    for name, g, r in zip(("table", "len", "src", "dst", "tok", "free", "count"), got, ref):
        assert_same(g, r, f"{what} {name}")
    return got


def beams_case(rng, n_req, beams, prompt, more, page, spare):
    """Beams of n_req requests, each request's on the pages of its prompt."""
    shared = prompt // page
    lens = np.repeat(prompt + rng.integers(0, more + 1, n_req), beams)
    each = -(-lens // page) - shared
    n_pages = int(shared * n_req + each.sum() + spare)
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(lens), int((-(-lens // page)).max()) + 2), -1, np.int32)
    at = shared * n_req
    for s in range(len(lens)):
        q = s // beams
        table[s, :shared] = ids[q * shared:(q + 1) * shared]
        table[s, shared:shared + each[s]] = ids[at:at + each[s]]
        at += each[s]
    parent = np.arange(len(lens)) // beams * beams + rng.integers(0, beams, len(lens))
    return parent.astype(np.int32), lens.astype(np.int32), table, page, n_pages


@pytest.mark.parametrize("n_req,beams,prompt,more,page,spare", [
    (1, 1, 0, 1, 16, 0), (1, 4, 300, 40, 16, 9), (2, 3, 16, 1, 16, 6), (5, 5, 100, 30, 1, 30), (60, 8, 500, 90, 32, 900),
    (1000, 2, 20, 5, 16, 3000), (3, 64, 700, 300, 8, 4000), (1, 8192, 40, 7, 16, 9000), (7, 4, 33, 9, 65536, 40),
    (40, 3, 3000, 500, 1, 20000)])
def test_fork(n_req, beams, prompt, more, page, spare):
    rng = np.random.default_rng(n_req + prompt)
    say(f"fork: {n_req} x {beams}, prompt {prompt}, page {page}")
    check_fork(*beams_case(rng, n_req, beams, prompt, more, page, spare))


def test_fork_free_pages_of_many_tiles():
    """Page counts around a workgroup's tile, and a million pages."""
    rng = np.random.default_rng(1)
    for spare in (4095, 4096, 4097, 12300, 1 << 20):
        check_fork(*beams_case(rng, 5, 4, 90, 30, 16, spare), what=f"{spare} spare")


def test_fork_orders():
    """Rows dropped, rows doubled, no rows, parents that are none; an open page that
    another row holds as a full one, or with another length; pinned pages; short
    tables, wider rows, missing pages and lengths past the table."""
    rng = np.random.default_rng(6)
    parent, lens, table, page, n_pages = beams_case(rng, 4, 3, 100, 40, 16, 60)
    check_fork(np.full(12, -1), lens, table, page, n_pages, what="all freed")
    check_fork(np.full(30, 5), lens, table, page, n_pages, what="all of one")
    check_fork(np.zeros(0, np.int32), lens, table, page, n_pages, what="no rows")
    check_fork(np.array([-2 ** 31, 2 ** 31 - 1, 12, 11, -1, 0]), lens, table, page, n_pages, what="parents that are none")
    check_fork(np.arange(12), lens, table, page, n_pages, ld_out=table.shape[1] + 7, what="wider rows")
    check_fork(parent, lens, table, page, n_pages, pinned=rng.integers(0, 2, n_pages), what="pinned")
    check_fork(parent, lens, table, page, n_pages, pinned=np.ones(n_pages), what="all pinned")
    t = np.array([[5, 6, -1], [5, 6, -1], [5, 6, 7], [8, 6, -1]])
    for lens_ in ([20, 30, 40, 17], [20, 30, 32, 17], [20, 20, 0, 32], [33, 47, 48, 16], [16, 16, 16, 16], [1, 2, 3, 0]):
        check_fork(np.array([0, 1, 2, 3]), lens_, t, 16, 12, what=f"shared pages {lens_}")
        check_fork(np.array([3, 1, 1, 0, 2, 2]), lens_, t, 16, 12, what=f"shared pages {lens_}")
    lens2 = lens.copy()
    lens2[:4] = [-5, 0, 2 ** 31 - 1, table.shape[1] * 16 + 3]
    t2 = table.copy()
    t2[5, 1], t2[6, 2], t2[7], t2[8, 0] = -1, n_pages, 2 ** 31 - 1, -2 ** 31
    check_fork(parent, lens2, t2, page, n_pages, what="bad tables")
    check_fork(np.arange(12), lens2, t2, page, n_pages, what="bad tables")
    check_fork(np.arange(12), lens, np.zeros((12, 0), np.int32), page, n_pages, what="no table")
    last = t2.copy()
    for s in range(12):  # open pages that are missing
        last[s, -(-int(lens[s]) // 16) - 1] = -1
    check_fork(parent, lens, last, page, n_pages, what="open pages missing")


def test_fork_shortage():
    """Fewer free pages than copies: the last rows go without; once pages are freed
    the same call gives all."""
    rng = np.random.default_rng(7)
    parent, lens, table, page, n_pages = beams_case(rng, 3, 6, 40, 7, 16, 3)
    lens = np.where(lens % 16 == 0, lens + 1, lens)
    first = np.arange(18) // 6 * 6
    table[:] = table[first]
    lens = lens[first]
    pinned = np.ones(n_pages, np.uint8)
    pinned[np.unique(table[table >= 0])] = 0
    spare = np.flatnonzero(pinned)
    pinned[spare[:4]] = 0
    got = check_fork(first, lens, table, page, n_pages, pinned, what="short")
    assert got[6].tolist() == [0, 15] and (got[3] >= 0).sum() == 4
    got = check_fork(first, lens, table, page, n_pages, None, what="again")
    assert got[6][1] == 15


@pytest.mark.parametrize("n_seq,most,page,spare", [
    (1, 10, 16, 0), (1, 0, 16, 3), (5, 200, 16, 40), (150, 2500, 16, 6000), (300, 90, 8, 9000), (3, 70000, 1, 300000),
    (8192, 20, 16, 100), (2, 100, 65536, 1), (40, 500, 16, 0)])
def test_compact(n_seq, most, page, spare):
    rng = np.random.default_rng(n_seq + most)
    say(f"compact: {n_seq} up to {most}, page {page}, {spare} spare")
    lens = rng.integers(0, most + 1, n_seq)
    have = -(-lens // page)
    n_pages = int(have.sum()) + spare + 1
    ids = rng.permutation(n_pages)
    table = np.full((n_seq, int(have.max()) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(have):
        table[s, :n] = ids[at:at + n]
        at += n
    if n_seq > 20:  # shared pages, missing ones, lengths past the table
        table[3:6] = table[2]
        lens[3:6] = lens[2]
        table[7, 0], table[8, 0], lens[9], lens[10] = -1, n_pages, 2 ** 31 - 1, -4
    check_compact(lens, table, page, n_pages)


def check_compact(lens, table, page, n_pages, ld_out=None):
    n, ld = table.shape
    ld_out = ld if ld_out is None else ld_out
    a, b = ints(lens), ints(table)
    out = [torch.full(s, -77, dtype=d, device="cuda:0")
           for s, d in (((n, ld_out), torch.int32), ((n_pages // 2,), torch.int32), ((n_pages // 2,), torch.int32),
                        ((2,), torch.int64))]
    ws, size = pages_ws(n_pages)
    s2x.call("s2x_kv_compact", ptr(a), ptr(b), n, ld, page, n_pages, ptr(out[0]), ld_out, ptr(out[1]) if n_pages > 1 else None,
             ptr(out[2]) if n_pages > 1 else None, ptr(out[3]), ptr(ws), size, stream())
    got = [host(o) for o in out]
    for name, g, r in zip(("table", "src", "dst", "count"), got, compact_ref(lens, table, page, n_pages, ld_out)):
        assert_same(g, r, name)
    return got


def test_compact_borders():
    for n_pages, held in ((4096, range(4095, 2047, -1)), (8192, range(0, 8192, 2)), (8193, [8192]), (3, [2, 1]), (1, [0]),
                          (9000, range(4096, 8192)), (5, []), (4096 * 3, range(4096 * 2))):
        held = np.array(list(held), np.int32)
        table = np.full((1, len(held) + 1), -1, np.int32)
        table[0, :len(held)] = held
        check_compact([len(held)], table, 1, n_pages, ld_out=len(held) + 4)
    check_compact(np.zeros(0, np.int32), np.zeros((0, 3), np.int32), 16, 50)


@pytest.mark.parametrize("heads,page,d,kind,by,gap,n_cache", [
    (1, 1, 8, "f16", "head", 0, 1), (2, 16, 72, "f16", "head", 0, 3), (2, 16, 72, "bf16", "token", 0, 2),
    (8, 64, 128, "bf16", "head", 0, 1), (8, 64, 128, "f16", "token", 0, 1), (3, 8, 40, "f16", "head", 8, 2),
    (3, 8, 40, "f16", "token", 16, 2), (4, 2048, 256, "bf16", "head", 0, 1), (2, 16, 64, "f16", "token", 0, 130),
    (1, 32, 128, "f16", "head", 24, 1)])
def test_copy_pages(heads, page, d, kind, by, gap, n_cache):
    """Whole pages and first places, ids that are none, a number on the device; every
    byte elsewhere stays."""
    rng = np.random.default_rng(heads * page + d)
    n_pages = 12
    caches = [Cache(n_pages, heads, page, d, kind, by, gap, fill=lambda s: torch.randn(s, device="cuda:0")) for _ in range(n_cache)]
    arr = (s2x.KVCache * n_cache)(*[c.c for c in caches])
    src = np.array([3, -1, 7, 0, 5, 2, 9, 3], np.int32)
    dst = np.array([4, 6, 8, 1, n_pages, 2, -2 ** 31, 10], np.int32)
    good = [0, 2, 3, 7]
    for n_tok, n, n_dev in ((None, 8, None), ([page, 3, page // 2, 0, 1, 1, 1, 1], 8, None), ([2 ** 31 - 1, 0, -5, 1, 0, 0, 0, page], 8, 8),
                            (None, 8, 3), (None, 3, 2 ** 40), (None, 8, -1), (None, 8, 0)):
        before = [[m.clone() for m in c.mem] for c in caches]
        nd = None if n_dev is None else torch.tensor([n_dev], dtype=torch.int64, device="cuda:0")
        td = None if n_tok is None else ints(n_tok)
        a, b = ints(src), ints(dst)
        s2x.call("s2x_kv_copy_pages", arr, n_cache, ptr(a), ptr(b), ptr(td), n, ptr(nd), stream())
        torch.cuda.synchronize()
        for c, mems in zip(caches, before):
            want = [m.clone() for m in mems]
            for w in want:
                v = w[..., :d] if by == "head" else w[..., :d].transpose(1, 2)
                old = v.clone()
                for i in good:
                    if i < (n if n_dev is None else min(n, n_dev)):
                        k = page if n_tok is None else min(max(n_tok[i], 0), page)
                        v[int(dst[i]), :, :k] = old[int(src[i]), :, :k]
            for w, m in zip(want, c.mem):
                assert torch.equal(w.view(torch.int16), m.view(torch.int16)), (n_tok, n, n_dev)
                m.normal_()


# ---------------------------------------------------------------------------
# attention over a shared prefix
# ---------------------------------------------------------------------------
def prefix_inputs(rng, groups, hq, hkv, d, kind, page, by, gap=0, spread=1.5):
    """groups: (prefix, [own tokens]) each; own < 0: a sequence that sees that much
    less than the prefix.  Rows of the table for the library, whose pages of the
    prefix only a group's first row has, and for the reference, where all have."""
    lens, rows, held = [], [], 0
    for p, owns in groups:
        n0 = p // page
        shared = list(range(held, held + n0))
        held += n0
        for o in owns:
            own = list(range(held, held + max(0, -(-(p + o) // page) - n0)))
            held += len(own)
            lens.append(p + o)
            rows.append((shared, own))
    n_pages = held + 1
    cache = Cache(n_pages, hkv, page, d, kind, by, gap)
    ids = rng.permutation(n_pages).astype(np.int32)
    ld = max([len(a) + len(b) for a, b in rows] + [1]) + 1
    table = np.full((len(rows), ld), -1, np.int32)
    ref = table.copy()
    s = 0
    for p, owns in groups:
        n0, first = p // page, s
        for o in owns:
            shared, own = rows[s]
            ref[s, :n0], ref[s, n0:n0 + len(own)] = ids[shared], ids[own]
            table[s] = ref[s]
            if s > first:
                table[s, :n0] = rng.integers(-1, n_pages, n0)  # (not looked at)
            for j in range(len(own) if s > first else n0 + len(own)):
                j = n0 + j if s > first else j
                c = min(page, max(p + o, p if s == first else 0) - j * page)
                if c <= 0:
                    continue
                for m in (cache.k, cache.v):
                    m[int(ref[s, j]), :, :c] = torch.from_numpy(rng.standard_normal((hkv, c, d)).astype(np.float32)).to("cuda:0")
            if s > first and p % page and len(own):  # the prefix's last tokens, the same in each
                for m in (cache.k, cache.v):
                    m[int(ref[s, n0]), :, :p % page] = m[int(ref[first, n0]), :, :p % page].clone()
            s += 1
    q = torch.from_numpy((rng.standard_normal((len(rows), hq, d)) * spread).astype(np.float32)).to(TYPES[kind])
    starts = np.concatenate([[0], np.cumsum([len(o) for _, o in groups])]).astype(np.int32)
    return q, cache, table, ref, np.array(lens), starts, np.array([p for p, _ in groups], np.int32)


def run_prefix(q, cache, table, lens, starts, plen, scale, out_kind, max_group=None, max_prefix=None, max_own=None, tok_start=None,
               n_seq=None, lse=True, qpad=0, opad=0, ws=None, st=None):
    n, hq, d = q.shape
    n_seq = len(lens) if n_seq is None else n_seq
    qd = torch.full((n, hq * d + qpad), NAN, dtype=q.dtype, device="cuda:0")
    qd[:, :hq * d] = q.reshape(n, -1).to("cuda:0")
    out = torch.full((n, hq * d + opad), NAN, dtype=TYPES[out_kind], device="cuda:0")
    ls = nans(n, hq) if lse else None
    sizes = np.diff(starts)
    owns = [int(l) - int(p) for g, p in enumerate(plen) for l in lens[max(starts[g], 0):max(starts[g + 1], 0)]]
    mg = int(max(sizes, default=0)) if max_group is None else max_group
    mp = int(max(plen, default=0)) if max_prefix is None else max_prefix
    mo = max(owns + [0]) if max_own is None else max_own
    t = [ints(a) for a in (table, lens, starts, plen)]
    ts = None if tok_start is None else ints(tok_start)
    size = s2x.lib.s2x_attn_paged_prefix_workspace_size(len(plen), mg, mp, mo, hq, cache.n_head, d)
    if ws is None:
        ws = torch.full((max(size, 1),), 0xff, dtype=torch.uint8, device="cuda:0")  # NaNs
    torch.cuda.synchronize()
    s2x.call("s2x_attn_paged_prefix", ptr(qd), hq * d + qpad, n, ptr(ts), cache.ref(), ptr(t[0]), table.shape[1], ptr(t[1]), n_seq,
             ptr(t[2]), ptr(t[3]), len(plen), mg, mp, mo, hq, scale, ptr(out), CODES[out_kind], hq * d + opad, ptr(ls), ptr(ws),
             size, st or stream())
    torch.cuda.synchronize()
    assert torch.isnan(out[:, hq * d:]).all()
    return out[:, :hq * d].double().cpu().numpy().reshape(n, hq, d), None if ls is None else host(ls)


def compare(got, lse, q, cache, ref_table, lens, scale, out_kind, rows=None):
    ref, size, rlse, top, seen = attn_ref(q.float().numpy(), cache, ref_table, lens, 1 << 30, scale, 0)
    d = q.shape[2]
    rows = np.arange(len(lens)) if rows is None else rows
    # as for the attention without a prefix: a score's products and scalings, exp
    # by 2 ulp, the terms of a probability, a rounding a key in the two sums
    score = (d + 6) * U * top
    prob = {"f16": 2.0 ** -21, "bf16": 2.0 ** -22}[cache.kind]
    n = seen[:, None]
    rel = 2 * score + 4 * U + prob + 2 * (n + 8) * U
    tol = rel[:, :, None] * size + HALF_STEP[out_kind] * np.abs(ref) + 2.0 ** -25
    within(got[rows], ref[rows], tol[rows], "out")
    if lse is not None:
        none = np.isinf(rlse)
        assert (lse[rows][none[rows]] == -np.inf).all()
        tol = score + (n + 8) * U + 4 * U * np.abs(np.where(none, 0, rlse))
        within(np.where(none, 0, lse)[rows], np.where(none, 0, rlse)[rows], tol[rows], "lse")


@pytest.mark.parametrize("groups,hq,hkv,d,kind,out_kind,page,by", [
    ([(1, [0])], 1, 1, 64, "f16", "f16", 16, "head"),
    ([(0, [0, 1, 17])], 2, 1, 64, "f16", "f32", 16, "head"),
    ([(33, [1, 2, 3, 4]), (16, [5, 0, 40])], 4, 2, 128, "f16", "f32", 16, "head"),
    ([(300, [7, 60, 0, 1]), (64, [3]), (129, [1, 1, 1])], 16, 16, 72, "f16", "f32", 16, "head"),
    ([(300, [7, 60, 0, 1]), (64, [3]), (129, [1, 1, 1])], 16, 16, 72, "bf16", "f32", 1, "token"),
    ([(100, [5] * 5)], 4, 1, 128, "bf16", "bf16", 64, "head"),                    # 20 columns
    ([(257, [5, 9] * 4)], 8, 2, 64, "f16", "f16", 8, "token"),                    # 32
    ([(511, list(range(13)))], 12, 4, 96, "f16", "f32", 32, "head"),              # 39
    ([(64, [1] * 16)], 4, 1, 128, "f16", "f16", 16, "head"),                      # 64
    ([(65, [1] * 17)], 4, 1, 128, "bf16", "f32", 16, "token"),                    # 68
    ([(700, [30, 400, 2] * 10)], 16, 4, 128, "f16", "f16", 16, "head"),           # 120
    ([(1000, [3] * 33), (10, [4] * 7)], 16, 4, 128, "bf16", "bf16", 16, "head"),  # 132: 8 waves
    ([(190, [3] * 70)], 4, 1, 72, "f16", "f32", 16, "head"),                      # two tiles of columns
    ([(90, [3] * 140)], 8, 2, 80, "bf16", "bf16", 2, "token"),
    ([(200, [3, 50] * 10)], 4, 1, 256, "f16", "f16", 16, "head"),                 # 80 columns of 256
    ([(200, [3, 50] * 4)], 8, 2, 192, "bf16", "f32", 16, "head"),
    ([(130, [3, 5] * 3)], 5, 1, 248, "f16", "f32", 32, "token"),
    ([(500, [9] * 40)], 4, 1, 200, "bf16", "f32", 4, "head"),
    ([(70, [3, 5] * 9)], 2, 2, 8, "f16", "f32", 16, "head"),
    ([(70, [3, 5] * 3)], 17, 1, 40, "f16", "f32", 16, "head"),                    # 17 query heads on one
    ([(70, [3, 500])], 48, 1, 64, "bf16", "f32", 16, "token"),
    ([(5000, [700, 3, 900])], 8, 2, 128, "f16", "f32", 16, "head"),               # many chunks
    ([(9000, [1] * 20)], 8, 2, 128, "bf16", "f32", 2048, "head"),
    ([(p, [1, 2]) for p in range(0, 200, 9)], 4, 4, 64, "f16", "f16", 16, "head")])
def test_prefix(groups, hq, hkv, d, kind, out_kind, page, by):
    say(f"prefix: {groups[:3]} {hq}/{hkv} x {d} {kind}->{out_kind} page {page} {by}")
    rng = np.random.default_rng(sum(p for p, _ in groups) + d)
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, groups, hq, hkv, d, kind, page, by)
    got, lse = run_prefix(q, cache, table, lens, starts, plen, d ** -0.5, out_kind)
    compare(got, lse, q, cache, ref, lens, d ** -0.5, out_kind)
    again, _ = run_prefix(q, cache, table, lens, starts, plen, d ** -0.5, out_kind, lse=False)
    assert_same(again, got, "without lse")


@pytest.mark.parametrize("share,size", [(2, 5), (2, 20), (4, 40), (4, 80)])
def test_prefix_shorter_sequences(share, size):
    """Sequences that end inside the prefix, or hold nothing at all."""
    rng = np.random.default_rng(size)
    p = 400
    owns = [int(x) for x in rng.integers(-p, 30, size)]
    owns[1], owns[2], owns[3] = -p, -1, -64
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, [(p, owns)], share, 1, 128, "f16", 16, "head")
    got, lse = run_prefix(q, cache, table, lens, starts, plen, 0.1, "f32")
    compare(got, lse, q, cache, ref, lens, 0.1, "f32")
    assert (got[1] == 0).all() and (lse[1] == -np.inf).all()


@pytest.mark.parametrize("share", [2, 4, 16])
def test_prefix_bounds(share):
    """Lengths past the limits and the table, negative ones, pages that are none,
    strides, groups larger than said, starts that are no sequences."""
    rng = np.random.default_rng(12)
    groups = [(200, [20, 100, 9, 64, 7]), (90, [50, 5, 5]), (333, [1, 30])]
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, groups, 2 * share, 2, 72, "f16", 16, "token", gap=8)
    args = (0.12, "f32")
    got, lse = run_prefix(q, cache, table, lens, starts, plen, *args, qpad=8, opad=24)
    compare(got, lse, q, cache, ref, lens, 0.12, "f32")
    # a prefix past max_prefix: the rest is the sequences' own, so their rows need it
    got, lse = run_prefix(q, cache, ref, lens, starts, plen, *args, max_prefix=150, max_own=1000)
    compare(got, lse, q, cache, ref, lens, 0.12, "f32")
    got, lse = run_prefix(q, cache, ref, lens, starts, plen, *args, max_prefix=0, max_own=1000)
    compare(got, lse, q, cache, ref, lens, 0.12, "f32")
    # own tokens past max_own are not seen
    cut = np.minimum(lens, np.repeat(plen, np.diff(starts)) + 13)
    got, lse = run_prefix(q, cache, table, lens, starts, plen, *args, max_own=13)
    compare(got, lse, q, cache, ref, cut, 0.12, "f32")
    got, lse = run_prefix(q, cache, table, lens, starts, plen, *args, max_own=0)
    compare(got, lse, q, cache, ref, np.repeat(plen, np.diff(starts)), 0.12, "f32")
    # larger groups than said, sequences of no group
    got, lse = run_prefix(q, cache, table, lens, starts, plen, *args, max_group=2)
    rows = np.array([0, 1, 5, 6, 8, 9])
    compare(got, lse, q, cache, ref, lens, 0.12, "f32", rows)
    assert np.isnan(np.delete(got, rows, 0)).all() and np.isnan(np.delete(lse, rows, 0)).all()
    got, lse = run_prefix(q, cache, table, lens, np.array([5, 8], np.int32), plen[1:2], *args, max_own=100)
    compare(got, lse, q, cache, ref, lens, 0.12, "f32", np.array([5, 6, 7]))
    assert np.isnan(np.delete(got, [5, 6, 7], 0)).all()
    for bad in ([-3, 2, 10], [8, 5, 5], [10, 12, 14], [-2 ** 31, 2 ** 31 - 1, -5]):
        got, _ = run_prefix(q, cache, table, lens, np.array(bad), plen[:2], *args, max_group=3, max_own=100)
        assert np.isnan(got).all() or bad[0] == -3
    got, _ = run_prefix(q, cache, ref, lens, np.array([8, 2 ** 31 - 1]), plen[2:], *args, max_group=3, max_own=100)
    compare(got, None, q, cache, ref, lens, 0.12, "f32", np.array([8, 9]))
    # bad pages are unseen places
    t2, r2 = table.copy(), ref.copy()
    for s, j, id_ in ((0, 3, -1), (0, 11, cache.n_pages), (5, 0, 2 ** 31 - 1), (1, 14, -2 ** 31), (8, 20, -1)):
        t2[s, j] = id_
        group = [s] if j >= plen[np.searchsorted(starts, s, "right") - 1] // 16 else range(
            starts[np.searchsorted(starts, s, "right") - 1], starts[np.searchsorted(starts, s, "right")])
        for i in group:
            r2[i, j] = id_
    # (entry 20 of row 8 lies across the prefix's end: the others hold its places)
    r2[9, 20] = -1
    t2[9, 20] = -1
    got, lse = run_prefix(q, cache, t2, lens, starts, plen, *args)
    compare(got, lse, q, cache, r2, lens, 0.12, "f32")
    got, lse = run_prefix(q, cache, t2[:, :10].copy(), lens, starts, plen, *args)
    compare(got, lse, q, cache, r2[:, :10], lens, 0.12, "f32")
    for n in (-5, -2 ** 31, 2 ** 31 - 1):
        lens2 = lens.copy()
        lens2[[1, 5, 9]] = n
        got, lse = run_prefix(q, cache, table, lens2, starts, plen, *args, max_own=100)
        keep = np.setdiff1d(np.arange(10), [1, 5, 9])
        compare(got, lse, q, cache, ref, lens2 if n < 0 else lens, 0.12, "f32", None if n < 0 else keep)
    got, lse = run_prefix(q, cache, np.zeros((10, 0), np.int32), lens, starts, plen, *args, max_own=100)
    assert (got == 0).all() and (lse == -np.inf).all()


@pytest.mark.parametrize("share", [2, 8])
def test_prefix_packed_rows(share):
    """Rows by tok_start: idle sequences, sequences with several rows, starts that
    are no rows."""
    rng = np.random.default_rng(13)
    groups = [(200, [20, 100, 9, 64, 7]), (90, [50, 5, 5])]
    q8, cache, table, ref, lens, starts, plen = prefix_inputs(rng, groups, 2 * share, 2, 64, "bf16", 16, "head")
    tok = np.array([0, 1, 1, 4, 5, 5, 6, 8, 9], np.int32)
    q = torch.from_numpy(rng.standard_normal((11, 2 * share, 64)).astype(np.float32)).bfloat16()
    last = {s: int(tok[s + 1]) - 1 for s in range(8) if tok[s + 1] > tok[s]}
    got, lse = run_prefix(q, cache, table, lens, starts, plen, 0.12, "f32", tok_start=tok)
    rows = list(last)
    full = torch.zeros(8, 2 * share, 64).bfloat16()
    full[rows] = q[[last[s] for s in rows]]
    g2, l2 = np.zeros((8, 2 * share, 64)), np.zeros((8, 2 * share), np.float32)
    g2[rows], l2[rows] = got[[last[s] for s in rows]], lse[[last[s] for s in rows]]
    compare(g2, l2, full, cache, ref, lens, 0.12, "f32", np.array(rows))
    others = np.setdiff1d(np.arange(11), list(last.values()))
    assert np.isnan(got[others]).all() and np.isnan(lse[others]).all()
    tok = np.array([-1, -3, 2, 1, 5, 30, 2 ** 31 - 1, -2 ** 31, 9], np.int32)
    got, _ = run_prefix(q, cache, table, lens, starts, plen, 0.12, "f32", tok_start=tok)
    full[:] = q[4]
    want, _ = run_prefix(full, cache, table, lens, starts, plen, 0.12, "f32")
    assert_same(got[4], want[3], "row 4")
    assert np.isnan(np.delete(got, 4, 0)).all()


@pytest.mark.parametrize("hq,size", [(2, 4), (4, 24)])
def test_prefix_score_range(hq, size):
    """Scores far apart, equal ones, a scale of either sign; NaNs in a group stay
    in it."""
    rng = np.random.default_rng(5)
    groups = [(600, [9] * size)] * 2
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, groups, hq, 1, 128, "bf16", 16, "head")
    q = q * 20
    for scale in (1.0, -1.0, 0.0):
        got, lse = run_prefix(q, cache, table, lens, starts, plen, scale, "f32")
        compare(got, lse, q, cache, ref, lens, scale, "f32")
    cache.v[int(ref[0, 2]), 0, 5] = NAN
    clean, _ = run_prefix(q, cache, table, lens, starts, plen, 0.05, "f32")
    assert np.isnan(clean[:size]).any(axis=2).all() and np.isfinite(clean[size:]).all()
