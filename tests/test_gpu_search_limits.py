"""What the header says of the beam search's operators at its ends: the selection's
error and order, prefixes of freed and of odd groups, pinned pages in a compaction,
calls at once and over one workspace.

u = 2^-24, the half step of an f32 at 1."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import TYPES, Cache
from gpu_util import assert_same, dev, host, ptr, say, stream
from search_util import beam_scores, compact_ref, fork_ref
from test_gpu_decode import NAN, U
from test_gpu_search import (INF, beam_case, beams_case, check_compact, compare, ints, nans, prefix_inputs, rms_case, run_beam,
                             run_fork, run_prefix, run_rms)

pytestmark = pytest.mark.gpu


def few_values(vocab, places, beams, kind):
    """beams: (score, values) each; the values at `places`, -inf elsewhere."""
    x = torch.full((1, len(beams), vocab), -INF)
    for b, (_, values) in enumerate(beams):
        x[0, b, places] = torch.tensor(values, dtype=torch.float32)
    return x.to(TYPES[kind]), np.array([[s for s, _ in beams]], np.float32)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [0, 50, 300, 1000, 3990, 4090, 4100, 60000, -50, -300, -1000, -4100])
@pytest.mark.parametrize("vocab,places", [(3, [0, 1, 2]), (70000, [7, 30001, 69999])])
def test_beam_large_logits(kind, top, vocab, places):
    """Three values whose largest is far from 0, side by side and in parts of the row
    of their own.  An exponential is off by 2 u, its argument by up to 2.3 u times the
    value's distance from the top (0.4 on average), and two additions by 2 u, or, of
    values apart (a fifth of the whole), a wave's and a part's scale by 2 u each: 5 u,
    6 with the terms of f64, below 2^-21, and half a step of the f32 score."""
    x, s = few_values(vocab, places, [(-1.0, [top, top - 1.5, top - 3])], kind)
    ref = beam_scores(x[0].float().numpy(), s[0], None, 0)[0, places]
    parent, token, score = run_beam(x, s, 3)
    order = np.argsort(-ref, kind="stable")
    assert parent[0].tolist() == [0, 0, 0] and token[0].tolist() == [places[i] for i in order]
    assert (np.abs(score[0] - ref[order]) <= 6 * U + U * np.abs(ref[order])).all(), (score[0] - ref[order]) / U


@pytest.mark.parametrize("vocab,places", [(3, [0, 1, 2]), (70000, [7, 30001, 69999])])
def test_beam_order_of_unlike_beams(vocab, places):
    """Beams whose logits lie apart and whose scores differ by a few 1e-6, 50 u and more:
    the order is the scores', and no continuation counts more than its beam."""
    for high, low in ((900, 100), (300, 0), (3900, -1000), (4090, 4100), (50, -800)):
        for a, b in ((-1.00001, -1.0), (-1.000003, -1.0), (-1.0, -1.00001), (-1.0, -1.000003)):
            x, s = few_values(vocab, places, [(a, [high, high - 50, high - 100]), (b, [low, low - 50, low - 100])], "f32")
            parent, token, score = run_beam(x, s, 2)
            assert parent[0].tolist() == ([0, 1] if a > b else [1, 0]), (high, low, a, b, score)
            assert token[0].tolist() == [places[0]] * 2
            # (e^-50 of the whole: nothing; an exponential 2 u, the score's rounding 1 u)
            assert (np.abs(score[0] - np.sort(s[0])[::-1]) <= 4 * U).all(), (score, s)


def check_closely(logits, scores, n_out):
    """Each place's score within the documented error of that place's in 64 bits, the
    very candidate where its neighbours are further off.  An exponential is off by
    2 u, its argument by up to 2.3 u times the distance from its wave's top, which over
    a wave's 8,192 values is at most 6.2 on average (E exp(1 + E) = 8,191), three
    additions in f32, and a wave's and a part's scale 2 u each: 23.3 u."""
    tol = 23.3 * U
    parent, token, score = run_beam(logits, scores, n_out)
    vocab, x = logits.shape[2], logits.float().numpy()
    for r in range(len(x)):
        s = beam_scores(x[r], scores[r], None, 0)
        flat = np.argsort(-s, axis=None, kind="stable")[:n_out + 1]
        best = s.flatten()[flat]
        got = np.array([s[p - r * x.shape[1], t] for p, t in zip(parent[r], token[r])])
        assert (np.abs(got - best[:n_out]) <= 2 * tol).all(), r
        assert (np.abs(score[r] - got) <= tol + U * np.abs(got)).all(), (r, np.abs(score[r] - got).max() / U)
        gap = np.concatenate([[np.inf], -np.diff(best)])
        sure = np.minimum(gap[:-1], gap[1:]) > 2 * tol
        at = (parent[r] - r * x.shape[1]) * vocab + token[r]
        assert (at[sure] == flat[:n_out][sure]).all(), r
    return score


@pytest.mark.parametrize("n,beams,vocab,kind,n_out", [
    (1, 4, 32000, "f32", 4), (3, 5, 50021, "f16", 10), (2, 8, 256000, "bf16", 16), (70, 4, 40001, "f32", 2),
    (1, 16, 98304, "bf16", 64), (5, 3, 257, "f16", 8)])
@pytest.mark.parametrize("spread,mean", [(1e-3, 0.0), (0.7, 15.0), (2.5, 0.0), (4.0, -900.0), (8.0, 3000.0), (1000.0, 5000.0)])
def test_beam_error(n, beams, vocab, kind, n_out, spread, mean):
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy((rng.standard_normal((n, beams, vocab), dtype=np.float32) * spread + mean).astype(np.float32)).to(TYPES[kind])
    check_closely(x, -rng.uniform(0, 3, (n, beams)).astype(np.float32), n_out)


@pytest.mark.parametrize("kind,vocab,per", [("f32", 32768, 4), ("f16", 65536, 8), ("bf16", 65536, 8)])
def test_beam_sums_that_repeat(kind, vocab, per):
    """Rows whose every lane has the same values, a 0 and p - 1 of -d again and again:
    roundings that do not average out.  129 rows of two parts of 16 loads a lane.  All tops
    are 0, so that c and the scales are exact: an exponential 2 u, its argument 1.3 u
    times the distance (2.8 at most on average), three additions: 9 u.
    The beam's score is its row's log-sum-exp, so that S is next to 0."""
    rng = np.random.default_rng(3)
    col = np.arange(vocab)
    place = col // (256 * per) * per + col % per  # of the lane's values
    period = 2 ** rng.integers(1, 6, 129)
    d = np.exp(rng.uniform(np.log(0.05), np.log(4.0), 129))
    d[:6], period[:6] = [2.5625, 2.9375, 3.15625, 2.58984375, 2.741, 3.9695], [32, 16, 32, 32, 32, 32]
    x = torch.from_numpy(np.where(place[None] % period[:, None] == 0, 0.0, -d[:, None]).astype(np.float32)).to(TYPES[kind])
    v = x.double().numpy()
    lse = np.log(np.exp(v).sum(1))
    scores = lse.astype(np.float32)[:, None]
    parent, token, score = run_beam(x[:, None], scores, 1)
    want = scores[:, 0].astype(np.float64) - lse
    assert (parent[:, 0] == np.arange(129)).all() and (token == 0).all()
    err = np.abs(score[:, 0] - want)
    assert (err <= 9 * U + U * np.abs(want)).all(), (err.max() / U, int(err.argmax()))


def same_s_order(x, scores, n_out):
    """Places of a request whose every beam has one S for all its tokens (logits too
    small to change it): by beam's score, then the lower beam, the larger logit, the
    lower token."""
    beams, vocab = x.shape
    out = []
    for b in sorted(range(beams), key=lambda b: (-scores[b], b)):
        out += [(b, int(t)) for t in np.argsort(-x[b].astype(np.float64), kind="stable")[:n_out]]
    return out[:n_out]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("beams,vocab,n_out", [(1, 3, 3), (1, 3000, 64), (2, 70000, 5), (4, 32000, 4), (1, 300001, 64), (3, 1000003, 64),
                                               (64, 9000, 64), (8, 200000, 60)])
def test_beam_order_of_equal_scores(beams, vocab, n_out, kind):
    """Logits of some 1e-20 that differ where S, in f64, does not: of one beam's the
    larger logit is ahead, in whatever part or round of the join it lies, then the
    lower token; of two beams' the lower beam.  Few of them among others, and rows of
    nothing else (more equal scores than a list takes)."""
    rng = np.random.default_rng(vocab + beams)
    for values, dense in ((40, True), (1 << 30, True), (40, False)):
        tiny = rng.integers(0, values, (beams, vocab)).astype(np.float32) * np.float32(1e-20 / values * 40)
        x = tiny if dense else np.where(rng.random((beams, vocab)) < max(0.01, 5.0 / vocab), tiny, np.float32(-1.0))
        x[1:] = x[0]  # (one sum in all beams)
        t = torch.from_numpy(x[None].copy()).to(TYPES[kind])
        v = t[0].float().numpy()
        for scores in (np.full(beams, -3.0), np.where(np.arange(beams) == beams - 1, -2.0, -3.0), -2.0 - np.arange(beams) % 3):
            want = same_s_order(v, scores, n_out)
            if not dense:  # (the others lie a whole 1 below)
                want = [w for w in want if v[w] > -0.5]
            parent, token, score = run_beam(t, scores[None].astype(np.float32), n_out)
            n = min(len(want), n_out)
            if not dense:  # only of the first beam are the next in order known
                n = next((i for i, w in enumerate(want) if w[0] != want[0][0]), n)
            got = [(int(p), int(k)) for p, k in zip(parent[0], token[0])]
            assert got[:n] == want[:n], (dense, values, scores[:4])
            assert (np.diff(score[0]) <= 0).all()


@pytest.mark.parametrize("share,size,d,kind,freed", [
    (2, 5, 128, "f16", [0]), (1, 6, 72, "bf16", [0, 1, 3]), (2, 20, 64, "bf16", [0]), (4, 40, 128, "f16", [0, 1, 2, 39]),
    (4, 33, 128, "bf16", [0]), (3, 9, 256, "f16", [0, 8]), (8, 6, 200, "bf16", [0]), (1, 90, 64, "f16", list(range(70))),
    (1, 12, 64, "f16", list(range(12)))])
def test_prefix_of_a_freed_first_sequence(share, size, d, kind, freed):
    """Sequences of a group that s2x_kv_fork frees, its first among them: the others
    see the prefix as before, from the first that is left, also one that ends inside
    it behind which the values are no numbers."""
    rng = np.random.default_rng(size)
    p, at = 700, 333
    owns = [int(o) for o in rng.integers(0, 30, size)]
    groups = [(90, [3, 4]), (p, owns), (40, [7])]
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, groups, 2 * share, 2, d, kind, 16, "head")
    table = ref.copy()  # (every row's own: those of freed ones go)
    parent = np.arange(len(lens))
    parent[np.array(freed) + 2] = -1
    out, lens2, src, dst, _, _, _ = run_fork(parent, lens, table, 16, cache.n_pages, pinned=np.zeros(cache.n_pages))
    live = np.setdiff1d(np.arange(len(lens)), np.array(freed) + 2)
    # (rows of a group share its whole pages only: nothing to copy)
    assert (src == -1).all() and (out[live] == table[live]).all() and (out[np.array(freed) + 2] == -1).all()
    assert (lens2[np.array(freed) + 2] == 0).all()
    # what the other rows have at the prefix is not looked at
    left = [i for i in range(size) if i not in freed]
    for i in left[1:]:
        out[2 + i, :p // 16] = rng.integers(-1, cache.n_pages, p // 16)
    table[np.array(freed) + 2] = -1
    if size - 2 in left:
        lens2[size] = at  # (ends inside the prefix)
    got, lse = run_prefix(q, cache, out, lens2, starts, plen, 0.1, "f32", max_own=40)
    compare(got, lse, q, cache, table, lens2, 0.1, "f32")
    if size - 2 in left:
        cache.v[int(ref[2 + left[0], (at + 20) // 16]), :, 3] = NAN
        got, lse = run_prefix(q, cache, out, lens2, starts, plen, 0.1, "f32", max_own=40)
        rows = np.array([0, 1, size, size + 2])
        assert np.isnan(got[np.setdiff1d(live, rows)]).all(axis=2).all() if len(left) > 1 else True
        compare(got[rows], lse[rows], q[rows], cache, table[rows], lens2[rows], 0.1, "f32")


@pytest.mark.parametrize("share", [2, 4, 16])
def test_prefix_group_behind_one_that_is_none(share):
    """Starts of -3, 2, 10: the first group is none, the second its first three
    sequences, whose prefix lies in the first one's pages; all other rows stay."""
    rng = np.random.default_rng(12)
    groups = [(200, [20, 100, 9, 64, 7]), (90, [50, 5, 5]), (333, [1, 30])]
    q, cache, _, ref, lens, _, _ = prefix_inputs(rng, groups, 2 * share, 2, 72, "f16", 16, "token", gap=8)
    got, lse = run_prefix(q, cache, ref, lens, np.array([-3, 2, 10]), np.array([200, 90]), 0.12, "f32", max_group=3, max_own=300)
    rows = np.array([2, 3, 4])
    compare(got, lse, q, cache, ref, lens, 0.12, "f32", rows)
    assert np.isnan(np.delete(got, rows, 0)).all() and np.isnan(np.delete(lse, rows, 0)).all()


def test_compact_with_pinned_pages():
    """A fork that keeps pinned pages while their sequence is freed, then a compaction
    that is given them as further rows: their content is where those rows say, and
    that of the sequences where theirs do."""
    rng = np.random.default_rng(11)
    page, n_pages, n, ld = 16, 300, 12, 9
    ids = rng.permutation(n_pages).astype(np.int32)
    lens = rng.integers(1, ld * page + 1, n)
    table = np.full((n, ld), -1, np.int32)
    for s in range(n):
        have = -(-int(lens[s]) // page)
        table[s, :have] = ids[s * ld:s * ld + have]
    # the pages of rows 0 and 5, which go, and two of no row
    keep = np.concatenate([table[0][table[0] >= 0], table[5][table[5] >= 0], ids[200:202]])
    pinned = np.zeros(n_pages, np.uint8)
    pinned[keep] = 1
    parent = np.array([-1, 1, 2, 3, 4, -1, 6, 7, 7, 8, 9, 10])
    cache = Cache(n_pages, 2, page, 64, "f16", fill=lambda shape: torch.randn(shape, device="cuda:0"))
    out, lens2, src, dst, tok, free, count = run_fork(parent, lens, table, page, n_pages, pinned=pinned)
    assert not set(keep.tolist()) & (set(free.tolist()) | set(dst.tolist()))
    t = [ints(a) for a in (src, dst, tok)]
    s2x.call("s2x_kv_copy_pages", cache.ref(), 1, ptr(t[0]), ptr(t[1]), ptr(t[2]), n, None, stream())
    torch.cuda.synchronize()
    k, v = (c.clone() for c in (cache.k, cache.v))
    rows = -(-len(keep) // ld)
    more = np.full((rows, ld), -1, np.int32)
    more.flat[:len(keep)] = keep
    table2 = np.concatenate([out, more])
    lens3 = np.concatenate([lens2, [page * int((r >= 0).sum()) for r in more]])
    new, src, dst, count = check_compact(lens3, table2, page, n_pages)
    a, b, c = ints(src), ints(dst), torch.tensor([int(count[1])], dtype=torch.int64, device="cuda:0")
    s2x.call("s2x_kv_copy_pages", cache.ref(), 1, ptr(a), ptr(b), None, len(src), ptr(c), stream())
    torch.cuda.synchronize()
    held = table2 >= 0
    assert new[held].max() == count[0] - 1 and ((new >= 0) == held).all()
    to, fro = (torch.from_numpy(x[held].astype(np.int64)).to("cuda:0") for x in (new, table2))
    assert torch.equal(cache.k[to], k[fro]) and torch.equal(cache.v[to], v[fro])
    # without those rows the pages are given up
    assert count[0] > compact_ref(lens2, out, page, n_pages, ld)[3][0]


# ---------------------------------------------------------------------------
# calls at once, and one after the other over one workspace
# ---------------------------------------------------------------------------
class Job:
    """A call over buffers of its own: outputs `out`, filled before every run, a
    workspace of `need` bytes, `call(ws, stream)`."""

    def __init__(self, name, keep, out, need, call):
        self.name, self.keep, self.out, self.need, self.call = name, keep, out, need, call

    def clear(self):
        for o in self.out:
            o.fill_(NAN if o.is_floating_point() else -77)

    def values(self):
        return [o.clone() for o in self.out]

    def check(self, want, what):
        for i, (o, w) in enumerate(zip(self.out, want)):
            a, b = (t.contiguous().view(torch.uint8) for t in (o, w))
            assert torch.equal(a, b), (self.name, i, what)


def workspace(n):
    return torch.full((max(1, n),), 0xff, dtype=torch.uint8, device="cuda:0")


def full(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device="cuda:0")


def fork_job(seed, *shape):
    parent, lens, table, page, n_pages = case = beams_case(np.random.default_rng(seed), *shape)
    n, ld = table.shape
    t = [ints(a) for a in (parent, lens, table)]
    out = [full((n, ld), torch.int32), *(full((n,), torch.int32) for _ in range(4)), full((n_pages,), torch.int32), full((2,), torch.int64)]
    need = s2x.lib.s2x_kv_pages_workspace_size(n_pages)
    job = Job(f"fork {shape}", t, out, need, lambda ws, st: s2x.call(
        "s2x_kv_fork", ptr(t[0]), n, ptr(t[1]), ptr(t[2]), n, ld, page, n_pages, None, ptr(out[0]), ld, *[ptr(o) for o in out[1:]],
        ptr(ws), need, st))
    job.ref = fork_ref(parent, lens, table, page, n_pages, None, ld)
    return job


def compact_job(seed, n_seq, most, n_pages):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, most + 1, n_seq)
    have = -(-lens // 16)
    ids, at = rng.permutation(n_pages), 0
    table = np.full((n_seq, int(have.max())), -1, np.int32)
    for s, h in enumerate(have):
        table[s, :h] = ids[at:at + h]
        at += h
    ld, half = table.shape[1], n_pages // 2
    t = [ints(lens), ints(table)]
    cache = Cache(n_pages, 1, 16, 8, "f16", fill=lambda shape: torch.randn(shape, device="cuda:0"))
    out = [full((n_seq, ld), torch.int32), full((half,), torch.int32), full((half,), torch.int32), full((2,), torch.int64)]
    need = s2x.lib.s2x_kv_pages_workspace_size(n_pages)

    def call(ws, st):
        s2x.call("s2x_kv_compact", ptr(t[0]), ptr(t[1]), n_seq, ld, 16, n_pages, ptr(out[0]), ld, ptr(out[1]), ptr(out[2]),
                 ptr(out[3]), ptr(ws), need, st)
        # (no copy_dst is a copy_src: the same again and again)
        s2x.call("s2x_kv_copy_pages", cache.ref(), 1, ptr(out[1]), ptr(out[2]), None, half, ctypes.c_void_p(out[3].data_ptr() + 8), st)
    job = Job(f"compact {n_seq} {n_pages}", [t, cache], out, need, call)
    job.ref = compact_ref(lens, table, 16, n_pages, ld)
    job.cache, job.before = cache, [c.clone() for c in (cache.k, cache.v)]
    return job


def prefix_job(seed, groups, hq, hkv, d, kind):
    q, cache, table, _, lens, starts, plen = prefix_inputs(np.random.default_rng(seed), groups, hq, hkv, d, kind, 16, "head")
    n, mg, mp = len(lens), int(np.diff(starts).max()), int(plen.max())
    mo = max(max(o) for _, o in groups)
    t = [q.to("cuda:0"), *(ints(a) for a in (table, lens, starts, plen))]
    out = [nans(n, hq * d), nans(n, hq)]
    need = s2x.lib.s2x_attn_paged_prefix_workspace_size(len(plen), mg, mp, mo, hq, hkv, d)
    return Job(f"prefix {hq}/{hkv} x {d}", [t, cache], out, need, lambda ws, st: s2x.call(
        "s2x_attn_paged_prefix", ptr(t[0]), hq * d, n, None, cache.ref(), ptr(t[1]), table.shape[1], ptr(t[2]), n, ptr(t[3]), ptr(t[4]),
        len(plen), mg, mp, mo, hq, 0.09, ptr(out[0]), 0, hq * d, ptr(out[1]), ptr(ws), need, st))


def beam_job(seed, n, beams, vocab, kind, n_out):
    x, s = beam_case(seed, n, beams, vocab, kind)
    t = [x.to("cuda:0"), dev(s)]
    out = [full((n, n_out), d) for d in (torch.int32, torch.int32, torch.float32)]
    need = s2x.lib.s2x_beam_select_workspace_size(n, beams, vocab, n_out)
    code = {"f32": 0, "f16": 1, "bf16": 2}[kind]
    return Job(f"beam {n} {beams} {vocab}", t, out, need, lambda ws, st: s2x.call(
        "s2x_beam_select", ptr(t[0]), code, vocab, n, beams, vocab, ptr(t[1]), None, 0, n_out, *[ptr(o) for o in out], ptr(ws), need, st))


def rms_job(seed, m, h):
    x, r, w = rms_case(seed, m, h, "f32", "f32")
    k = -(-h // 32) * 32
    t = [x.to("cuda:0"), r.to("cuda:0"), dev(w)]
    out = [nans(m, h), full((m, k), torch.int8), full((m, k // 32), torch.int32), nans(m, h)]
    return Job(f"norm {m} x {h}", t, out, 0, lambda ws, st: s2x.call(
        "s2x_add_rmsnorm_quantize_q8_1", ptr(t[0]), 0, h, ptr(t[1]), 0, h, h, m, ptr(t[2]), 1e-6, ptr(out[0]), h, k, ptr(out[1]),
        ptr(out[2]), ptr(out[3]), 0, h, st))


def page_jobs():
    """Forks in one workgroup, of few pages and of many tiles of them, and compactions
    of few and of many, two of each."""
    return [fork_job(1, 3, 4, 90, 30, 16, 40), fork_job(2, 9, 5, 300, 60, 16, 700), fork_job(3, 60, 8, 900, 90, 16, 3000),
            fork_job(4, 200, 6, 40, 30, 16, 21000), fork_job(5, 40, 8, 500, 90, 16, 50000), fork_job(6, 7, 300, 70, 20, 8, 90000),
            compact_job(7, 40, 900, 9000), compact_job(8, 300, 200, 12000), compact_job(9, 200, 1500, 70000),
            compact_job(10, 5, 9000, 40001)]


def settled(job):
    """The call alone: its outputs, those of the pages against the plain form."""
    ws = workspace(job.need)
    job.clear()
    torch.cuda.synchronize()
    job.call(ws, stream())
    torch.cuda.synchronize()
    for i, r in enumerate(getattr(job, "ref", [])):
        assert_same(host(job.out[i]).reshape(r.shape), r, f"{job.name} {i}")
    if hasattr(job, "cache"):
        src, dst, n = host(job.out[1]), host(job.out[2]), int(host(job.out[3])[1])
        for c, b in zip((job.cache.k, job.cache.v), job.before):
            b[dst[:n].tolist()] = b[src[:n].tolist()].clone()
            assert torch.equal(c, b), job.name
    return job.values()


def test_every_operator_on_two_streams_at_once():
    """All launches on both streams before any wait, each over buffers and a workspace
    of its own: the bits of the call alone."""
    jobs = page_jobs() + [
        prefix_job(1, [(700, [30, 5, 60]), (90, [3, 4])], 8, 2, 128, "f16"), prefix_job(2, [(900, [30, 5, 60, 1] * 5)], 8, 2, 128, "bf16"),
        prefix_job(3, [(400, [9] * 40)], 4, 1, 72, "f16"), prefix_job(4, [(50, [300, 2])] * 9, 4, 4, 64, "bf16"),
        beam_job(5, 3, 4, 20011, "f32", 8), beam_job(6, 30, 4, 30000, "bf16", 4), beam_job(7, 1, 32, 40000, "f16", 64),
        rms_job(8, 33, 2100), rms_job(9, 700, 512), rms_job(10, 3000, 100)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    handles = [ctypes.c_void_p(s.cuda_stream) for s in streams]
    want = [settled(j) for j in jobs]
    spaces = [workspace(j.need) for j in jobs]
    for r in range(4):
        say(f"round {r}")
        for j in jobs:
            j.clear()
        torch.cuda.synchronize()
        for i, j in enumerate(jobs):
            j.call(spaces[i], handles[(i + r) % 2])
        torch.cuda.synchronize()
        for j, w in zip(jobs, want):
            j.check(w, f"round {r}")


def test_page_calls_over_one_workspace():
    """Captured forks and compactions of different rows and pages, replayed in turn
    over the same workspace with eager work between: nothing of one is left for
    another."""
    jobs = page_jobs()
    want = [settled(j) for j in jobs]
    ws = workspace(max(j.need for j in jobs))
    graphs = []
    for j in jobs:
        j.call(ws, stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            j.call(ws, stream())
        graphs.append(g)
    rng = np.random.default_rng(1)
    for r in range(3):
        for i in rng.permutation(len(jobs)):
            jobs[i].clear()
            graphs[i].replay()
            torch.cuda.synchronize()
            jobs[i].check(want[i], f"round {r}")
            torch.randn(300, 300, device="cuda:0").sum()


@pytest.mark.parametrize("m,h", [(1, 64), (2, 33), (37, 1157), (200, 4096)])
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (3, 2, 1, 0), (2, 0, 3, 1)])
def test_rms_columns_of_one_buffer(m, h, order):
    """x, the residual, h and y as columns of one buffer, with columns of none between."""
    x, r, w = rms_case(h, m, h, "f32", "f32")
    wd, gap = dev(w), 5
    mem = nans(m, 4 * h + gap)
    at = [i * h + (gap if i > 1 else 0) for i in order]
    xs, rs, hs, ys = (mem[:, a:a + h] for a in at)
    xs.copy_(x)
    rs.copy_(r)
    s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(xs), 0, mem.shape[1], ptr(rs), 0, mem.shape[1], h, m, ptr(wd), 1e-6, ptr(hs), mem.shape[1],
             0, None, None, ptr(ys), 0, mem.shape[1], stream())
    ho, y, _, _ = run_rms(x, r, w, out="y")
    torch.cuda.synchronize()
    assert torch.equal(hs, ho) and torch.equal(ys, y)
    assert torch.equal(xs.cpu(), x) and torch.equal(rs.cpu(), r) and torch.isnan(mem[:, 2 * h:2 * h + gap]).all()
