"""The beam search's operators as they are used: together over several steps, in
graphs, on two streams at once, over one workspace, in caches past 2^32 elements."""
import ctypes

import numpy as np
import pytest
import torch

import s2x
from decode_util import TYPES, Cache, attn_ref
from gpu_util import assert_same, dev, empty, host, ptr, say, stream
from test_gpu_decode import NAN, U, Q4, q4_weight, within
from test_gpu_search import beam_case, beams_case, check_beam, check_rms, compare, ints, nans, prefix_inputs, rms_case, run_beam, run_fork, run_prefix, run_rms

pytestmark = pytest.mark.gpu


class Search:
    """A one-layer model under beam search, over buffers that stay: every call of
    a step in the documented order."""

    def __init__(self, n_req, beams, prompt, hq, hkv, d, hidden, vocab, page, steps, kind):
        rng = np.random.default_rng(5)
        self.n_req, self.beams, self.hq, self.hkv, self.d = n_req, beams, hq, hkv, d
        self.hidden, self.vocab, self.page, self.kind = hidden, vocab, page, kind
        n = self.n = n_req * beams
        self.wide, self.ctx_w = (hq + 2 * hkv) * d, hq * d
        self.qkv, self.o, self.head = (Q4(*q4_weight(rng, a, b)) for a, b in
                                       ((self.wide, hidden), (hidden, self.ctx_w), (vocab, hidden)))
        self.max_own = steps + prompt % page + page
        per = -(-(prompt + steps + 1) // page)
        n_pages = n_req * (prompt // page) + n * (per - prompt // page + 2)
        self.cache = Cache(n_pages, hkv, page, d, kind)
        for c in (self.cache.k, self.cache.v):
            c.copy_(torch.randn(c.shape, device="cuda:0"))
        # the prompts: every beam of a request on the same pages, the open one too
        ids = rng.permutation(n_pages).astype(np.int32)
        held = -(-prompt // page)
        table = np.full((n, per), -1, np.int32)
        for s in range(n):
            table[s, :held] = ids[s // beams * held:(s // beams + 1) * held]
        i32, i64, f32 = torch.int32, torch.int64, torch.float32
        self.table, self.table2 = ints(table), empty((n, per), i32)
        self.len, self.len_out, self.pos = ints(np.full(n, prompt)), empty((n,), i32), empty((n,), i32)
        self.new, self.start = ints(np.ones(n)), empty((n + 1,), i32)
        self.slots, self.used = empty((n,), i64), empty((2,), i64)
        self.free = torch.full((n_pages,), -1, dtype=i32, device="cuda:0")
        self.count = empty((2,), i64)
        self.copy = empty((3, n), i32)
        self.parent, self.token, self.score = ints(np.arange(n)), empty((n,), i32), dev(np.zeros(n, np.float32))
        self.scores = dev(np.where(np.arange(n) % beams == 0, 0.0, -np.inf).astype(np.float32))
        self.group = ints(np.arange(0, n + 1, beams))
        self.plen = ints(np.full(n_req, prompt // page * page))
        self.max_prefix = prompt // page * page
        self.x, self.res, self.h = (torch.zeros(n, hidden, device="cuda:0") for _ in range(3))
        self.wn = dev(rng.normal(1, 0.1, hidden).astype(np.float32))
        self.wq, self.wk = (dev(rng.normal(1, 0.1, d).astype(np.float32)) for _ in range(2))
        self.freq = dev(10000.0 ** (-np.arange(0, d, 2) / d))
        self.planes = [(empty((n, k), torch.int8), empty((n, k // 32), i32)) for k in (hidden, self.ctx_w, hidden)]
        self.y, self.q = empty((n, self.wide), f32), empty((n, self.ctx_w), TYPES[kind])
        self.ctx, self.out, self.logits = empty((n, self.ctx_w), f32), empty((n, hidden), f32), empty((n, vocab), f32)
        lib = s2x.lib
        self.ws = [torch.full((max(1, z),), 0xff, dtype=torch.uint8, device="cuda:0") for z in (
            lib.s2x_kv_pages_workspace_size(n_pages),
            lib.s2x_attn_paged_prefix_workspace_size(n_req, beams, self.max_prefix, self.max_own, hq, hkv, d),
            lib.s2x_beam_select_workspace_size(n_req, beams, vocab, beams))]

    def fork(self):
        """Rows by self.parent: the tables in their new order, open pages apart."""
        n, st, c = self.n, stream(), self.cache
        src, dst, tok = self.copy
        s2x.call("s2x_kv_fork", ptr(self.parent), n, ptr(self.len), ptr(self.table), n, self.table.shape[1], self.page, c.n_pages,
                 None, ptr(self.table2), self.table.shape[1], ptr(self.len_out), ptr(src), ptr(dst), ptr(tok), ptr(self.free),
                 ptr(self.count), ptr(self.ws[0]), self.ws[0].numel(), st)
        s2x.call("s2x_kv_copy_pages", c.ref(), 1, ptr(src), ptr(dst), ptr(tok), n, None, st)
        self.table.copy_(self.table2)
        self.len.copy_(self.len_out)

    def step(self):
        n, st, c, (q0, d0), (q1, d1), (q2, d2) = self.n, stream(), self.cache, *self.planes
        h, w = self.ctx_w, self.hidden
        self.fork()
        s2x.call("s2x_kv_slots", ptr(self.len), ptr(self.new), n, ptr(self.free), self.free.numel(), self.page, c.n_pages,
                 ptr(self.table), self.table.shape[1], n, ptr(self.len_out), ptr(self.start), ptr(self.pos), ptr(self.slots),
                 ptr(self.used), st)
        s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(self.x), 0, w, ptr(self.res), 0, w, w, n, ptr(self.wn), 1e-6, ptr(self.h), w,
                 w, ptr(q0), ptr(d0), None, 0, 0, st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.qkv.h, ptr(q0), ptr(d0), n, ptr(self.y), self.wide, None, None, 0, st)
        s2x.call("s2x_qk_norm_rope_kv", ptr(self.y), 0, self.wide, n, self.hq, ptr(self.wq), ptr(self.wk), 1e-6, ptr(self.freq),
                 self.d, 0, ptr(self.pos), ptr(self.slots), ptr(self.q), h, c.ref(), st)
        s2x.call("s2x_attn_paged_prefix", ptr(self.q), h, n, ptr(self.start), c.ref(), ptr(self.table), self.table.shape[1],
                 ptr(self.len_out), n, ptr(self.group), ptr(self.plen), self.n_req, self.beams, self.max_prefix, self.max_own,
                 self.hq, self.d ** -0.5, ptr(self.ctx), 0, h, None, ptr(self.ws[1]), self.ws[1].numel(), st)
        s2x.call("s2x_quantize_q8_1", ptr(self.ctx), h, n, h, h, ptr(q1), ptr(d1), st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.o.h, ptr(q1), ptr(d1), n, ptr(self.out), w, None, None, 0, st)
        s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(self.out), 0, w, ptr(self.h), 0, w, w, n, ptr(self.wn), 1e-6, ptr(self.res), w,
                 w, ptr(q2), ptr(d2), None, 0, 0, st)
        s2x.call("s2x_mul_mat_q4_0_q8_1", self.head.h, ptr(q2), ptr(d2), n, ptr(self.logits), self.vocab, None, None, 0, st)
        s2x.call("s2x_beam_select", ptr(self.logits), 0, self.vocab, self.n_req, self.beams, self.vocab, ptr(self.scores), None, 0,
                 self.beams, ptr(self.parent), ptr(self.token), ptr(self.score), ptr(self.ws[2]), self.ws[2].numel(), st)
        self.scores.copy_(self.score)
        self.len.copy_(self.len_out)


def tokens_of(s, lens, table):
    """Keys and values that each row's table gives, (len, hkv, d) each."""
    k, v = (host(c.float()) for c in (s.cache.k, s.cache.v))
    out = []
    for n, row in zip(lens, table):
        t = np.arange(n)
        out.append((k[row[t // s.page], :, t % s.page], v[row[t // s.page], :, t % s.page]))
    return out


@pytest.mark.parametrize("n_req,beams,prompt,hq,hkv,d,kind", [
    (3, 4, 37, 8, 2, 64, "f16"), (2, 6, 48, 4, 4, 72, "bf16"), (1, 24, 200, 8, 2, 128, "f16"), (4, 1, 5, 8, 8, 64, "bf16")])
def test_search(n_req, beams, prompt, hq, hkv, d, kind):
    """Twenty steps: each beam's keys and values are those of its own history,
    whatever beams came and went, its context that of 64 bits over them, the pages
    held and free all pages, no page lost."""
    s = Search(n_req, beams, prompt, hq, hkv, d, 288, 1003, 16, 20, kind)
    rng = np.random.default_rng(8)
    say(f"search: {n_req} x {beams}, prompt {prompt}, {hq}/{hkv} x {d} {kind}")
    torch.cuda.synchronize()
    n = s.n
    history = tokens_of(s, [prompt] * n, host(s.table))
    for i in range(20):
        s.x.copy_(dev(rng.standard_normal((n, 288)).astype(np.float32)))
        s.res.copy_(dev(rng.standard_normal((n, 288)).astype(np.float32)))
        parent = host(s.parent).copy()
        s.step()
        torch.cuda.synchronize()
        lens, table = host(s.len), host(s.table)
        assert (lens == prompt + i + 1).all()
        now = tokens_of(s, lens, table)
        for b in range(n):
            for a, (old, new) in enumerate(zip(history[parent[b]], now[b])):
                assert_same(new[:-1], old, f"step {i} beam {b} {'kv'[a]}")
        ref, size, _, top, _ = attn_ref(host(s.q.float()).reshape(n, hq, d), s.cache, table, lens, 1 << 20, d ** -0.5, 0)
        tol = (2 * (d + 6) * U * top + {"f16": 2.0 ** -20, "bf16": 2.0 ** -21}[kind] + 2 * (lens.max() + 8) * U)[:, :, None] * size
        within(host(s.ctx).reshape(n, hq, d), ref, tol, f"step {i} context")
        # the last page of every row is its own; held and free pages are all pages
        last = table[np.arange(n), (lens - 1) // 16]
        assert len(set(last.tolist())) == n
        taken, spare = int(host(s.used)[0]), int(host(s.count)[0])
        held = set(table[table >= 0].tolist())
        free = host(s.free)[taken:spare].tolist()
        assert not held & set(free) and len(held) + len(free) == s.cache.n_pages
        history = now
    # scores are sums of log-probabilities, best first, and finite
    score = host(s.score).reshape(n_req, beams)
    assert np.isfinite(score).all() and (np.diff(score, axis=1) <= 0).all()


def captured(f):
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        f()
    torch.cuda.current_stream().wait_stream(st)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f()
    return graph


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_search_captured(kind):
    """The whole step in a graph, replayed with eager work between, against eager
    steps over buffers of their own: the same bits at every step."""
    a, b = (Search(3, 5, 70, 8, 2, 128, 1152, 5003, 16, 12, kind) for _ in range(2))
    start = {k: v.clone() for k, v in vars(b).items() if isinstance(v, torch.Tensor)}
    for x, y in zip(a.cache.mem, b.cache.mem):
        y.copy_(x)
    mem = [m.clone() for m in b.cache.mem]
    graph = captured(a.step)
    for k, v in start.items():
        getattr(a, k).copy_(v)
    for m, old in zip(a.cache.mem, mem):
        m.copy_(old)
    rng = np.random.default_rng(9)
    for i in range(10):
        x, r = (dev(rng.standard_normal((15, 1152)).astype(np.float32)) for _ in range(2))
        for s in (a, b):
            s.x.copy_(x)
            s.res.copy_(r)
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        torch.cuda.synchronize()
        for name in ("table", "len", "copy", "free", "count", "parent", "token", "score", "ctx", "logits", "res", "h"):
            assert torch.equal(getattr(a, name), getattr(b, name)), (i, name)
        for m0, m1 in zip(a.cache.mem, b.cache.mem):
            assert torch.equal(m0.view(torch.int16), m1.view(torch.int16)), i
        torch.randn(1000, 1000, device="cuda:0").sum()  # eager work between replays


def test_two_graphs_over_one_workspace():
    """Two captured calls of each operator over the same workspace, replayed in
    turn: nothing of one is left for the other."""
    rng = np.random.default_rng(2)
    cases = [prefix_inputs(rng, g, 8, 2, 128, "f16", 16, "head") for g in
             ([(700, [30, 5, 60]), (90, [3, 4])], [(333, [9] * 12), (1200, [100])])]
    want = [run_prefix(c[0], c[1], c[2], c[4], c[5], c[6], 0.09, "f32", max_group=12, max_prefix=1200, max_own=100) for c in cases]
    size = s2x.lib.s2x_attn_paged_prefix_workspace_size(2, 12, 1200, 100, 8, 2, 128)
    ws, graphs, outs = empty((size,), torch.uint8), [], []
    keep = []
    for q, cache, table, _, lens, starts, plen in cases:
        n = len(lens)
        t = [q.to("cuda:0"), ints(table), ints(lens), ints(starts), ints(plen), nans(n, 8, 128), nans(n, 8)]
        keep.append(t)

        def call(t=t, n=n, cache=cache):
            s2x.call("s2x_attn_paged_prefix", ptr(t[0]), 1024, n, None, cache.ref(), ptr(t[1]), t[1].shape[1], ptr(t[2]), n,
                     ptr(t[3]), ptr(t[4]), 2, 12, 1200, 100, 8, 0.09, ptr(t[5]), 0, 1024, ptr(t[6]), ptr(ws), size, stream())
        graphs.append(captured(call))
        outs.append(t[5:])
    for i in range(4):
        for g, o, (ref, lse) in zip(graphs, outs, want):
            o[0].fill_(NAN)
            g.replay()
            torch.cuda.synchronize()
            assert_same(host(o[0]).astype(np.float64), ref, f"round {i}")
            assert_same(host(o[1]), lse, f"round {i}")
            torch.randn(500, 500, device="cuda:0").sum()
    # the selection
    size = s2x.lib.s2x_beam_select_workspace_size(4, 3, 9001, 6)
    ws, graphs, outs, want = empty((size,), torch.uint8), [], [], []
    for seed in (1, 2):
        x, sc = beam_case(seed, 4, 3, 9001, "bf16")
        want.append(run_beam(x, sc, 6))
        t = [x.to("cuda:0"), dev(sc), empty((4, 6), torch.int32), empty((4, 6), torch.int32), empty((4, 6), torch.float32)]
        keep.append(t)

        def call(t=t):
            s2x.call("s2x_beam_select", ptr(t[0]), s2x.TYPE_BF16, 9001, 4, 3, 9001, ptr(t[1]), None, 0, 6, ptr(t[2]), ptr(t[3]),
                     ptr(t[4]), ptr(ws), size, stream())
        graphs.append(captured(call))
        outs.append(t[2:])
    for i in range(4):
        for g, o, w in zip(graphs, outs, want):
            for z in o:
                z.zero_()
            g.replay()
            torch.cuda.synchronize()
            for z, r in zip(o, w):
                assert_same(host(z), r, f"round {i}")


def test_repeats_and_streams():
    """Every operator on two streams at once, each over a workspace of its own, many
    times: the bits of the call alone."""
    rng = np.random.default_rng(3)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    handles = [ctypes.c_void_p(s.cuda_stream) for s in streams]
    x, sc = beam_case(3, 6, 4, 20011, "f16")
    p = prefix_inputs(rng, [(900, [30, 5, 60, 1] * 5)], 8, 2, 128, "bf16", 16, "head")
    f = beams_case(rng, 50, 6, 400, 60, 16, 3000)
    r = rms_case(4, 33, 2100, "f32", "f32")
    want = [run_beam(x, sc, 8), run_prefix(p[0], p[1], p[2], p[4], p[5], p[6], 0.1, "bf16"), run_fork(*f)]
    first = run_rms(*r, out="q8 y")
    for i in range(6):
        st = handles[i % 2]
        for got, ref in ((run_beam(x, sc, 8, st=st), want[0]),
                         (run_prefix(p[0], p[1], p[2], p[4], p[5], p[6], 0.1, "bf16", st=st), want[1])):
            for g, w in zip(got, ref):
                assert_same(g, w, f"repeat {i}")
        for a, b in zip(run_rms(*r, out="q8 y"), first):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    # at once: launches on both streams before any wait
    sets = []
    for i in range(8):
        xs, scs = beam_case(20 + i, 3, 4, 20011, "f32")
        size = s2x.lib.s2x_beam_select_workspace_size(3, 4, 20011, 8)
        sets.append((xs, scs, [xs.to("cuda:0"), dev(scs), empty((3, 8), torch.int32), empty((3, 8), torch.int32),
                               empty((3, 8), torch.float32), empty((size,), torch.uint8)], size))
    torch.cuda.synchronize()
    for i, (_, _, t, size) in enumerate(sets):
        s2x.call("s2x_beam_select", ptr(t[0]), 0, 20011, 3, 4, 20011, ptr(t[1]), None, 0, 8, ptr(t[2]), ptr(t[3]), ptr(t[4]),
                 ptr(t[5]), size, handles[i % 2])
    torch.cuda.synchronize()
    for xs, scs, t, _ in sets:
        for z, w in zip(t[2:5], run_beam(xs, scs, 8)):
            assert_same(host(z), w, "at once")


def test_cache_past_32_bits():
    """A cache of 2^33 elements a plane (pages 2^29 apart): copies between its ends and
    the attention over a prefix there."""
    n_pages, ldp, page, d = 17, 1 << 29, 64, 128
    mem = [torch.zeros((n_pages - 1) * ldp + page * d, dtype=torch.float16, device="cuda:0") for _ in range(2)]
    views = [torch.as_strided(m, (n_pages, 1, page, d), (ldp, page * d, d, 1)) for m in mem]
    for v in views:
        v[:] = torch.randn(v.shape, device="cuda:0").half()
    c = s2x.KVCache(k=mem[0].data_ptr(), v=mem[1].data_ptr(), type=s2x.TYPE_F16, page_size=page, n_pages=n_pages, n_head=1, d_head=d,
                    ld_page=ldp, ld_head=page * d, ld_tok=d)
    src, dst = ints([16, 0, 13]), ints([1, 15, 2])
    before = [v.clone() for v in views]
    s2x.call("s2x_kv_copy_pages", ctypes.byref(c), 1, ptr(src), ptr(dst), None, 3, None, stream())
    torch.cuda.synchronize()
    for v, b in zip(views, before):
        for a, z in ((16, 1), (0, 15), (13, 2)):
            b[z] = b[a]
        assert torch.equal(v, b)

    class Far:
        def __init__(self):
            (self.k, self.v), self.n_head, self.n_pages, self.kind, self.page = views, 1, n_pages, "f16", page

        def ref(self):
            return ctypes.byref(c)
    cache = Far()
    table = np.array([[16, 15, 3, 14, -1], [16, 15, 3, 9, 12]], np.int32)
    lens = np.array([230, 300])
    q = torch.randn(2, 24, d).half()
    for hq in (4, 24):
        got, lse = run_prefix(q[:, :hq].contiguous(), cache, table, lens, np.array([0, 2]), np.array([192]), 0.09, "f32")
        compare(got, lse, q[:, :hq], cache, table, lens, 0.09, "f32")


@pytest.mark.parametrize("share,size,d,kind", [(2, 5, 128, "f16"), (1, 3, 72, "bf16"), (2, 20, 64, "bf16"), (4, 40, 128, "f16"),
                                               (4, 33, 128, "bf16"), (3, 9, 256, "f16"), (8, 6, 200, "bf16")])
@pytest.mark.parametrize("what", [NAN, np.inf])
def test_prefix_unseen_tokens(share, size, d, kind, what):
    """Tokens of the prefix that a shorter sequence does not see, whatever they are:
    NaN or infinite keys and values that others see, or none."""
    rng = np.random.default_rng(size)
    p, at = 700, 333
    owns = [int(x) for x in rng.integers(0, 30, size)]
    short = {1: at - p, 2: at - 13 - p, 0: -p}  # sees up to the bad token, the tile before, nothing
    if size > 8:
        short[size - 1] = short[size // 2] = at - 1 - p
    for s, o in short.items():
        owns[s] = o
    q, cache, table, ref, lens, starts, plen = prefix_inputs(rng, [(p, owns)], 2 * share, 2, d, kind, 16, "head")
    for c in (cache.k, cache.v):
        c[int(ref[0, at // 16]), :, at % 16] = what
    cache.v[int(ref[0, (at + 300) // 16]), :, 3] = what
    got, lse = run_prefix(q, cache, table, lens, starts, plen, 0.1, "f32")
    rows = np.array(sorted(short))
    compare(got[rows], lse[rows], q[rows], cache, ref[rows], lens[rows], 0.1, "f32")
    assert (got[0] == 0).all() and (lse[0] == -np.inf).all()
    others = np.setdiff1d(np.arange(size), rows)
    assert np.isnan(got[others]).all(axis=2).all()
    # no sequence as long as the prefix: nothing behind the longest is a token
    lens = np.minimum(lens, at)
    got, lse = run_prefix(q, cache, table, lens, starts, plen, 0.1, "f32")
    compare(got, lse, q, cache, ref, lens, 0.1, "f32")
    # a bad value that a shorter sequence does see, and only that
    bad = torch.zeros_like(cache.v[0, :, 0, 0])
    bad[0] = what
    cache.v[int(ref[0, 20]), :, 2, 1] = bad
    lens = np.where(np.arange(size) % 2, lens, np.minimum(lens, 322))
    got, lse = run_prefix(q, cache, table, lens, starts, plen, 0.1, "f32")
    sees = lens > 322
    clean = got.copy()
    clean[sees, :share, 1] = 0
    assert not np.isfinite(got[sees, :share, 1]).any() and np.isfinite(clean).all() and np.isfinite(lse[lens > 0]).all()
    rows = np.flatnonzero(~sees)
    compare(got[rows], lse[rows], q[rows], cache, ref[rows], lens[rows], 0.1, "f32")


@pytest.mark.parametrize("m,h", [((1 << 22) + 4099, 8), ((1 << 20) + 777, 520)])
def test_rms_more_rows_than_workgroups(m, h):
    x = torch.randn(m, h, device="cuda:0").half()
    w = torch.randn(h, device="cuda:0")

    def run(x):
        n, k_pad = len(x), -(-h // 32) * 32
        out = nans(n, h, dtype=torch.float16), empty((n, k_pad), torch.int8), empty((n, k_pad // 32), torch.int32)
        s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(x), s2x.TYPE_F16, h, ptr(x), s2x.TYPE_F16, h, h, n, ptr(w), 1e-5, None, 0, k_pad,
                 ptr(out[1]), ptr(out[2]), ptr(out[0]), s2x.TYPE_F16, h, stream())
        return out
    whole = run(x)
    for a, b in ((0, 5000), (m // 2, m // 2 + 70000), (m - 9000, m)):
        for g, w_ in zip(whole, run(x[a:b].clone())):
            assert torch.equal(g[a:b], w_), (a, b)
    y = 2 * x.double()
    y = y / torch.sqrt((y * y).mean(1, keepdim=True) + 1e-5) * w.double()
    # (an eps of f32, inv and two products of f32, the rounding to f16)
    assert ((whole[0].double() - y).abs() <= (2.0 ** -11 + 4 * U) * y.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("m", [1, 7, 131])
@pytest.mark.parametrize("h", [8, 63, 64, 65, 127, 128, 129, 255, 256, 257, 4097, 8192, 8193])
def test_rms_widths_around_the_rules(m, h):
    """Rows of an eighth of a wave and up, the last workgroup not full."""
    for x_kind, r_kind in (("f32", "f32"), ("bf16", "bf16")):
        check_rms(*rms_case(m * h, m, h, x_kind, r_kind))


def test_rms_rows_far_apart():
    """Rows 2^32 elements apart, the largest stride."""
    far, h = 1 << 32, 1157
    mem = torch.zeros(2 * far + h, dtype=torch.float16, device="cuda:0")
    rows = torch.as_strided(mem, (3, h), (far, 1))
    x, r, w = rms_case(1, 3, h, "f16", "f16")
    rows.copy_(x)
    wd, rd, y = dev(w), r.to("cuda:0"), nans(3, h)
    s2x.call("s2x_add_rmsnorm_quantize_q8_1", ptr(mem), s2x.TYPE_F16, far, ptr(rd), s2x.TYPE_F16, h, h, 3, ptr(wd), 1e-6, ptr(mem), far,
             0, None, None, ptr(y), 0, h, stream())
    near, want, _, _ = run_rms(x, r, w, out="y")
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(rows, near)
    assert not mem[h:far].any() and not mem[far + h:2 * far].any()


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_beam_many_long_rows(kind):
    """The longest parts of rows with the most continuations: the largest lists."""
    n, beams, vocab = 40, 8, 131072
    g = torch.Generator(device="cuda:0").manual_seed(3)
    x = torch.randn(n, beams, vocab, device="cuda:0", generator=g).to(TYPES[kind])
    x[1], x[2] = 1.5, torch.arange(vocab, device="cuda:0") / 2048  # (all equal; ascending)
    sc = -np.arange(n * beams, dtype=np.float32).reshape(n, beams) % 7
    got = run_beam(x, sc, 64)
    for r in (0, 1, 2, n - 1):
        one = run_beam(x[r:r + 1].clone(), sc[r:r + 1], 64)
        assert_same(got[0][r], one[0][0] + r * beams, f"parent {r}")
        assert_same(got[1][r], one[1][0], f"token {r}")
        # (other parts of a row: other orders of its sum)
        assert np.allclose(got[2][r], one[2][0], rtol=0, atol=2 * (128 + 60) * U + 4 * U * 20)
    check_beam(x[3:5].cpu(), sc[3:5], 64)


@pytest.mark.parametrize("n,beams,vocab,kind,n_out", [(2, 32, 40000, "f32", 64), (1, 64, 100000, "bf16", 64), (3, 9, 270000, "f16", 60)])
def test_beam_joins_of_many_candidates(n, beams, vocab, kind, n_out):
    """More candidates than a round of the join takes, of 256 threads and of 1,024; equal
    ones among them."""
    x, sc = beam_case(beams, n, beams, vocab, kind)
    check_beam(x, sc, n_out)
    x[:], sc[:] = 0.5, -3.0
    parent, token, score = run_beam(x, sc, n_out)
    assert (parent == np.arange(n)[:, None] * beams).all() and (token == np.arange(n_out)).all()


def test_prefix_most_sequences():
    """65,535 sequences, more own tokens' parts than workgroups."""
    n, h, d, page, own = 65535, 32, 64, 16, 300
    rng = np.random.default_rng(6)
    cache = Cache(500, h, page, d, "f16")
    for c in (cache.k, cache.v):
        c.copy_(torch.randn(c.shape, device="cuda:0"))
    lens = rng.integers(0, own + 1, n)
    lens[-1], lens[0] = own, 1
    table = rng.integers(0, 500, (n, -(-own // page))).astype(np.int32)
    q = torch.randn(n, h * d, device="cuda:0").half()
    t = [ints(a) for a in (table, lens, np.arange(0, n + 1, 3), np.zeros(n // 3))]
    size = s2x.lib.s2x_attn_paged_prefix_workspace_size(n // 3, 3, 0, own, h, h, d)
    say(f"prefix: {n} sequences, workspace {size >> 20} MiB")
    ws, out, lse = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda:0"), nans(n, h * d, dtype=torch.float16), nans(n, h)
    s2x.call("s2x_attn_paged_prefix", ptr(q), h * d, n, None, cache.ref(), ptr(t[0]), table.shape[1], ptr(t[1]), n, ptr(t[2]), ptr(t[3]),
             n // 3, 3, 0, own, h, 0.1, ptr(out), s2x.TYPE_F16, h * d, ptr(lse), ptr(ws), size, stream())
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()
    rows = np.concatenate([[0, 1, 2, n - 2, n - 1], rng.integers(0, n, 60)])
    at = torch.from_numpy(rows).to("cuda:0")
    compare(out[at].double().cpu().numpy().reshape(-1, h, d), host(lse[at]), q[at].cpu().reshape(-1, h, d), cache, table[rows], lens[rows],
            0.1, "f16")
