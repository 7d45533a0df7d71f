"""The operators of a beam search over a paged cache, each in its plain form and
through the library.

A generating model that searches with beams runs, beside the products, the
cache's slots and the norms of a decode step: the norm between two products,
with the residual's addition and the next product's 8-bit activation (`rms`),
the selection of the next beams over all beams and the vocabulary (`beam`), the
beams' block tables in their new order with the pages that two of them would
write to copied, or a cache's pages moved to its front (`pages`), and the
attention of beams, or of requests under one system prompt, whose first tokens
are the same (`prefix`).  `run` computes them with elementary torch operations
where `own` is false and calls the library's entry points (include/s2x.h) where
it is true.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # s2x_type
EPS = 1e-6
DONE_TOKEN = 1


def listed():
    return [
        # the norm before the QKV product of one sequence's token, at the
        # encoder's own width
        {"name": "rms_1x1152", "op": "rms", "rows": 1, "h": 1152, "x": "f32", "res": "f32", "out": "q8"},
        # a batch of sequences' tokens, a width that is no multiple of 32
        {"name": "rms_130x4304", "op": "rms", "rows": 130, "h": 4304, "x": "f32", "res": "f32", "out": "q8"},
        # a prompt's rows in 16 bits, for a product in 16 bits
        {"name": "rms_8191x4096", "op": "rms", "rows": 8191, "h": 4096, "x": "bf16", "res": "bf16", "out": "bf16"},
        # one request's beams: latency
        {"name": "beam_1x4x32000", "op": "beam", "n_req": 1, "n_beam": 4, "vocab": 32000, "n_out": 4, "x": "f32",
         "done": False},
        # a batch of searches, an odd vocabulary, spare candidates for beams that end
        {"name": "beam_13x5x50021", "op": "beam", "n_req": 13, "n_beam": 5, "vocab": 50021, "n_out": 10, "x": "f16",
         "done": True},
        # the text tower's vocabulary under a large batch
        {"name": "beam_64x8x256000", "op": "beam", "n_req": 64, "n_beam": 8, "vocab": 256000, "n_out": 16, "x": "bf16",
         "done": True},
        # one request's four beams in their new order, a small model's layers
        {"name": "fork_1x4", "op": "pages", "how": "fork", "n_req": 1, "n_beam": 4, "prompt": 300, "len_max": 340, "page": 16,
         "spare": 64, "layers": 2, "hkv": 16, "d": 72, "type": "f16", "by": "head"},
        # a batch of searches over long prompts
        {"name": "fork_60x8", "op": "pages", "how": "fork", "n_req": 60, "n_beam": 8, "prompt": 3000, "len_max": 3400,
         "page": 32, "spare": 2000, "layers": 4, "hkv": 8, "d": 128, "type": "bf16", "by": "head"},
        # a cache after many requests came and went, its pages moved to the front
        {"name": "compact_150", "op": "pages", "how": "compact", "n_req": 150, "n_beam": 1, "prompt": 0, "len_max": 2500,
         "page": 16, "spare": 6000, "layers": 3, "hkv": 8, "d": 128, "type": "f16", "by": "token"},
        # the beams of three requests, the encoder's head layout, f32 context for the quantizer
        {"name": "prefix_3x4_16x72", "op": "prefix", "n_group": 3, "group_max": 4, "equal": True, "prefix_max": 700,
         "own_max": 60, "hq": 16, "hkv": 16, "d": 72, "type": "f16", "out": "f32", "page": 16, "by": "head"},
        # requests under a few system prompts, ragged groups, small pages, token-major cache
        {"name": "prefix_9_ragged", "op": "prefix", "n_group": 9, "group_max": 30, "equal": False, "prefix_max": 6000,
         "own_max": 900, "hq": 32, "hkv": 8, "d": 128, "type": "f16", "out": "f16", "page": 16, "by": "token"},
        # one long document, many questions
        {"name": "prefix_1x64_long", "op": "prefix", "n_group": 1, "group_max": 64, "equal": True, "prefix_max": 32001,
         "own_max": 500, "hq": 32, "hkv": 8, "d": 128, "type": "bf16", "out": "bf16", "page": 64, "by": "head"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rms", "rms", "beam", "beam", "pages", "pages", "prefix", "prefix", "prefix"])
    if op == "rms":
        h = _log_int(rng, 64, 16384)
        kind = rng.choice(["f32", "f16", "bf16"])
        return {"op": op, "rows": _log_int(rng, 1, max(1, 8191 * 4096 // (h * (2 if kind == "f32" else 1)))), "h": h,
                "x": kind, "res": rng.choice(["f32", kind, "none"]), "out": rng.choice(["q8", "q8", kind])}
    if op == "beam":
        vocab = _log_int(rng, 1000, 256000)
        kind = rng.choice(["f32", "f16", "bf16"])
        n_beam = rng.choice([1, 2, 3, 4, 5, 8, 12, 16, 32])
        most = 64 * 8 * 256000 // (vocab * n_beam * (2 if kind == "f32" else 1))
        return {"op": op, "n_req": _log_int(rng, 1, max(1, min(most, 400 // n_beam + 60))), "n_beam": n_beam, "vocab": vocab,
                "n_out": n_beam * rng.choice([1, 2]), "x": kind, "done": rng.random() < 0.5}
    if op == "pages":
        how = rng.choice(["fork", "fork", "compact"])
        n_beam = rng.choice([2, 3, 4, 5, 8, 12]) if how == "fork" else 1
        n_req = _log_int(rng, 1, 480 // n_beam)
        page = rng.choice([16, 16, 32, 64])
        prompt = _log_int(rng, 20, 4000) if how == "fork" else 0
        len_max = prompt + _log_int(rng, 10, 500) if how == "fork" else _log_int(rng, 50, 4000)
        hkv, d = rng.choice([(16, 72), (8, 128), (8, 64), (4, 128), (2, 256)])
        # (the cache within 0.8 GB)
        most = 100_000 // (page * hkv * d * 4 // 8192)
        held = n_req * (prompt // page + n_beam * (2 + (len_max - prompt) // page))
        n_req = max(1, n_req * most // held) if held > most else n_req
        return {"op": op, "how": how, "n_req": n_req, "n_beam": n_beam, "prompt": prompt, "len_max": len_max, "page": page,
                "spare": _log_int(rng, 16, 2000) + n_req * n_beam, "layers": rng.choice([1, 2, 3]), "hkv": hkv, "d": d,
                "type": rng.choice(["f16", "bf16"]), "by": rng.choice(["head", "token"])}
    hkv = rng.choice([1, 2, 4, 8, 16])
    hq = hkv * rng.choice([1, 1, 2, 4, 4, 8])
    n_group = _log_int(rng, 1, 40)
    group = _log_int(rng, 1, max(1, min(64, 120 // n_group)))
    d = rng.choice([64, 72, 96, 128, 128, 192, 256])
    most = 32001 * 64 * 32 * 128 // (n_group * group * hq * d)
    own_max = _log_int(rng, 1, 1000)
    return {"op": op, "n_group": n_group, "group_max": group, "equal": rng.random() < 0.5,
            "prefix_max": _log_int(rng, 10, max(11, min(32001, most, 300_000 // n_group))), "own_max": own_max, "hq": hq,
            "hkv": hkv, "d": d, "type": (kind := rng.choice(["f16", "bf16"])), "out": rng.choice(["f32", kind]),
            "page": rng.choice([8, 16, 32, 64, 128]), "by": rng.choice(["head", "token"])}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 31)
    return g


def _normal(g, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=g, device=DEV) * std + mean


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(n, page):
    return -(-n // page)


def _cache(case, layers, n_pages, g):
    """Keys and values of the layers: (layers, pages, heads, page, d) by head,
    (layers, pages, page, heads, d) by token, both seen as the first."""
    shape = (layers, n_pages, case["hkv"], case["page"], case["d"])
    if case["by"] == "token":
        shape = (layers, n_pages, case["page"], case["hkv"], case["d"])
    out = []
    for _ in range(2):
        t = torch.empty(shape, dtype=TYPES[case["type"]], device=DEV).normal_(generator=g)
        out.append(t if case["by"] == "head" else t.transpose(2, 3))
    return out


def _group_sizes(case):
    r = random.Random(f"groups {case['n_group']} {case['group_max']} {case['equal']}")
    if case["equal"]:
        return [case["group_max"]] * case["n_group"]
    sizes = [_log_int(r, 1, case["group_max"]) for _ in range(case["n_group"])]
    sizes[0] = case["group_max"]
    return sizes


def _prefix_lens(case):
    """Tokens that each group shares, and each sequence's own behind them."""
    r = random.Random(f"prefix {case['n_group']} {case['prefix_max']} {case['own_max']}")
    prefix = [_log_int(r, max(1, case["prefix_max"] // 8), case["prefix_max"]) for _ in range(case["n_group"])]
    prefix[0] = case["prefix_max"]
    own_len = [[_log_int(r, 1, case["own_max"]) for _ in range(n)] for n in _group_sizes(case)]
    own_len[0][0] = case["own_max"]
    return prefix, own_len


def _page_lens(case):
    """Lengths of the sequences: each request's beams within one token of one
    another, none a request that has ended."""
    r = random.Random(f"pages {case['how']} {case['n_req']} {case['n_beam']} {case['len_max']}")
    out = []
    for i in range(case["n_req"]):
        lo = max(1, case["prompt"], case["len_max"] // 10)
        n = case["len_max"] if i == 0 else _log_int(r, min(lo, case["len_max"]), case["len_max"])
        out += [0 if case["how"] == "compact" and i % 11 == 10 else n] * case["n_beam"]
    return out


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case}
    if op == "rms":
        m, h = case["rows"], case["h"]
        k_pad = _pages(h, 32) * 32
        s["x"] = _normal(g, m, h).to(TYPES[case["x"]])
        if case["res"] != "none":
            # a residual stream with a few large channels
            s["resid"] = (_normal(g, m, h, std=2.0) * torch.exp(0.7 * _normal(g, h))).to(TYPES[case["res"]])
        s["w"] = _normal(g, h, std=0.2, mean=1.0)
        if own:
            if case["res"] != "none":
                s["h"] = torch.empty(m, h, dtype=TYPES[case["res"]], device=DEV)
            if case["out"] == "q8":
                s["q"] = torch.empty(m, k_pad, dtype=torch.int8, device=DEV)
                s["ds"] = torch.empty(m, k_pad // 32, 2, dtype=torch.float16, device=DEV)
            else:
                s["y"] = torch.empty(m, h, dtype=TYPES[case["out"]], device=DEV)
        return s
    if op == "beam":
        n, beams, vocab = case["n_req"], case["n_beam"], case["vocab"]
        x = torch.empty(n * beams, vocab, device=DEV).normal_(generator=g).mul_(2.5)
        x[:, torch.randint(0, vocab, (vocab // 100 + 1,), generator=g, device=DEV)] = -math.inf  # tokens that may not follow
        s["logits"] = x.to(TYPES[case["x"]])
        s["scores"] = -5.0 - 20.0 * torch.rand(n, beams, generator=g, device=DEV)
        if case["done"]:
            s["done"] = (torch.rand(n, beams, generator=g, device=DEV) < 0.15).to(torch.uint8)
        if own:
            s["out"] = [torch.empty(n, case["n_out"], dtype=t, device=DEV)
                        for t in (torch.int32, torch.int32, torch.float32)]
            s["ws"] = _workspace(_lib().lib.s2x_beam_select_workspace_size(n, beams, vocab, case["n_out"]))
        return s
    if op == "pages":
        lens, page, beams = _page_lens(case), case["page"], case["n_beam"]
        shared = case["prompt"] // page  # whole pages of the prompt, held by all beams of a request
        n_seq = len(lens)
        each = [max(0, _pages(n, page) - shared) for n in lens]
        width = max(_pages(n, page) for n in lens) + 4
        n_held = shared * case["n_req"] + sum(each)
        n_pages = n_held + case["spare"]
        ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        at = torch.arange(width, device=DEV)[None, :]
        seq = torch.arange(n_seq, device=DEV)[:, None]
        first = torch.cumsum(_i32(each).long(), 0)[:, None] - _i32(each).long()[:, None] + shared * case["n_req"]
        take = torch.where(at < shared, seq // beams * shared + at, first + at - shared)
        have = _i32([_pages(n, page) for n in lens]).long()[:, None]
        table = torch.where(at < have, ids[take.clamp(0, n_pages - 1)], torch.full((), -1, dtype=torch.int32, device=DEV))
        s["table"], s["len"], s["n_pages"] = table.contiguous(), _i32(lens), n_pages
        if case["how"] == "fork":
            pick = (torch.rand(n_seq, generator=g, device=DEV) ** 2 * beams).long().clamp(max=beams - 1)
            s["parent"] = (seq[:, 0] // beams * beams + pick).to(torch.int32)
        s["k"], s["v"] = _cache(case, case["layers"], n_pages, g)
        if own:
            n_copy = n_seq if case["how"] == "fork" else n_pages // 2
            s["out"] = {"table": torch.empty_like(s["table"]), "len": torch.empty_like(s["len"]),
                        "copy": torch.empty(3, n_copy, dtype=torch.int32, device=DEV),
                        "free": torch.empty(n_pages, dtype=torch.int32, device=DEV),
                        "count": torch.empty(2, dtype=torch.int64, device=DEV)}
            s["caches"] = (_lib().KVCache * case["layers"])(*[_kv_cache(case, k, v) for k, v in zip(s["k"], s["v"])])
            s["ws"] = _workspace(_lib().lib.s2x_kv_pages_workspace_size(n_pages))
        return s
    sizes = _group_sizes(case)
    prefix, own_len = _prefix_lens(case)
    page, n_seq = case["page"], sum(sizes)
    width = _pages(case["prefix_max"] + case["own_max"], page) + 1
    # whole pages of the prefix are the group's, the others a sequence's own;
    # the tokens of the prefix that share a page with the sequence's own are
    # the same in all of them (copied when it was forked)
    shared, rows, used = [], [], 0
    for n in prefix:
        shared.append((used, n // page))
        used += n // page
    copies = [[], []]
    for i, (n, more) in enumerate(zip(prefix, own_len)):
        firsts = []
        for m in more:
            count = _pages(n + m, page) - n // page
            rows.append((shared[i], used, count))
            firsts.append(used)
            used += count
        if n % page:
            copies[0] += firsts[1:]
            copies[1] += [firsts[0]] * (len(firsts) - 1)
    n_pages = used + 2
    ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    a0, an, b0, bn = (torch.tensor(v, device=DEV)[:, None] for v in zip(*[(r[0][0], r[0][1], r[1], r[2]) for r in rows]))
    at = torch.arange(width, device=DEV)[None, :]
    take = torch.where(at < an, a0 + at, b0 + at - an)
    s["table"] = torch.where(at < an + bn, ids[take.clamp(0, n_pages - 1)],
                             torch.full((), -1, dtype=torch.int32, device=DEV)).contiguous()
    k, v = _cache(case, 1, n_pages, g)
    s["k"], s["v"] = k[0], v[0]
    if copies[0]:
        to, src = (ids[torch.tensor(c, device=DEV)].long() for c in copies)
        s["k"][to], s["v"][to] = s["k"][src], s["v"][src]
    s["len"] = _i32([n + m for n, more in zip(prefix, own_len) for m in more])
    s["start"] = _i32([sum(sizes[:i]) for i in range(len(sizes) + 1)])
    s["prefix"] = _i32(prefix)
    s["q"] = _normal(g, n_seq, case["hq"], case["d"], std=1.5).to(TYPES[case["type"]])
    s["scale"] = 1.0 / math.sqrt(case["d"])
    if own:
        s["out"] = torch.empty(n_seq, case["hq"], case["d"], dtype=TYPES[case["out"]], device=DEV)
        s["lse"] = torch.empty(n_seq, case["hq"], device=DEV)
        s["cache"] = _kv_cache(case, s["k"], s["v"])
        s["ws"] = _workspace(_lib().lib.s2x_attn_paged_prefix_workspace_size(
            case["n_group"], case["group_max"], case["prefix_max"], case["own_max"], case["hq"], case["hkv"], case["d"]))
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
def _lib():
    path = os.path.join(os.getcwd(), "hbd-siglip2.cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import s2x
    return s2x


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _workspace(n_bytes):
    return torch.empty(max(1, n_bytes), dtype=torch.uint8, device=DEV)


def _kv_cache(case, k, v):
    return _lib().KVCache(k=k.data_ptr(), v=v.data_ptr(), type=CODES[case["type"]], page_size=case["page"],
                          n_pages=k.shape[0], n_head=case["hkv"], d_head=case["d"], ld_page=k.stride(0),
                          ld_head=k.stride(1), ld_tok=k.stride(2))


def _own(s):
    case, s2x = s["case"], _lib()
    op = case["op"]
    if op == "rms":
        m, h, q8 = case["rows"], case["h"], case["out"] == "q8"
        res = CODES["f32" if case["res"] == "none" else case["res"]]
        s2x.call("s2x_add_rmsnorm_quantize_q8_1", _p(s["x"]), CODES[case["x"]], h, _p(s.get("resid")), res, h, h, m,
                 _p(s["w"]), EPS, _p(s.get("h")), h, s["q"].shape[1] if q8 else 0, _p(s.get("q")), _p(s.get("ds")),
                 _p(s.get("y")), CODES["f32" if q8 else case["out"]], h, _stream())
        y = s["q"].view(m, -1, 32) * s["ds"][:, :, :1] if q8 else s["y"]
        return {"h": s["h"], "y": y} if "h" in s else {"y": y}
    if op == "beam":
        parent, token, score = s["out"]
        s2x.call("s2x_beam_select", _p(s["logits"]), CODES[case["x"]], case["vocab"], case["n_req"], case["n_beam"],
                 case["vocab"], _p(s["scores"]), _p(s.get("done")), DONE_TOKEN, case["n_out"], _p(parent), _p(token),
                 _p(score), _p(s["ws"]), s["ws"].numel(), _stream())
        return {"parent": parent, "token": token, "score": score}
    if op == "pages":
        o, table = s["out"], s["table"]
        n_seq, width = table.shape
        src, dst, count = o["copy"]
        if case["how"] == "fork":
            s2x.call("s2x_kv_fork", _p(s["parent"]), n_seq, _p(s["len"]), _p(table), n_seq, width, case["page"],
                     s["n_pages"], None, _p(o["table"]), width, _p(o["len"]), _p(src), _p(dst), _p(count), _p(o["free"]),
                     _p(o["count"]), _p(s["ws"]), s["ws"].numel(), _stream())
            s2x.call("s2x_kv_copy_pages", s["caches"], case["layers"], _p(src), _p(dst), _p(count), n_seq, None, _stream())
            return {"table": o["table"], "len": o["len"], "src": src, "dst": dst, "places": count, "free": o["free"],
                    "count": o["count"], "k": s["k"], "v": s["v"]}
        s2x.call("s2x_kv_compact", _p(s["len"]), _p(table), n_seq, width, case["page"], s["n_pages"], _p(o["table"]), width,
                 _p(src), _p(dst), _p(o["count"]), _p(s["ws"]), s["ws"].numel(), _stream())
        s2x.call("s2x_kv_copy_pages", s["caches"], case["layers"], _p(src), _p(dst), None, src.numel(),
                 ctypes.c_void_p(o["count"].data_ptr() + 8), _stream())
        return {"table": o["table"], "src": src, "dst": dst, "count": o["count"], "k": s["k"], "v": s["v"]}
    n_seq, hq, d = s["q"].shape
    s2x.call("s2x_attn_paged_prefix", _p(s["q"]), hq * d, n_seq, None, ctypes.byref(s["cache"]), _p(s["table"]),
             s["table"].shape[1], _p(s["len"]), n_seq, _p(s["start"]), _p(s["prefix"]), case["n_group"], case["group_max"],
             case["prefix_max"], case["own_max"], hq, s["scale"], _p(s["out"]), CODES[case["out"]], hq * d, _p(s["lse"]),
             _p(s["ws"]), s["ws"].numel(), _stream())
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_rms(s):
    case = s["case"]
    m, h = case["rows"], case["h"]
    x = s["x"].float()
    if "resid" in s:
        x = x + s["resid"].float()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * s["w"]
    if case["out"] == "q8":
        k_pad = _pages(h, 32) * 32
        b = torch.cat([y, y.new_zeros(m, k_pad - h)], 1).view(m, -1, 32)
        amax = b.abs().amax(2, keepdim=True)
        q = torch.round(b * torch.where(amax > 0, 127.0 / amax, amax)).clamp(-128, 127)
        y = (q * (amax / 127.0).half().float()).half()
    else:
        y = y.to(TYPES[case["out"]])
    return {"h": x.to(TYPES[case["res"]]), "y": y} if "resid" in s else {"y": y}


def _plain_beam(s):
    """Scores in 64 bits: which of two beams' candidates is ahead hangs on
    sums of many terms.  A value and its place in one 64-bit key: the larger
    value first, of equal ones the lower place."""
    case, logits = s["case"], s["logits"]
    n, beams, vocab, n_out = case["n_req"], case["n_beam"], case["vocab"], case["n_out"]
    x = logits.float() + 0.0
    top = x.amax(1, keepdim=True)
    lse = torch.log(torch.exp((x - top).double()).sum(1)) + top[:, 0].double()
    bits = x.view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() * (1 << 32) + torch.arange(vocab - 1, -1, -1, device=DEV)
    first = torch.topk(key, min(n_out, vocab), dim=1).values
    token = vocab - 1 - (first & 0xffffffff)
    score = s["scores"].double().view(-1, 1) + torch.gather(x, 1, token).double() - lse[:, None]
    if "done" in s:  # a beam that has ended goes on as it is
        done = s["done"].view(-1, 1) != 0
        only = torch.zeros_like(score, dtype=torch.bool)
        only[:, 0] = True
        score = torch.where(done, torch.where(only, s["scores"].double().view(-1, 1), -math.inf), score)
        token = torch.where(done, DONE_TOKEN, token)
    score, token = score.view(n, -1), token.view(n, -1)
    score, at = torch.sort(score, dim=1, descending=True, stable=True)
    score, at = score[:, :n_out], at[:, :n_out]
    there = score > -math.inf
    parent = torch.arange(n, device=DEV)[:, None] * beams + at // min(n_out, vocab)
    return {"parent": torch.where(there, parent, -1).to(torch.int32),
            "token": torch.where(there, torch.gather(token, 1, at), -1).to(torch.int32), "score": score.float()}


def _copied(s, src, dst):
    """The whole of pages src to pages dst, in keys and values; -1: none (as
    the last page on itself)."""
    there = (src >= 0) & (dst >= 0)
    last = s["n_pages"] - 1
    src, dst = torch.where(there, src, last).long(), torch.where(there, dst, last).long()
    return src, dst


def _plain_fork(s):
    case, page, n_pages = s["case"], s["case"]["page"], s["n_pages"]
    parent = s["parent"].long()
    n, width = parent.numel(), s["table"].shape[1]
    length = s["len"].long()[parent]
    at = torch.arange(width, device=DEV)[None, :]
    have = (length + page - 1)[:, None] // page
    table = torch.where(at < have, s["table"][parent].long(), -1)
    # a row's last page is open where it is not full; it may be held by that row alone
    row = torch.arange(n, device=DEV)[:, None]
    open_ = (at == have - 1) & (length % page != 0)[:, None]
    mark = torch.full((n_pages + 1,), 1 << 30, dtype=torch.int64, device=DEV)
    mark.scatter_reduce_(0, torch.where(table >= 0, table, n_pages).flatten(),
                         torch.where(open_, 1 + row, 0).expand(n, width).flatten(), "amin")
    mark = mark[:n_pages]
    last = torch.where(open_, table, -1).amax(1)
    wants = (last >= 0) & (mark[last.clamp(min=0)] != 1 + row[:, 0])
    # the free pages in order, the rows' copies from the front
    is_free = mark == 1 << 30
    rank = torch.cumsum(is_free, 0) - 1
    free = torch.full((n_pages + 1,), -1, dtype=torch.int64, device=DEV)
    free[torch.where(is_free, rank, n_pages)] = torch.arange(n_pages, device=DEV)
    free[n_pages] = -1
    k = torch.cumsum(wants, 0) - 1
    n_copy, n_free = wants.sum(), is_free.sum()
    new = torch.where(wants, free[k.clamp(0, n_pages)], -1)
    table = torch.where(open_ & wants[:, None], new[:, None], table)
    left = free[(torch.arange(n_pages, device=DEV) + n_copy).clamp(max=n_pages)]
    src = torch.where(wants, last, -1)
    places = torch.where(wants, length % page, 0)
    # the places of a copied page that hold tokens
    a, b = _copied(s, src, new)
    seen = (torch.arange(page, device=DEV)[None, :] < places[:, None])[None, :, None, :, None]
    for c in (s["k"], s["v"]):
        c[:, b] = torch.where(seen, c[:, a], c[:, b])
    return {"table": table.to(torch.int32), "len": length.to(torch.int32), "src": src.to(torch.int32),
            "dst": new.to(torch.int32), "places": places.to(torch.int32), "free": left.to(torch.int32),
            "count": torch.stack([(n_free - n_copy).clamp(min=0), n_copy]), "k": s["k"], "v": s["v"]}


def _plain_compact(s):
    case, page, n_pages = s["case"], s["case"]["page"], s["n_pages"]
    at = torch.arange(s["table"].shape[1], device=DEV)[None, :]
    have = (s["len"].long() + page - 1)[:, None] // page
    table = torch.where(at < have, s["table"].long(), -1)
    held = torch.zeros(n_pages + 1, dtype=torch.bool, device=DEV)
    held[torch.where(table >= 0, table, n_pages).flatten()] = True
    held = held[:n_pages]
    n_held = held.sum()
    id_ = torch.arange(n_pages, device=DEV)
    moves, hole = held & (id_ >= n_held), ~held & (id_ < n_held)
    n_move = moves.sum()
    most = n_pages // 2
    lists = []
    for which in (moves, hole):
        t = torch.full((most + 1,), -1, dtype=torch.int64, device=DEV)
        t[torch.where(which, torch.cumsum(which, 0) - 1, most)] = id_
        lists.append(t[:most])
    to = id_.clone()
    src, dst = lists
    to = torch.where(moves, dst[(torch.cumsum(moves, 0) - 1).clamp(0, most - 1)], to)
    table = torch.where(table >= 0, to[table.clamp(min=0)], -1)
    a, b = _copied(s, src, dst)
    for c in (s["k"], s["v"]):
        c[:, b] = c[:, a]
    return {"table": table.to(torch.int32), "src": src.to(torch.int32), "dst": dst.to(torch.int32),
            "count": torch.stack([n_held, n_move]), "k": s["k"], "v": s["v"]}


def _part(q, k, v, seen, scale):
    """Sums over the seen keys of one part: maximum, sum of exponentials and
    weighted values; nothing seen: -inf and zeros."""
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    score = torch.where(seen, score, torch.full((), -math.inf, device=DEV))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return top, e.sum(-1, keepdim=True), torch.matmul(e, v)


def _rows(s, rows, first, n):
    """Keys and values of tokens first .. first + n - 1 of the table's rows, in
    f32 (rows, heads, n, d)."""
    page, width = s["case"]["page"], s["table"].shape[1]
    t = first[:, None] + torch.arange(n, device=DEV)[None, :]
    ids = torch.gather(s["table"][rows].long(), 1, (t // page).clamp(max=width - 1)).clamp(min=0)
    return [c[ids, :, t % page].float().transpose(1, 2).contiguous() for c in (s["k"], s["v"])]


def _plain_prefix(s):
    case = s["case"]
    n_seq, hq, d = s["q"].shape
    hkv, groups, size = case["hkv"], case["n_group"], case["group_max"]
    share = hq // hkv
    start, prefix = s["start"].long(), s["prefix"].long()
    # queries of a group together (groups, heads, size * share, d)
    member = start[:-1, None] + torch.arange(size, device=DEV)[None, :]
    real = member < start[1:, None]
    q = s["q"].float().view(n_seq, hkv, share, d)
    qg = q[member.clamp(max=n_seq - 1)].transpose(1, 2).reshape(groups, hkv, size * share, d)
    k, v = _rows(s, start[:-1], torch.zeros_like(prefix), case["prefix_max"])
    seen = (torch.arange(case["prefix_max"], device=DEV)[None, :] < prefix[:, None])[:, None, None, :]
    parts = [t.view(groups, hkv, size, share, -1).transpose(1, 2)[real] for t in _part(qg, k, v, seen, s["scale"])]
    # each sequence's own tokens
    group = torch.bucketize(torch.arange(n_seq, device=DEV), start[1:], right=True)
    k, v = _rows(s, torch.arange(n_seq, device=DEV), prefix[group], case["own_max"])
    seen = (torch.arange(case["own_max"], device=DEV)[None, :] < (s["len"].long() - prefix[group])[:, None])[:, None, None, :]
    top, den, num = _part(q, k, v, seen, s["scale"])
    m = torch.maximum(top, parts[0])
    a, b = torch.exp(parts[0] - m), torch.exp(top - m)
    den = parts[1] * a + den * b
    out = (parts[2] * a + num * b) / den
    return {"out": out.reshape(n_seq, hq, d).to(TYPES[case["out"]]), "lse": (torch.log(den) + m).reshape(n_seq, hq)}


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    if case["op"] == "pages":
        return _plain_fork(s) if case["how"] == "fork" else _plain_compact(s)
    return {"rms": _plain_rms, "beam": _plain_beam, "prefix": _plain_prefix}[case["op"]](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definitions in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
    if op == "rms":
        m, h = case["rows"], case["h"]
        k_pad = _pages(h, 32) * 32
        out = m * (k_pad + k_pad // 8) if case["out"] == "q8" else m * h * size[case["out"]]
        return {"bytes": m * h * (size[case["x"]] + 2 * size[case["res"]]) + out + 4 * h, "flops": 6 * m * h}
    if op == "beam":
        rows = case["n_req"] * case["n_beam"]
        live = rows * 0.85 if case["done"] else rows
        return {"bytes": live * case["vocab"] * size[case["x"]] + 5 * rows + 12 * case["n_req"] * case["n_out"],
                "flops": 4 * live * case["vocab"]}
    if op == "pages":
        lens, page, beams = _page_lens(case), case["page"], case["n_beam"]
        shared = case["prompt"] // page
        entries = sum(_pages(n, page) for n in lens)
        held = shared * case["n_req"] + sum(max(0, _pages(n, page) - shared) for n in lens)
        n_pages = held + case["spare"]
        token = case["layers"] * case["hkv"] * case["d"] * 2 * 2
        if case["how"] == "fork":
            # of n rows that pick among n beams with the square's distribution, those that share theirs
            alive = sum(1 - (1 - (math.sqrt((i + 1) / beams) - math.sqrt(i / beams))) ** beams for i in range(beams))
            copied = case["n_req"] * (beams - alive) * (page / 2) * token
        else:
            copied = held * (n_pages - held) / n_pages * page * token
        return {"bytes": 8 * entries + 4 * n_pages + 12 * len(lens) + 2 * copied, "flops": 2 * entries}
    prefix, own_len = _prefix_lens(case)
    sizes = _group_sizes(case)
    token, page = case["hkv"] * case["d"] * 4, case["page"]
    own_all = sum(sum(m) for m in own_len)
    hq, d, n = case["hq"], case["d"], sum(sizes)
    io = n * hq * (d * (2 + size[case["out"]]) + 4)
    return {"bytes": (sum(prefix) + own_all) * token + (sum(prefix) + own_all) // page * 4 + io,
            "flops": (sum(a * b for a, b in zip(prefix, sizes)) + own_all) * hq * d * 4}


def _exact_copies(s, pairs, places):
    """The caches in 64 bits with the pages of `pairs` copied, one by one."""
    out = []
    for c in (s["k"], s["v"]):
        c = c.double()
        for (a, b), n in zip(pairs, places):
            c[:, b, :, :n] = c[:, a, :, :n]
        out.append(c)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rms":
        h = case["h"]
        x = s["x"].double()
        if "resid" in s:
            x = x.add(s["resid"].double())
        y = x * torch.rsqrt(x.pow(2).sum(1, keepdim=True) / h + EPS) * s["w"].double()
        if case["out"] == "q8":
            b = torch.nn.functional.pad(y, (0, -h % 32)).unflatten(1, (-1, 32))
            step = b.abs().amax(2, keepdim=True) / 127
            y = torch.where(step > 0, torch.round(b / step), torch.zeros_like(b)) * step.half().double()
        return {"h": x, "y": y} if "resid" in s else {"y": y}
    if op == "beam":
        n, beams, n_out = case["n_req"], case["n_beam"], case["n_out"]
        x = s["logits"].double()
        best = []
        for r in range(n):
            p = torch.log_softmax(x[r * beams:(r + 1) * beams], 1) + s["scores"][r].double()[:, None]
            if "done" in s:
                over = s["done"][r] != 0
                p[over] = -math.inf
                p[over, DONE_TOKEN] = s["scores"][r].double()[over]
            best.append(p.flatten().topk(n_out).values)
        return {"parent": None, "token": None, "score": torch.stack(best)}
    if op == "pages":
        page, table = case["page"], s["table"].cpu().tolist()
        lens = s["len"].cpu().tolist()
        pairs, places = [], []
        if case["how"] == "fork":
            rows = [(table[p][:_pages(lens[p], page)], lens[p]) for p in s["parent"].cpu().tolist()]
            held = {id_ for ids, _ in rows for id_ in ids}
            free = iter(sorted(set(range(s["n_pages"])) - held))
            # (whole pages are never an open one here: the beams' own begin with one)
            kept = {}
            for i, (ids, n) in enumerate(rows):
                if n % page and kept.setdefault(ids[-1], i) != i:
                    pairs.append((ids[-1], next(free)))
                    places.append(n % page)
        else:
            held = sorted({id_ for ids, n in zip(table, lens) for id_ in ids[:_pages(n, page)]})
            holes = sorted(set(range(len(held))) - set(held))
            pairs = list(zip([i for i in held if i >= len(held)], holes))
            places = [page] * len(pairs)
        k, v = _exact_copies(s, pairs, places)
        out = {"table": None, "src": None, "dst": None, "count": None, "k": k, "v": v}
        return {**out, "len": None, "places": None, "free": None} if case["how"] == "fork" else out
    # one sequence after the other, over all its tokens
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    out, lse = [], []
    for i, n in enumerate(s["len"].cpu().tolist()):
        t = torch.arange(n, device=DEV)
        ids = s["table"][i].long()[t // page]
        k, v = (c[ids, :, t % page].double().transpose(0, 1) for c in (s["k"], s["v"]))
        score = torch.matmul(s["q"][i].double().view(hkv, hq // hkv, d), k.transpose(1, 2).contiguous()) * s["scale"]
        lse.append(torch.logsumexp(score, -1).view(hq))
        out.append(torch.matmul(torch.softmax(score, -1), v.contiguous()).view(hq, d))
    return {"out": torch.stack(out), "lse": torch.stack(lse)}
