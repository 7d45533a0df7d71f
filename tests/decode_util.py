"""Inputs and plain 64-bit forms of the decode step's operators (the C-ABI's
kv_slots, qk_norm_rope_kv, attn_paged and mul_mat_q4_0 entry points)."""
import ctypes

import numpy as np
import torch

import s2x

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": s2x.TYPE_F32, "f16": s2x.TYPE_F16, "bf16": s2x.TYPE_BF16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# -- Q4_0 -------------------------------------------------------------------
def q4_0_blocks(q, d):
    """Raw blocks, uint8 (N, K / 32, 18), of nibbles q (N, K) in 0 .. 15 and
    f16 scales d (N, K / 32)."""
    n, k = q.shape
    b = q.reshape(n, k // 32, 32).astype(np.uint8)
    raw = np.empty((n, k // 32, 18), np.uint8)
    raw[:, :, :2] = np.ascontiguousarray(d.astype(np.float16)).view(np.uint8).reshape(n, k // 32, 2)
    raw[:, :, 2:] = b[:, :, :16] | (b[:, :, 16:] << 4)
    return raw


def q8_0_blocks(q, d):
    """The same weight as raw Q8_0 blocks, uint8 (N, K / 32, 34)."""
    n, k = q.shape
    raw = np.empty((n, k // 32, 34), np.uint8)
    raw[:, :, :2] = np.ascontiguousarray(d.astype(np.float16)).view(np.uint8).reshape(n, k // 32, 2)
    raw[:, :, 2:] = (q.astype(np.int16) - 8).astype(np.int8).view(np.uint8).reshape(n, k // 32, 32)
    return raw


def q8_1_planes(rng, m, k):
    """int8 quants (m, k) and words (m, k / 32) as the quantizer writes them."""
    q = rng.integers(-127, 128, (m, k)).astype(np.int8)
    d = (rng.uniform(0.001, 0.03, (m, k // 32))).astype(np.float16)
    s = (q.reshape(m, k // 32, 32).sum(2, dtype=np.int64) * d.astype(np.float64)).astype(np.float16)
    return q, d.view(np.uint16).astype(np.uint32) | (s.view(np.uint16).astype(np.uint32) << 16), d


# -- slots ------------------------------------------------------------------
def slots_ref(kv_len, n_new, free, page, n_pages, table, max_tok):
    table = table.copy()
    ld = table.shape[1]
    taken, rows, lens, starts = 0, [], [], [0]
    for b, (n0, n1) in enumerate(zip(kv_len, n_new)):
        n0, n1 = max(int(n0), 0), max(int(n1), 0)
        have, want = -(-n0 // page), -(-(n0 + n1) // page)
        new = {}
        for i in range(have, want):
            id_ = int(free[taken]) if taken < len(free) else -1
            new[i] = id_ if 0 <= id_ < n_pages else -1
            taken += 1
            if i < ld:
                table[b, i] = new[i]
        for t in range(n0, n0 + n1):
            i = t // page
            id_ = (new[i] if i in new else int(table[b, i])) if i < ld else -1
            rows.append((t, id_ * page + t % page if 0 <= id_ < n_pages else -1))
        lens.append(n0 + n1)
        starts.append(len(rows))
    n_tok = len(rows)
    rows = rows[:max_tok] + [(0, -1)] * max(0, max_tok - n_tok)
    pos = np.array([r[0] for r in rows], np.int32)
    slots = np.array([r[1] for r in rows], np.int64)
    return (table, np.array(lens, np.int32), np.minimum(starts, max_tok).astype(np.int32), pos, slots,
            np.array([taken, n_tok], np.int64))


# -- caches -----------------------------------------------------------------
class Cache:
    """K and V of n_pages pages as (pages, heads, page, d) views of memory laid
    out by head or by token, `gap` extra elements between rows of a page."""

    def __init__(self, n_pages, n_head, page, d, kind, by="head", gap=0, fill=None):
        self.kind, self.page, self.d, self.n_head, self.n_pages = kind, page, d, n_head, n_pages
        shape = (n_pages, n_head, page, d + gap) if by == "head" else (n_pages, page, n_head, d + gap)
        self.mem = []
        for _ in range(2):
            t = torch.full(shape, float("nan"), dtype=TYPES[kind], device="cuda:0")
            self.mem.append(t)
        views = [t[..., :d] if by == "head" else t[..., :d].transpose(1, 2) for t in self.mem]
        self.k, self.v = views
        if fill is not None:
            for c in views:
                c.copy_(fill(tuple(c.shape)))
        # (sizes of one have any stride: from the shape, not from torch)
        row = d + gap
        ld_head, ld_tok = (page * row, row) if by == "head" else (row, n_head * row)
        self.c = s2x.KVCache(k=self.mem[0].data_ptr(), v=self.mem[1].data_ptr(), type=CODES[kind],
                             page_size=page, n_pages=n_pages, n_head=n_head, d_head=d,
                             ld_page=n_head * page * row, ld_head=ld_head, ld_tok=ld_tok)

    def ref(self):
        return ctypes.byref(self.c)


# -- norms and rotation -----------------------------------------------------
def rotated(x, angle, d_rot, style):
    """x (rows, heads, d) in f64, the first d_rot values turned by angle
    (rows, d_rot / 2)."""
    out = x.copy()
    half = d_rot // 2
    j = np.arange(half)
    a, b = (j, j + half) if style == "half" else (2 * j, 2 * j + 1)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
    out[:, :, b] = x[:, :, b] * c + x[:, :, a] * s
    size = np.abs(x).copy()
    size[:, :, a] = size[:, :, b] = np.hypot(x[:, :, a], x[:, :, b])
    return out, size


def heads_ref(x, hq, hkv, d, wq, wk, eps, freq, d_rot, style, pos):
    """Query, key and value heads in f64 and the size of the values that each
    is a sum of."""
    x = x.astype(np.float64).reshape(len(x), hq + 2 * hkv, d)
    parts = []
    for h, w in ((x[:, :hq], wq), (x[:, hq:hq + hkv], wk)):
        if w is not None:
            h = h / np.sqrt((h * h).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        parts.append(rotated(h, pos.astype(np.float64)[:, None] * freq, d_rot, style))
    v = x[:, hq + hkv:]
    return parts[0], parts[1], (v, np.abs(v))


# -- attention --------------------------------------------------------------
def attn_ref(q, cache, table, lens, max_len, scale, window):
    """out, lse and their error scales in f64: sum softmax |v|, the largest
    sum |q k| scale, the keys seen.  Unseen: zeros and -inf."""
    n, hq, d = q.shape
    ld, page, hkv = table.shape[1], cache.page, cache.n_head
    k_all, v_all = cache.k.double().cpu().numpy(), cache.v.double().cpu().numpy()
    out, size = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    lse, top, seen = np.full((n, hq), -np.inf), np.zeros((n, hq)), np.zeros(n, int)
    q = q.astype(np.float64)
    for s in range(n):
        length = min(max(int(lens[s]), 0), max_len, ld * page)
        t = np.arange(max(0, length - window) if window else 0, length)
        ids = table[s][t // page] if len(t) else np.zeros(0, int)
        ok = (ids >= 0) & (ids < cache.n_pages)
        t, ids = t[ok], ids[ok]
        seen[s] = len(t)
        if not len(t):
            continue
        for h in range(hq):
            k, v = k_all[ids, h // (hq // hkv), t % page], v_all[ids, h // (hq // hkv), t % page]
            sc = (k @ q[s, h]) * scale
            m = sc.max()
            p = np.exp(sc - m)
            lse[s, h] = np.log(p.sum()) + m
            p = p / p.sum()
            out[s, h], size[s, h] = p @ v, p @ np.abs(v)
            top[s, h] = (np.abs(k) @ np.abs(q[s, h])).max() * abs(scale)
    return out, size, lse, top, seen
