// s2x_paged.h -- the kernel of attention over a paged cache for up to 16 query
// rows that see the same keys, one wave a tile of keys, in the forms that its
// callers launch: a sequence's query heads on a key head (s2x_paged.hip), and
// those of a group of sequences over the tokens that they share, or of each over
// its own ones (s2x_prefix.hip).
#pragma once

#include "s2x_decode.h"
#include "s2x_device.h"
#include "s2x_search.h"

namespace s2x {

constexpr int PA_ALIGN = 32;  // chunks begin at multiples of the largest tile

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

template <typename T> struct Pa;
// A probability enters the second product as a sum of terms of the cache's type:
// three of bf16, 8 bits each, hold an f32's 24; two of f16, 11 bits and a
// sign each, hold 23 (off by 2^-23 at most, twice f32's half step), and a third
// would change little where the sums round in f32.  bf16 with two, 17 bits, was
// 0.1 us of 10 to 16 faster, and where values cancel showed in a bf16 output too.
// f16 takes p * 2^15 (p <= 1), which keeps the second term's
// 2^-25 of the largest above the subnormal range.
template <> struct Pa<_Float16> {
    static constexpr int terms = 2;
    typedef v8h vec;
    static constexpr float up = 32768.0f, down = 1.0f / 32768.0f;
    static __device__ __forceinline__ v4f mfma(vec a, vec b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f mfma4(v4s a, v4s b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h, a), __builtin_bit_cast(v4h, b), c, 0, 0, 0);
    }
};
template <> struct Pa<__bf16> {
    static constexpr int terms = 3;
    typedef v8bf vec;
    static constexpr float up = 1.0f, down = 1.0f;
    static __device__ __forceinline__ v4f mfma(vec a, vec b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ v4f mfma4(v4s a, v4s b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
    }
};

// Keys [begin, len) of a sequence that its chunks cover, begin a tile's start.
struct PaRange {
    int64_t first, len, begin;
};
__device__ __forceinline__ PaRange pa_range(const AttnPaged &p, int s) {
    PaRange r;
    r.len = min((int64_t)min(max(p.kv_len[s], 0), p.max_len), p.ld_table << p.kv.page_shift);
    r.first = p.window > 0 ? max(r.len - p.window, (int64_t)0) : 0;
    r.begin = r.first & ~(int64_t)(PA_ALIGN - 1);
    return r;
}

// Row of q, out and lse that is sequence s's: s itself, or of packed rows the last
// that s brings; -1: it brings none, or none that the call has.  (PACKED at
// compile time: a test of the pointer in every workgroup, with or without a
// branch, was 0.1 to 0.4 us of 10 to 17.)
template <bool PACKED>
__device__ __forceinline__ int64_t pa_row(const AttnPaged &p, int s) {
    if constexpr (!PACKED) return s;
    const int32_t from = p.tok_start[s], to = p.tok_start[s + 1];
    return from >= 0 && to > from && to <= p.n_row ? to - 1 : -1;
}

// Values 4 e .. 4 e + 3 of head h: the sums over its keys by the sum of the
// exponentials (nothing seen: zeros, and lse = -inf by itself).
template <typename TC>
__device__ __forceinline__ void pa_write(const AttnPaged &p, int64_t row, int h, int d, int e, v4f a, float M, float L) {
    typedef TC vec4 __attribute__((ext_vector_type(4)));
    const int64_t at = row * p.ld_out + (int64_t)h * d + 4 * e;
    v4f y;
    vec4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = L == 0.0f ? 0.0f : a[i] * Pa<TC>::down / L;
        t[i] = (TC)f32_materialize(y[i]);
    }
    if (p.out_f32) *reinterpret_cast<v4f *>((float *)p.out + at) = y;
    else *reinterpret_cast<vec4 *>((TC *)p.out + at) = t;
    if (e == 0 && p.lse) p.lse[row * p.n_q_head + h] = (M + log2f(L)) * 0.693147180559945309f;
}

// The keys that a group's sequences share, and those of one sequence.
struct PaGroup {
    int     first, size;  // sequences (size 0: none)
    int64_t len;          // tokens of the prefix
};
__device__ __forceinline__ PaGroup pa_group(const AttnPrefix &p, int g) {
    const int a = p.group_start[g], b = p.group_start[g + 1];
    PaGroup r;
    r.first = a;
    r.size = a >= 0 && a < p.a.n_seq && b > a ? min(min(b, p.a.n_seq) - a, p.max_group) : 0;
    r.len = min((int64_t)min(max(p.prefix_len[g], 0), p.max_prefix), p.a.ld_table << p.a.kv.page_shift);
    return r;
}
// Whether sequence s is one that has been freed: no tokens, and a table that begins
// with no page (ld_table > 0).
__device__ __forceinline__ bool pa_freed(const AttnPaged &p, int s) {
    return p.kv_len[s] <= 0 && (uint32_t)p.table[s * p.ld_table] >= (uint32_t)p.kv.n_pages;
}
// The sequence whose pages are the group's prefix: the first that has not been freed
// (none: the first).  Of the whole wave.
__device__ __forceinline__ int pa_holder(const AttnPaged &p, const PaGroup &g) {
    for (int i0 = 0; i0 < g.size; i0 += WAVE) {
        const bool live = !pa_freed(p, g.first + min(i0 + (int)(threadIdx.x & 63), g.size - 1));
        const uint64_t m = __builtin_amdgcn_ballot_w64(live);
        if (m) return g.first + i0 + __builtin_ctzll(m);
    }
    return g.first;
}
// The last group that begins at or before sequence s (starts ascend; none: the
// first), and where it begins: each lane of the wave looks at one of 64 parts of
// the groups left, until one is.
__device__ __forceinline__ int pa_find(const AttnPrefix &p, int s, int &first) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = p.n_group;
    for (;;) {
        const int step = (n + 63) / 64;
        const int at = p.group_start[lo + min(lane * step, n - 1)];
        const int k = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane * step < n && at <= s)) - 1, 0);
        lo += k * step;
        n = min(step, n - k * step);
        if (n > 1) continue;
        first = __shfl(at, k);
        return lo;
    }
}
// tokens of sequence s (its table's, at most)
__device__ __forceinline__ int64_t pa_len(const AttnPaged &p, int s) {
    return min((int64_t)max(p.kv_len[s], 0), p.ld_table << p.kv.page_shift);
}
__device__ __forceinline__ PaRange pa_own(const AttnPrefix &p, const PaGroup &g, int s) {
    PaRange r;
    const int64_t len = pa_len(p.a, s);
    r.first = min(g.len, len);
    r.len = min(len, r.first + p.max_own);
    r.begin = r.first & ~(int64_t)(PA_ALIGN - 1);
    return r;
}
// row of q, out and lse that is sequence s's (-1: none)
__device__ __forceinline__ int64_t pa_row_of(const AttnPaged &p, int s) {
    return p.tok_start ? pa_row<true>(p, s) : s < p.n_row ? s : -1;
}

// What a launch covers: a sequence's tokens (ROWS: its query is row s, PACKED: by
// tok_start), the prefix of a group (PREFIX: columns are the query heads on a key
// head of all its sequences, at most 16) or a sequence's own tokens behind it (OWN).
// The last two leave their sums in the workspace, for the join of all parts.
enum PaMode { PA_ROWS, PA_PACKED, PA_PREFIX, PA_OWN };
__device__ __forceinline__ const AttnPaged &pa_base(const AttnPaged &p) { return p; }
__device__ __forceinline__ const AttnPaged &pa_base(const AttnPrefix &p) { return p.a; }

// Workgroup (or wave) bid -> (unit, chunk), head.  Workgroups go round the 8 XCDs: the
// heads of one chunk follow each other on one XCD (a token-major row's
// cache lines are shared between heads), and the chunks of a sequence
// lie on different ones (u = chunk n_seq + (s + chunk) % n_seq), since
// ragged sequences leave the later chunks empty.
struct PaWork {
    int unit, split, hp;
};
__device__ __forceinline__ PaWork pa_work(int bid, int n_unit, int n_split, int H) {
    const int U = n_unit * n_split, octs = U / 8 * 8;
    PaWork w;
    int u;
    if (bid < octs * H) {
        const int q8 = bid / 8, o = q8 / H;
        u = 8 * o + bid % 8;
        w.hp = q8 - o * H;
    } else {
        const int b = bid - octs * H;
        w.hp = b / (U - octs);
        u = octs + b - w.hp * (U - octs);
    }
    w.split = u / n_unit;
    w.unit = (u - w.split * n_unit + w.split) % n_unit;
    return w;
}

// DC: 32-value chunks of a head; EXACT: d_head = 32 DC; KT: 16-key parts of a
// tile; NW: waves of a workgroup.  w: what it does of its form's n_split chunks (of
// the n_parts that a row of the workspace has, from part0 on: PREFIX, OWN).
template <typename TC, int DC, bool EXACT, int KT, int NW, PaMode MODE, typename ARGS>
__device__ __forceinline__ void pa_body(const ARGS &args, const PaWork &w, int chunk, int n_split, int n_parts, int part0) {
    constexpr bool PACKED = MODE == PA_PACKED, GROUPS = MODE == PA_PREFIX || MODE == PA_OWN;
    const AttnPaged &p = pa_base(args);
    typedef typename Pa<TC>::vec vec;
    constexpr int DP = 32 * DC, DT = 2 * DC, VT = DC * KT;  // values padded, 16-value parts, V loads of a tile
    constexpr int TILE = 16 * KT, STEP = NW * TILE, NT = NW * WAVE, NP = Pa<TC>::terms;
    extern __shared__ __align__(16) uint8_t lds[];  // V tiles of the waves, then their sums
    __shared__ float ml[NW][2][16];
    // (one wave: it may be any of its workgroup, with a part of LDS of its own)
    const int place = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = NW == 1 ? 0 : place;
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int d = EXACT ? DP : p.kv.d_head, nch = d / 8;
    const int group = p.n_q_head / p.kv.n_head, parts = MODE == PA_PREFIX ? 1 : (group + 15) / 16;
    const int hk = w.hp / parts, h0 = hk * group + (w.hp - hk * parts) * 16, split = w.split;
    int s = w.unit, R = min(16, (hk + 1) * group - h0), slot = 0;
    PaRange kr;
    PaGroup gr = {};
    if constexpr (GROUPS) {
        int first;
        const int gi = MODE == PA_OWN ? pa_find(args, s, first) : w.unit;
        gr = pa_group(args, gi);
        slot = gi * args.max_group + (MODE == PA_OWN ? s - gr.first : 0);
        if (MODE == PA_OWN ? s < gr.first || s >= gr.first + gr.size : gr.size == 0) return;  // (uniform)
        if constexpr (MODE == PA_PREFIX) {
            s = gr.first;
            R = gr.size * group;
            kr = PaRange{0, gr.len, 0};
        } else {
            kr = pa_own(args, gr, s);
        }
    } else {
        kr = pa_range(p, s);
    }
    const int64_t start = kr.begin + (int64_t)split * chunk, end = min(start + chunk, kr.len);
    if (start >= end && (GROUPS || n_split > 1)) return;  // (uniform; an only chunk writes zeros)
    int64_t qrow, lim = 0;  // of column r; its prefix's end
    if constexpr (MODE == PA_PREFIX) {
        const int c = min(s + r / group, s + gr.size - 1);
        qrow = pa_row_of(p, c);
        lim = pa_len(p, c);
    } else if constexpr (MODE == PA_OWN) {
        qrow = pa_row_of(p, s);
        if (qrow < 0) return;  // (uniform)
    } else {
        qrow = pa_row<PACKED>(p, s);
        if (PACKED && qrow < 0) return;  // (uniform)
    }
    // whether some column sees less than all of the prefix
    const bool ragged = MODE == PA_PREFIX && __builtin_amdgcn_ballot_w64(lim < end) != 0;

    const TC *kp = (const TC *)p.kv.k + hk * p.kv.ld_head, *vp = (const TC *)p.kv.v + hk * p.kv.ld_head;
    const int32_t *row = p.table + s * p.ld_table;  // (PREFIX: of the first sequence, unless that has been freed)
    const uint32_t pmask = (1u << p.kv.page_shift) - 1, ldp = (uint32_t)p.kv.ld_page, ldt = (uint32_t)p.kv.ld_tok;
    TC *vl = reinterpret_cast<TC *>(lds) + place * TILE * d;

    vec q[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        q[c] = vec{};
        const int h = MODE == PA_PREFIX ? hk * group + r % group : h0 + r;
        if (r < R && (MODE != PA_PREFIX || qrow >= 0) && (EXACT || 32 * c + 8 * g < d))
            q[c] = *reinterpret_cast<const vec *>((const TC *)p.q + qrow * p.ld_q + (int64_t)h * d + 32 * c + 8 * g);
    }

    // Table entry of key t0 + lane % TILE (the row's last one for keys past it).
    // Only loaded here: a test of it would wait for all loads before it.
    auto entry_of = [&](int64_t t0) {
        return row[min((t0 + (lane & (TILE - 1))) >> p.kv.page_shift, p.ld_table - 1)];
    };
    vec k[KT][DC], v[VT];
    const uint32_t magic = (65536u + nch - 1) / nch;  // f / nch for f < 1,024
    uint32_t seen = 0;
    constexpr uint32_t ALL = ~0u;
    // Keys: lane / 4 of a 16-key part and a 16-byte piece lane % 4 of 64 (four
    // lanes a row: with a row a lane, as the MFMA wants them, each would be a
    // cache access of its own).  Values: piece f of the tile's rows in order.
    auto load = [&](int64_t t0, int32_t entry) {
        const int64_t t = t0 + (lane & (TILE - 1));
        const bool ok = t >= kr.first && t < end && (uint32_t)entry < (uint32_t)p.kv.n_pages;
        seen = (uint32_t)__builtin_amdgcn_ballot_w64(ok);  // (lanes repeat the tile's keys)
        const TC *ks[KT], *vs[VT];
        bool kok[KT], vok[VT];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            const int key = 16 * j + (lane >> 2);
            const uint32_t pid = (uint32_t)__shfl(entry, key);
            ks[j] = kp + ((uint64_t)pid * ldp + (((uint32_t)t0 + key) & pmask) * (uint64_t)ldt);
            kok[j] = seen >> key & 1;
        }
#pragma unroll
        for (int i = 0; i < VT; ++i) {
            // (past the tile's last piece: that one again, not stored)
            const uint32_t f = EXACT ? i * WAVE + lane : min(i * WAVE + lane, TILE * nch - 1);
            const uint32_t key = EXACT ? f / (DP / 8) : f * magic >> 16;
            const uint32_t pid = (uint32_t)__shfl(entry, (int)key);
            vs[i] = vp + ((uint64_t)pid * ldp + (((uint32_t)t0 + key) & pmask) * (uint64_t)ldt + 8 * (f - key * nch));
            vok[i] = seen >> key & 1;
        }
        const int e = 8 * (lane & 3);
        if (seen == ALL) {  // (uniform; no lane masks)
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int c = 0; c < DC; ++c)
                    k[j][c] = *reinterpret_cast<const vec *>(ks[j] + (EXACT || 32 * c + e < d ? 32 * c + e : 0));
#pragma unroll
            for (int i = 0; i < VT; ++i) v[i] = *reinterpret_cast<const vec *>(vs[i]);
        } else {
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int c = 0; c < DC; ++c) {
                    k[j][c] = vec{};
                    if (kok[j]) k[j][c] = *reinterpret_cast<const vec *>(ks[j] + (EXACT || 32 * c + e < d ? 32 * c + e : 0));
                }
#pragma unroll
            for (int i = 0; i < VT; ++i) {
                v[i] = vec{};
                if (vok[i]) v[i] = *reinterpret_cast<const vec *>(vs[i]);
            }
        }
    };

    float m = -INFINITY, l = 0.0f;
    v4f o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = v4f{0, 0, 0, 0};
    const float sc = p.scale * 1.44269504088896341f;  // log2(e)

    int64_t t0 = start + wave * TILE;
    int32_t next = -1;
    if (t0 < end) {
        int32_t here = entry_of(t0);
        next = entry_of(t0 + STEP);
        // (asked while the entries are on their way; uniform)
        if (MODE == PA_PREFIX && pa_freed(p, gr.first)) {
            row = p.table + pa_holder(p, gr) * p.ld_table;
            here = entry_of(t0);
            next = entry_of(t0 + STEP);
        }
        load(t0, here);
    }
    for (; t0 < end; t0 += STEP) {
        const uint32_t mask = seen;
#pragma unroll
        for (int i = 0; i < VT; ++i) {
            if (EXACT || i * WAVE + lane < TILE * nch)
                *reinterpret_cast<vec *>(vl + (i * WAVE + lane) * 8) = v[i];
        }
        v4f st[KT];
#pragma unroll
        for (int j = 0; j < KT; ++j) {
            st[j] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                v4i kk = __builtin_bit_cast(v4i, k[j][c]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    kk[w] = __shfl(kk[w], 4 * r + g);
                    if (!EXACT && 32 * c + 8 * g >= d) kk[w] = 0;  // (read from the row's start)
                }
                st[j] = Pa<TC>::mfma(__builtin_bit_cast(vec, kk), q[c], st[j]);
            }
        }
        if (t0 + STEP < end) {  // (k and v are free)
            load(t0 + STEP, next);
            next = entry_of(t0 + 2 * STEP);
        }
        // the softmax of head r over keys 4 g + i, 16 + 4 g + i
        float mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                st[j][i] = st[j][i] * sc;
                if (mask != ALL && !(mask >> (16 * j + 4 * g + i) & 1)) st[j][i] = -INFINITY;
                if (ragged && t0 + 16 * j + 4 * g + i >= lim) st[j][i] = -INFINITY;
                mt = fmaxf(mt, st[j][i]);
            }
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float mn = fmaxf(m, mt), base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l = l * alpha;
        vec pt[NP];  // (KT = 1: its first four)
#pragma unroll
        for (int j = 0; j < KT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(st[j][i] - base);
                l = l + e;
                float x = e * Pa<TC>::up;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    pt[n][4 * j + i] = (TC)x;
                    x = x - (float)pt[n][4 * j + i];
                }
            }
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = o[i] * alpha;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            if (!EXACT && 16 * i >= d) break;
            v4s a[KT];
#pragma unroll
            for (int j = 0; j < KT; ++j) {
                TC *src = vl + (16 * j + 4 * g + (r >> 2)) * d + 16 * i + (r & 3) * 4;
                a[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)src);
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const v8s pn = __builtin_bit_cast(v8s, pt[n]);
                if constexpr (KT == 2) {
                    const v8s a8 = __builtin_shufflevector(a[0], a[KT - 1], 0, 1, 2, 3, 4, 5, 6, 7);
                    o[i] = Pa<TC>::mfma(__builtin_bit_cast(vec, a8), pt[n], o[i]);
                } else {
                    o[i] = Pa<TC>::mfma4(a[0], __builtin_shufflevector(pn, pn, 0, 1, 2, 3), o[i]);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }

    // join the waves: o[i] is values 16 i + 4 g .. + 3 of head r
    l = l + __shfl_xor(l, 16);
    l = l + __shfl_xor(l, 32);
    if constexpr (NW == 1) {  // (nothing to join; a form that leaves its sums)
        if (r >= R) return;
        const int64_t at = ((int64_t)slot * p.n_q_head + h0 + r) * n_parts + part0 + split;
        float *ws = (float *)p.ws;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            if (!EXACT && 16 * i + 4 * g >= d) break;
            reinterpret_cast<v4f *>(ws)[at * (nch * 2) + 4 * i + g] = o[i];
        }
        if (g == 0)
            reinterpret_cast<float2 *>(ws + (int64_t)args.n_group * args.max_group * p.n_q_head * n_parts * d)[at] = make_float2(m, l);
        return;
    }
    float *ol = reinterpret_cast<float *>(lds);  // [wave][head < R][DP + 4]
    __syncthreads();
    if (r < R) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
            *reinterpret_cast<v4f *>(ol + (wave * R + r) * (DP + 4) + 16 * i + 4 * g) = o[i];
        if (g == 0) {
            ml[wave][0][r] = m;
            ml[wave][1][r] = l;
        }
    }
    __syncthreads();
    for (int i = tid; i < R * nch * 2; i += NT) {
        const int h = i / (nch * 2), e = i - h * (nch * 2);
        float M = ml[0][0][h];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, ml[w][0][h]);
        const float base = M == -INFINITY ? 0.0f : M;
        v4f a = {0, 0, 0, 0};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w][0][h] - base);
            L = fmaf(ml[w][1][h], f, L);
            const v4f x = *reinterpret_cast<const v4f *>(ol + (w * R + h) * (DP + 4) + 4 * e);
#pragma unroll
            for (int n = 0; n < 4; ++n) a[n] = fmaf(x[n], f, a[n]);
        }
        if constexpr (GROUPS) {
            // (a column's slot: its group's place and its own in it)
            const int64_t at = ((int64_t)(slot + (MODE == PA_OWN ? 0 : h / group)) * p.n_q_head +
                                (MODE == PA_OWN ? h0 + h : hk * group + h % group)) * n_parts + part0 + split;
            float *ws = (float *)p.ws;
            reinterpret_cast<v4f *>(ws)[at * (nch * 2) + e] = a;
            if (e == 0)
                reinterpret_cast<float2 *>(ws + (int64_t)args.n_group * args.max_group * p.n_q_head * n_parts * d)[at] = make_float2(M, L);
            continue;
        }
        const int64_t sh = (int64_t)s * p.n_q_head + h0 + h;
        if (n_split > 1) {
            float *ws = (float *)p.ws;
            const int64_t at = sh * n_split + split;
            reinterpret_cast<v4f *>(ws)[at * (nch * 2) + e] = a;
            if (e == 0)
                reinterpret_cast<float2 *>(ws + (int64_t)p.n_seq * p.n_q_head * n_split * d)[at] = make_float2(M, L);
        } else {
            pa_write<TC>(p, qrow, h0 + h, d, e, a, M, L);
        }
    }
}

}  // namespace s2x
