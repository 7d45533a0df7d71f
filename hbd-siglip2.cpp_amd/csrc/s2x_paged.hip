// s2x_paged.hip -- attention of one new token per sequence over a paged cache.
//
// out = sum_t softmax_t(q . k_t * scale) v_t for up to 16 query heads that
// share a key head, one pass over the keys with the running maximum and sum.
// Each key and value is read once and used for 4 R flops (R query heads a key
// head), far below the matrix pipe's rate: the bytes of the cache bound it.
//
// A wave takes tiles of 32 keys, each by itself (no barrier in the loop):
//  * S^T = K Q^T by v_mfma_f32_16x16x32: K's rows are the A operand, 16 bytes of
//    key lane % 16 a lane, exchanged between the lanes once loaded; the 16
//    query heads (zeros past R) are B, loaded once.
//  * S^T leaves that product with lane l holding head l % 16 and keys 4 g + i
//    (g = l / 16) -- the layout B wants of P^T in the second product, O^T =
//    V^T P^T, if its 8 values of k are taken as keys 4 g .. 4 g + 3 of the
//    tile's two halves.  So the probabilities never cross lanes.
//  * V^T as the A operand of that order is 4 consecutive keys of one value
//    index a lane: the transposing read of LDS (ds_read_b64_tr_b16) of V's
//    rows as they lie, staged in a part of LDS that is the wave's own.
//  * The next tile's keys and values are loaded once the scores have freed
//    the registers, and the page ids of the one after.
// A workgroup's waves join in LDS; a sequence's chunks, where there is more than
// one, in k_attn_join.  Measured (both launches): one sequence of 131,071
// tokens, 32 / 8 heads of 128, 101 us = 5.3 TB/s of keys and values, what a
// large copy reaches; 60 sequences up to 8,000 in pages of 16, 120 us = 4.6.
#include "s2x_decode.h"
#include "s2x_device.h"

namespace s2x {

constexpr int PA_ALIGN = 32;  // chunks begin at multiples of the largest tile
constexpr int PJ_NT = 256;    // threads of the join

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

// DC: 32-value chunks of a head; EXACT: d_head = 32 DC; KT: 16-key parts of a
// tile; NW: waves of a workgroup; PACKED: rows by tok_start.
template <typename TC, int DC, bool EXACT, int KT, int NW, bool PACKED>
__global__ __launch_bounds__(NW * WAVE) void k_attn_paged(AttnPaged p, int chunk, int n_split) {
    typedef typename Pa<TC>::vec vec;
    constexpr int DP = 32 * DC, DT = 2 * DC, VT = DC * KT;  // values padded, 16-value parts, V loads of a tile
    constexpr int TILE = 16 * KT, STEP = NW * TILE, NT = NW * WAVE, NP = Pa<TC>::terms;
    extern __shared__ __align__(16) uint8_t lds[];  // V tiles of the waves, then their sums
    __shared__ float ml[NW][2][16];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = EXACT ? DP : p.kv.d_head, nch = d / 8;
    const int group = p.n_q_head / p.kv.n_head, parts = (group + 15) / 16, H = p.kv.n_head * parts;
    // Workgroup -> (sequence, chunk), head.  Workgroups go round the 8 XCDs: the
    // heads of one chunk follow each other on one XCD (a token-major row's
    // cache lines are shared between heads), and the chunks of a sequence
    // lie on different ones (u = chunk n_seq + (s + chunk) % n_seq), since
    // ragged sequences leave the later chunks empty.
    const int U = p.n_seq * n_split, octs = U / 8 * 8;
    int u, hp;
    if ((int)blockIdx.x < octs * H) {
        const int q8 = blockIdx.x / 8, o = q8 / H;
        u = 8 * o + blockIdx.x % 8;
        hp = q8 - o * H;
    } else {
        const int b = blockIdx.x - octs * H;
        hp = b / (U - octs);
        u = octs + b - hp * (U - octs);
    }
    const int split = u / p.n_seq, s = (u - split * p.n_seq + split) % p.n_seq;
    const int hk = hp / parts, h0 = hk * group + (hp - hk * parts) * 16;
    const int R = min(16, (hk + 1) * group - h0);
    const PaRange kr = pa_range(p, s);
    const int64_t start = kr.begin + (int64_t)split * chunk, end = min(start + chunk, kr.len);
    if (start >= end && n_split > 1) return;  // (uniform; an only chunk writes zeros)
    const int64_t qrow = pa_row<PACKED>(p, s);
    if (PACKED && qrow < 0) return;  // (uniform)

    const TC *kp = (const TC *)p.kv.k + hk * p.kv.ld_head, *vp = (const TC *)p.kv.v + hk * p.kv.ld_head;
    const int32_t *row = p.table + s * p.ld_table;
    const uint32_t pmask = (1u << p.kv.page_shift) - 1, ldp = (uint32_t)p.kv.ld_page, ldt = (uint32_t)p.kv.ld_tok;
    TC *vl = reinterpret_cast<TC *>(lds) + wave * TILE * d;

    vec q[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        q[c] = vec{};
        if (r < R && (EXACT || 32 * c + 8 * g < d))
            q[c] = *reinterpret_cast<const vec *>((const TC *)p.q + qrow * p.ld_q + (int64_t)(h0 + r) * d + 32 * c + 8 * g);
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
        load(t0, entry_of(t0));
        next = entry_of(t0 + STEP);
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

// Chunks of a sequence joined: a workgroup per query head and 4 LANES values of
// it, LANES lanes of 4 values by PJ_NT / LANES groups of chunks, each with its
// own running maximum.  The first loads are of chunks that the launch has room
// for, whether the sequence has them or not, so that they do not wait for its
// length.
template <typename TC, int LANES, bool PACKED>
__global__ __launch_bounds__(PJ_NT) void k_attn_join(AttnPaged p, int chunk, int n_split) {
    constexpr int GROUPS = PJ_NT / LANES;
    __shared__ __align__(16) float part[GROUPS][LANES * 4 + 4];
    __shared__ float gm[GROUPS], gl[GROUPS];
    const int tid = threadIdx.x, d = p.kv.d_head, nq = d / 4, pieces = (nq + LANES - 1) / LANES;
    const int h = blockIdx.x / pieces, s = blockIdx.y;
    const int grp = tid / LANES, e = (blockIdx.x - h * pieces) * LANES + tid % LANES;
    const int64_t at = ((int64_t)s * p.n_q_head + h) * n_split;
    const v4f *ov = reinterpret_cast<const v4f *>(p.ws) + at * nq + min(e, nq - 1);
    const float2 *mlp = reinterpret_cast<const float2 *>((const float *)p.ws + (int64_t)p.n_seq * p.n_q_head * n_split * d) + at;
    float2 t = mlp[min(grp, n_split - 1)];
    v4f x = ov[(int64_t)min(grp, n_split - 1) * nq];
    const PaRange kr = pa_range(p, s);
    const int64_t qrow = pa_row<PACKED>(p, s);
    if (PACKED && qrow < 0) return;  // (uniform)
    const int n = kr.len > kr.begin ? (int)((kr.len - kr.begin + chunk - 1) / chunk) : 0;
    v4f a = {0, 0, 0, 0};
    float M = -INFINITY, L = 0.0f;
    for (int i = grp; i < n; i += GROUPS) {
        const int next = min(i + GROUPS, n - 1);
        const float2 tn = mlp[next];
        const v4f xn = ov[(int64_t)next * nq];
        const float mn = fmaxf(M, t.x), base = mn == -INFINITY ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(M - base), f1 = __builtin_amdgcn_exp2f(t.x - base);
        L = fmaf(t.y, f1, L * f0);
#pragma unroll
        for (int c = 0; c < 4; ++c) a[c] = fmaf(x[c], f1, a[c] * f0);
        M = mn;
        t = tn;
        x = xn;
    }
    *reinterpret_cast<v4f *>(&part[grp][(tid % LANES) * 4]) = a;
    if (tid % LANES == 0) {
        gm[grp] = M;
        gl[grp] = L;
    }
    __syncthreads();
    if (grp != 0 || e >= nq) return;
    float top = gm[0];
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) top = fmaxf(top, gm[i]);
    const float base = top == -INFINITY ? 0.0f : top;
    v4f y = {0, 0, 0, 0};
    L = 0.0f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const float f = __builtin_amdgcn_exp2f(gm[i] - base);
        L = fmaf(gl[i], f, L);
        const v4f z = *reinterpret_cast<const v4f *>(&part[i][tid * 4]);
#pragma unroll
        for (int c = 0; c < 4; ++c) y[c] = fmaf(z[c], f, y[c]);
    }
    pa_write<TC>(p, qrow, h, d, e, y, top, L);
}

// Chunk length, number of chunks and waves of a workgroup.  A step of a workgroup
// (128 keys of 128 halves and their values) takes 1.4 us however few are at
// work, some 45 bytes a ns and CU, so a launch wants all CUs at work to the end;
// a second launch, the join, is 3 us and its gap.
//  * no split for what it does not speed up: up to 320 tokens (3 sequences up
//    to 300, 16 heads of 72: 7.5 us, in chunks of 128 8.1; one of 500: 9.0
//    against 8.1) and, from 128 workgroups on, up to 1,024 (8 key heads of 128:
//    32 up to 500 10.2 us, in chunks of 128 12.3, 64 up to 700 16.3 against
//    20.4, 32 up to 1,000 16.1 against 15.6; 32 up to 2,000 26.9 against 23.4).
//    8 waves a workgroup, one of which fits a CU, where they have keys and the
//    launch is one round of them or the rounds few for the length (16 of 16
//    heads up to 200: 6.6 us, 4 waves 7.2; 64 of 8 heads up to 700: 16.5
//    against 19.3); 4 otherwise (64 of 8 heads up to 100: 6.3 us, 8 waves 9.8;
//    200 of 16 heads up to 300: 33 against 58, 200 of 8 up to 1,000: 55
//    against 62).
//  * with a window, as for sequences of its length.
//  * one sequence: two workgroups a CU (131,071 tokens, 8 key heads: chunks of
//    2,048 101.5 us, of 1,024 104, of 512 108; 2,000 tokens: of 128 8.7 us, of
//    256 10.2); a batch, whose lengths differ: 6 a CU, chunks of 256 to 768 (60
//    up to 8,000: 768 125 us, 1,024 124, 2,048 141, 384 138; 16 up to 8,000:
//    768 34.2, 512 36.5, 1,024 37.9; 8 up to 4,000: 256 17.3, 512 19.5, 128 21).
//  * more waves a workgroup in a split, loads of the next tile before the first
//    product: no faster.
struct PaPlan {
    int chunk, n_split, nw;
};
static PaPlan pa_plan_len(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head) {
    const int64_t units = n_seq * n_kv_head * ((n_q_head / n_kv_head + 15) / 16);
    const int64_t span = max_len + PA_ALIGN;  // (the first tile may begin before a window)
    if (max_len <= 320 || (units >= 128 && max_len <= 1024)) {
        const bool wide = max_len > 128 && (units <= 256 || (max_len > 512 && units <= 1024));
        return PaPlan{(int)((span + 127) / 128 * 128), 1, wide ? 8 : 4};
    }
    const int64_t wgs = 512 * (n_seq < 3 ? n_seq : 3);
    const int64_t least = span * units < 65536 ? 128 : 256, most = n_seq == 1 ? 2048 : 768;
    int64_t c = span * units / wgs;
    c = c < least ? least : c > most ? most : c;
    if (c < span * units >> 22) c = span * units >> 22;  // (a grid of at most 2^23)
    c = (c + 127) / 128 * 128;
    return PaPlan{(int)c, (int)((span + c - 1) / c), 4};
}
static PaPlan pa_plan(int64_t n_seq, int64_t max_len, int64_t window, int64_t n_q_head, int64_t n_kv_head) {
    const PaPlan P = pa_plan_len(n_seq, max_len, n_q_head, n_kv_head);
    if (window <= 0 || window >= max_len) return P;
    PaPlan W = pa_plan_len(n_seq, window, n_q_head, n_kv_head);
    if (W.n_split > P.n_split) {  // (no more chunks than the workspace, sized without a window, has room for)
        const int64_t span = window + PA_ALIGN;
        W.chunk = (int)(((span + P.n_split - 1) / P.n_split + 127) / 128 * 128);
        W.n_split = (int)((span + W.chunk - 1) / W.chunk);
    }
    return W;
}

size_t attn_paged_workspace(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head, int64_t d_head) {
    const int n = pa_plan(n_seq, max_len, 0, n_q_head, n_kv_head).n_split;
    return n > 1 ? (size_t)(n_seq * n_q_head) * n * (d_head + 2) * 4 : 0;
}

template <typename TC, int DC, bool EXACT, int KT, int NW, bool PACKED>
static hipError_t run_paged_w(const AttnPaged &p, const PaPlan &P, hipStream_t stream) {
    const int group = p.n_q_head / p.kv.n_head, R = group < 16 ? group : 16;
    const int64_t wgs = (int64_t)P.n_split * p.kv.n_head * ((group + 15) / 16) * p.n_seq;
    const int v = NW * KT * 16 * p.kv.d_head * 2 + 64, o = NW * R * (DC * 32 + 4) * 4, lds = v > o ? v : o;
    auto kern = k_attn_paged<TC, DC, EXACT, KT, NW, PACKED>;
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(NW * WAVE), lds, stream, p, P.chunk, P.n_split);
    return hipGetLastError();
}
template <typename TC, int DC, bool EXACT, bool PACKED>
static hipError_t run_paged(const AttnPaged &p, const PaPlan &P, hipStream_t stream) {
    constexpr int KT = DC > 4 ? 1 : 2;
    return P.nw == 8 ? run_paged_w<TC, DC, EXACT, KT, 8, PACKED>(p, P, stream)
                     : run_paged_w<TC, DC, EXACT, KT, 4, PACKED>(p, P, stream);
}
template <typename TC, bool PACKED>
static hipError_t run_paged_d(const AttnPaged &p, hipStream_t stream) {
    const PaPlan P = pa_plan(p.n_seq, p.max_len, p.window, p.n_q_head, p.kv.n_head);
    const int d = p.kv.d_head;
    const hipError_t e = d == 64   ? run_paged<TC, 2, true, PACKED>(p, P, stream)
                         : d == 128 ? run_paged<TC, 4, true, PACKED>(p, P, stream)
                         : d == 256 ? run_paged<TC, 8, true, PACKED>(p, P, stream)
                         : d < 64   ? run_paged<TC, 2, false, PACKED>(p, P, stream)
                         : d <= 96  ? run_paged<TC, 3, false, PACKED>(p, P, stream)
                         : d <= 192 ? run_paged<TC, 6, false, PACKED>(p, P, stream)
                                    : run_paged<TC, 8, false, PACKED>(p, P, stream);
    if (e != hipSuccess || P.n_split == 1) return e;
    // few chunks: whole heads a workgroup (60 sequences of at most 8: 10.9 us
    // with 32 values each, 5.0 with 128); many: more workgroups (128 chunks
    // of one sequence: 8.2 us with 128, 4.8 with 32)
    const bool few = P.n_split <= 16;
    const int width = few ? 128 : 32;
    auto join = few ? k_attn_join<TC, 32, PACKED> : k_attn_join<TC, 8, PACKED>;
    hipLaunchKernelGGL(join, dim3(p.n_q_head * ((d + width - 1) / width), p.n_seq), dim3(PJ_NT), 0, stream, p, P.chunk, P.n_split);
    return hipGetLastError();
}
hipError_t launch_attn_paged(const AttnPaged &p, hipStream_t stream) {
    if (p.tok_start)
        return p.kv.type == TY_F16 ? run_paged_d<_Float16, true>(p, stream) : run_paged_d<__bf16, true>(p, stream);
    return p.kv.type == TY_F16 ? run_paged_d<_Float16, false>(p, stream) : run_paged_d<__bf16, false>(p, stream);
}

}  // namespace s2x
