// s2x_prefix.hip -- attention of one new token per sequence where groups of
// sequences share their first tokens.
//
//   out = (sum over the prefix + sum over the own tokens), each with its running
//   maximum and sum, joined by e^(maximum - the larger one)
//
// The prefix's keys and values are read once for all query heads of the group that
// share a key head (its columns).  Up to 16 columns take the kernel of the decode
// step's attention, a wave a tile (s2x_paged.h), and so do the own tokens.  More
// columns: px_wide, whose waves share tiles of 32 keys in LDS and have 16 or 32
// columns each.  All leave sums in the workspace; k_prefix_join adds them.
//
// Measured (both launches): 3 groups of 4 on up to 700 tokens, 16 heads of 72, 11.9 us,
// latency and launches; 9 groups of up to 30, up to 6,000 tokens, 32 / 8 heads of 128, 71
// us = 2.3 TB/s, the own tokens 15 to 20 of it; 1 group of 64 on 32,001 tokens, bf16, 91 to
// 98 us = 345 to 370 TFLOP/s of the two products counted once (three terms of a
// probability make the second one three).  px_wide is bound by the issue of its
// instructions: a step of 32 keys and 128 columns takes a workgroup some 3,000 cycles, of
// which the matrix units work 46 %, with two workgroups a CU for the other half.  Each
// 256 registers; 8 waves of 16 columns in 128 spill (109 us against 79 of that time's).
#include "s2x_paged.h"

namespace s2x {

// Parts of a launch: the prefixes' in chunks of chunk_p, then the own tokens'.
struct PxPlan {
    int     nc, tiles;  // of the prefix; nc 0: the form of up to 16 columns
    int     chunk_p, split_p, chunk_o, split_o;
    int64_t wgs_p, wgs_o;
    __host__ __device__ int parts() const { return split_p + split_o; }
};

// Own tokens: a wave a sequence, key head and chunk (of few keys, mostly: four waves
// on one would be tiles of which some have none).  The four of a workgroup are
// neighbours in the order of workgroups of its XCD.
template <typename TC, int DC, bool EXACT, int KT>
__device__ __forceinline__ void px_own(const AttnPrefix &p, const PxPlan &P) {
    const int w = blockIdx.x - (int)P.wgs_p, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H = p.a.kv.n_head * ((p.a.n_q_head / p.a.kv.n_head + 15) / 16);
    for (int bid = w / 8 * 32 + wave * 8 + w % 8; bid < p.a.n_seq * P.split_o * H; bid += (int)P.wgs_o * 4)
        pa_body<TC, DC, EXACT, KT, 1, PA_OWN>(p, pa_work(bid, p.a.n_seq, P.split_o, H), P.chunk_o, P.split_o, P.parts(), P.split_p);
}

// A workgroup's part of the prefixes: the tiles of columns, then the heads, of one
// chunk follow each other on one XCD, the chunks of a group lie on different ones.
struct PxWork {
    int tile, hk, group, split;
};
__device__ __forceinline__ PxWork px_work(const AttnPrefix &p, const PxPlan &P) {
    const PaWork w = pa_work(blockIdx.x, p.n_group, P.split_p, p.a.kv.n_head * P.tiles);
    const int hk = w.hp / P.tiles;
    return PxWork{w.hp - hk * P.tiles, hk, w.unit, w.split};
}

constexpr int PX_TK = 32, PX_NT = 4 * WAVE;  // keys of a tile, threads
constexpr int PX_PAD_K = 8, PX_PAD_V = 16;   // rows in LDS end with these: reads of 16 rows spread over the banks

// The reference of a column's exponentials follows its largest score in steps: it
// moves once that is PX_ROOM (as a power of two) above, so that few tiles rescale
// the sums.  A probability is up to 2^PX_ROOM then, times 2^px_up for f16, whose
// second term reaches 2^-35 of the largest; the sums leave as Pa::up has them.
constexpr float PX_ROOM = 4.0f;
template <typename TC> constexpr float px_up = 0.0f;
template <> constexpr float px_up<_Float16> = 11.0f;

// Two probabilities (times 2^px_up) as sums of terms of the cache's type: bf16 by
// cutting off, which leaves nothing after three; f16 by rounding.
__device__ __forceinline__ void px_terms(float x, float y, uint32_t (&t)[2]) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const v2h h = __builtin_convertvector((v2f{f32_materialize(x), f32_materialize(y)}), v2h);
    const v2f r = {fmaf((float)h[0], -1.0f, x), fmaf((float)h[1], -1.0f, y)};
    t[0] = __builtin_bit_cast(uint32_t, h);
    t[1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, v2h));
}
__device__ __forceinline__ void px_terms(float x, float y, uint32_t (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t a = __builtin_bit_cast(uint32_t, x), b = __builtin_bit_cast(uint32_t, y);
        t[i] = __builtin_amdgcn_perm(b, a, 0x07060302);  // the upper halves
        x = x - __builtin_bit_cast(float, a & 0xffff0000u);
        y = y - __builtin_bit_cast(float, b & 0xffff0000u);
    }
}

// NC: 16-column parts of a wave.  A step: the next tile's pieces into registers,
// the products of this one, the pieces into the other half of LDS, one barrier.
// S^T and O^T as in s2x_paged.h.
template <typename TC, int DC, bool EXACT, int NC>
__device__ __forceinline__ void px_wide(const AttnPrefix &args, const PxPlan &P, const PxWork &w, const PaGroup &gr) {
    typedef typename Pa<TC>::vec vec;
    constexpr int DP = 32 * DC, DT = 2 * DC, NT = PX_NT, NP = Pa<TC>::terms;
    constexpr int PER = (PX_TK * (DP / 8) + NT - 1) / NT;  // pieces of a thread
    constexpr bool ALL = EXACT && PX_TK * (DP / 8) % NT == 0;  // all of them there
    extern __shared__ __align__(16) uint8_t lds[];
    const AttnPaged &p = args.a;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = EXACT ? DP : p.kv.d_head, nch = d / 8, sk = d + PX_PAD_K, sv = d + PX_PAD_V;
    const int share = p.n_q_head / p.kv.n_head;
    const int hk = w.hk, split = w.split, cols = gr.size * share, c0 = w.tile * (16 * NC * 4);
    const int64_t start = (int64_t)split * P.chunk_p, end = min(start + P.chunk_p, gr.len);
    if (c0 >= cols || start >= end) return;  // (uniform)

    const TC *kp = (const TC *)p.kv.k + hk * p.kv.ld_head, *vp = (const TC *)p.kv.v + hk * p.kv.ld_head;
    const int32_t *row = p.table + (int64_t)gr.first * p.ld_table;
    const uint32_t pmask = (1u << p.kv.page_shift) - 1, ldp = (uint32_t)p.kv.ld_page, ldt = (uint32_t)p.kv.ld_tok;
    TC *kl = reinterpret_cast<TC *>(lds), *vl = kl + 2 * PX_TK * sk;

    // Table entries: of key t0 + lane % 32 (`mask`, for which keys there are) and of
    // the keys of this thread's pieces; the row's last one for keys past it.
    struct Entries {
        int32_t mask, piece[PER];
    };
    const int last = (int)p.ld_table - 1, shift = p.kv.page_shift;
    const uint32_t magic = (65536u + nch - 1) / nch;  // f / nch for f < 1,024
    auto key_of = [&](int i) -> uint32_t {
        const uint32_t f = i * NT + tid;
        return (EXACT ? f / (DP / 8) : f * magic >> 16) & (PX_TK - 1);
    };
    auto entries = [&](int64_t t0) {
        Entries e;
        e.mask = row[min((int)((uint32_t)(t0 + (lane & (PX_TK - 1))) >> shift), last)];
#pragma unroll
        for (int i = 0; i < PER; ++i) e.piece[i] = row[min((int)((uint32_t)(t0 + key_of(i)) >> shift), last)];
        return e;
    };
    // Two tiles under way where the registers allow: a step of a workgroup takes over a
    // microsecond, a load from memory two under full use.  Where a page is none the
    // first one is loaded, and zeros are stored.
    constexpr int AHEAD = DC > 4 ? 1 : 2;
    struct Piece {
        vec      k[PER], v[PER];
        uint32_t seen;
    } even, odd;
    auto load = [&](Piece &x, int64_t t0, const Entries &e) {
        x.seen = (uint32_t)__builtin_amdgcn_ballot_w64(t0 + (lane & (PX_TK - 1)) < end && (uint32_t)e.mask < (uint32_t)p.kv.n_pages);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t f = i * NT + tid, key = key_of(i);
            const uint32_t pid = (uint32_t)e.piece[i] < (uint32_t)p.kv.n_pages ? (uint32_t)e.piece[i] : 0u;
            const uint32_t piece = ALL || f < (uint32_t)(PX_TK * nch) ? f - (EXACT ? f / (DP / 8) : f * magic >> 16) * nch : 0u;
            const uint64_t at = (uint64_t)pid * ldp + ((((uint32_t)t0 + key) & pmask) * (uint64_t)ldt + 8 * piece);
            x.k[i] = *reinterpret_cast<const vec *>(kp + at);
            x.v[i] = *reinterpret_cast<const vec *>(vp + at);
        }
    };
    auto store = [&](Piece &x, int buf) {
        if (x.seen != ~0u) {  // (uniform)
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (!(x.seen >> key_of(i) & 1)) x.k[i] = x.v[i] = vec{};
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t f = i * NT + tid, key = EXACT ? f / (DP / 8) : f * magic >> 16;
            if (ALL || f < (uint32_t)(PX_TK * nch)) {
                *reinterpret_cast<vec *>(kl + (buf * PX_TK + key) * sk + 8 * (f - key * nch)) = x.k[i];
                *reinterpret_cast<vec *>(vl + (buf * PX_TK + key) * sv + 8 * (f - key * nch)) = x.v[i];
            }
        }
    };
    Entries next;
    {
        Entries e0 = entries(start), e1 = entries(start + PX_TK);
        next = AHEAD == 2 ? entries(start + 2 * PX_TK) : e1;
        if (pa_freed(p, gr.first)) {  // (asked while the entries are on their way; uniform)
            row = p.table + (int64_t)pa_holder(p, gr) * p.ld_table;
            e0 = entries(start), e1 = entries(start + PX_TK);
            next = AHEAD == 2 ? entries(start + 2 * PX_TK) : e1;
        }
        load(even, start, e0);
        if constexpr (AHEAD == 2) load(odd, start + PX_TK, e1);
    }

    // the queries; a negative scale goes into them, so that the largest score is
    // the largest product, and so does one of zero (an unseen place is -inf)
    const int w0 = c0 + wave * 16 * NC;
    const bool live = w0 < cols, neg = p.scale < 0.0f;
    const float sc = p.scale == 0.0f ? 1.0f : fabsf(p.scale) * 1.44269504088896341f;  // log2(e)
    vec q[NC][DC];
    int64_t lim[NC];
    bool ragged = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = w0 + 16 * n + r, i = min(c, cols - 1) / share, s = gr.first + i;
        const int64_t qrow = pa_row_of(p, s);
        lim[n] = pa_len(p, s);
        ragged |= __builtin_amdgcn_ballot_w64(lim[n] < end) != 0;
#pragma unroll
        for (int k = 0; k < DC; ++k) {
            v4u t = {0, 0, 0, 0};
            if (c < cols && qrow >= 0 && (EXACT || 32 * k + 8 * g < d))
                t = *reinterpret_cast<const v4u *>((const TC *)p.q + qrow * p.ld_q + (int64_t)(hk * share + c - i * share) * d +
                                                   32 * k + 8 * g);
            if (neg) t = t ^ 0x80008000u;
            if (p.scale == 0.0f) t = v4u{0, 0, 0, 0};
            q[n][k] = __builtin_bit_cast(vec, t);
        }
    }

    float m[NC], l[NC];
    v4f o[NC][DT];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[n][i] = v4f{0, 0, 0, 0};
    }
    store(even, 0);
    __syncthreads();
    auto step = [&](Piece &x, Piece &y, int buf, int64_t t0) {  // tile t0, loaded by way of x; y: the next one
        const uint32_t mask = x.seen;
        // the keys out of LDS, then the loads of tiles to come (their entries first: a
        // wait for one is a wait for the loads before it, too), then the scores
        const TC *kt = kl + buf * PX_TK * sk;
        vec kk[DC][2];
#pragma unroll
        for (int k = 0; k < DC; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                kk[k][j] = vec{};
                if (EXACT || 32 * k + 8 * g < d) kk[k][j] = *reinterpret_cast<const vec *>(kt + (16 * j + r) * sk + 32 * k + 8 * g);
            }
        if (t0 + AHEAD * PX_TK < end) {  // (uniform)
            const Entries after = entries(t0 + (AHEAD + 1) * PX_TK);
            load(x, t0 + AHEAD * PX_TK, next);
            next = after;
        }
        if (live) {
            TC *vt = vl + buf * PX_TK * sv;
            v4f st[NC][2];
#pragma unroll
            for (int k = 0; k < DC; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int n = 0; n < NC; ++n) st[n][j] = Pa<TC>::mfma(kk[k][j], q[n][k], k ? st[n][j] : v4f{0, 0, 0, 0});
            // V's fragments (columns past d: the row's end, into sums that are not kept)
            vec a8[DT];
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                v4s a[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    TC *src = vt + (16 * j + 4 * g + (r >> 2)) * sv + min(16 * i, EXACT ? DP : d) + (r & 3) * 4;
                    a[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)src);
                }
                a8[i] = __builtin_bit_cast(vec, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
            }
            if (mask != ~0u || ragged) {  // (uniform)
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const int left = (int)min(max(lim[n] - t0, (int64_t)0), (int64_t)PX_TK);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int key = 16 * (e >> 2) + 4 * g + (e & 3);
                        if (!(mask >> key & 1) || key >= left) st[n][e >> 2][e & 3] = -INFINITY;
                    }
                }
            }
            float mt[NC];
            bool above = false;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                mt[n] = st[n][0][0];
#pragma unroll
                for (int e = 1; e < 8; ++e) mt[n] = fmaxf(mt[n], st[n][e >> 2][e & 3]);
                mt[n] = mt[n] * sc;
                above |= mt[n] > m[n] + PX_ROOM;
            }
            if (__builtin_amdgcn_ballot_w64(above) != 0) {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    mt[n] = fmaxf(mt[n], __shfl_xor(mt[n], 16));
                    mt[n] = fmaxf(mt[n], __shfl_xor(mt[n], 32));
                    const float mn = fmaxf(m[n], mt[n]), b = mn == -INFINITY ? 0.0f : mn;
                    const float alpha = __builtin_amdgcn_exp2f(m[n] - b);
                    m[n] = mn;
                    l[n] = l[n] * alpha;
#pragma unroll
                    for (int i = 0; i < DT; ++i) o[n][i] = o[n][i] * alpha;
                }
            }
            // column part n's probabilities, then its products while n + 1's
            // probabilities are computed
            uint32_t pt[NC][NP][4];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                // (times 2^px_up, which the sum of them is then divided by)
                const float base = (m[n] == -INFINITY ? 0.0f : m[n]) - px_up<TC>;
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float x = __builtin_amdgcn_exp2f(fmaf(st[n][e >> 2][e & 3], sc, -base));
                    const float y = __builtin_amdgcn_exp2f(fmaf(st[n][e >> 2][(e & 3) + 1], sc, -base));
                    l[n] = l[n] + (x + y);
                    uint32_t t[NP];
                    px_terms(x, y, t);
#pragma unroll
                    for (int k = 0; k < NP; ++k) pt[n][k][e >> 1] = t[k];
                }
#pragma unroll
                for (int k = 0; k < NP; ++k)
#pragma unroll
                    for (int i = 0; i < DT; ++i)
                        o[n][i] = Pa<TC>::mfma(a8[i], __builtin_bit_cast(vec, (v4u{pt[n][k][0], pt[n][k][1], pt[n][k][2], pt[n][k][3]})),
                                               o[n][i]);
            }
            if constexpr (NC == 2) {
                __builtin_amdgcn_sched_group_barrier(0x406, 80, 0);  // part 0's probabilities
#pragma unroll
                for (int i = 0; i < NP * DT; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x406, 4, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x8, NP * DT, 0);
            }
        }
        if (t0 + PX_TK < end) store(y, buf ^ 1);
        __syncthreads();
    };
    for (int64_t t0 = start; t0 < end; t0 += 2 * PX_TK) {
        step(even, AHEAD == 2 ? odd : even, 0, t0);
        if (t0 + PX_TK < end) step(AHEAD == 2 ? odd : even, even, 1, t0 + PX_TK);
    }

    // o[n][i] is values 16 i + 4 g .. + 3 of column w0 + 16 n + r
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        l[n] = l[n] + __shfl_xor(l[n], 16);
        l[n] = l[n] + __shfl_xor(l[n], 32);
        const int c = w0 + 16 * n + r;
        if (c >= cols) continue;
        // (both sums carry 2^px_up; the join takes o with Pa::up, l without)
        l[n] = l[n] * (px_up<TC> == 0.0f ? 1.0f : 0x1p-11f);
        const float more = px_up<TC> == 0.0f ? 1.0f : 16.0f;
        const int i = c / share;
        const int64_t at = ((int64_t)(w.group * args.max_group + i) * p.n_q_head + hk * share + c - i * share) * P.parts() + split;
        v4f *ov = reinterpret_cast<v4f *>(p.ws) + at * (d / 4);
#pragma unroll
        for (int k = 0; k < DT; ++k) {
            if (!EXACT && 16 * k + 4 * g >= d) break;
            ov[4 * k + g] = o[n][k] * more;
        }
        if (g == 0)
            reinterpret_cast<float2 *>((float *)p.ws + (int64_t)args.n_group * args.max_group * p.n_q_head * P.parts() * d)[at] =
                make_float2(m[n], l[n]);
    }
}

// One launch of all parts.  WIDE: some group may have more than 16 columns; each
// takes the form of its own number.  (The second bound: two workgroups a CU, the
// registers that leaves.)
template <typename TC, int DC, bool EXACT, int KT, bool WIDE>
__global__ __launch_bounds__(PX_NT, 2) void k_attn_prefix(AttnPrefix p, PxPlan P) {
    if (blockIdx.x >= P.wgs_p) return px_own<TC, DC, EXACT, KT>(p, P);
    const PxWork w = px_work(p, P);
    if constexpr (WIDE) {
        const PaGroup gr = pa_group(p, w.group);
        const int cols = gr.size * (p.a.n_q_head / p.a.kv.n_head);
        if (cols > 16) {
            if constexpr (DC <= 4)
                if (P.nc == 2 && cols > 64) return px_wide<TC, DC, EXACT, 2>(p, P, w, gr);
            return px_wide<TC, DC, EXACT, 1>(p, P, w, gr);
        }
        if (w.tile) return;
    }
    pa_body<TC, DC, EXACT, KT, 4, PA_PREFIX>(p, PaWork{w.group, w.split, w.hk}, P.chunk_p, P.split_p, P.parts(), 0);
}

// Four values, from c on, of the sum over the prefix's keys [from, to), relative to
// the score m: for a sequence that ends inside a chunk.  The chunk's sums count keys
// behind its end 0 times their value, which is no 0 where that is infinite or NaN;
// then those that it sees once more, one after the other.  (A wrong sum shows: it is
// no number.  m and the sum of the exponentials do not hang on the values.)
template <typename TC>
__device__ __forceinline__ v4f px_seen_only(const AttnPaged &p, int seq, int hk, const TC *q, int c, int64_t from, int64_t to, float m) {
    typedef TC vec4 __attribute__((ext_vector_type(4)));
    const int32_t *row = p.table + seq * p.ld_table;
    v4f o = {0, 0, 0, 0};
    for (int64_t t = from; t < to; ++t) {
        const int32_t id = row[t >> p.kv.page_shift];
        if (id < 0 || id >= p.kv.n_pages) continue;
        const int64_t at = (int64_t)hk * p.kv.ld_head + id * p.kv.ld_page + (t & ((1 << p.kv.page_shift) - 1)) * p.kv.ld_tok;
        const TC *kp = (const TC *)p.kv.k + at;
        float s = 0.0f;
        for (int i = 0; i < p.kv.d_head; i += 4) {
            const vec4 a = *reinterpret_cast<const vec4 *>(kp + i), b = *reinterpret_cast<const vec4 *>(q + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) s = fmaf((float)a[k], (float)b[k], s);
        }
        const float x = __builtin_amdgcn_exp2f(s * (p.scale * 1.44269504088896341f) - (m == -INFINITY ? 0.0f : m)) * Pa<TC>::up;
        const vec4 v = *reinterpret_cast<const vec4 *>((const TC *)p.kv.v + at + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = fmaf(x, (float)v[k], o[k]);
    }
    return o;
}

// The parts of a sequence's prefix and of its own tokens joined, as k_attn_join
// does the chunks: a workgroup per query head and 128 values of it.
// The first PXJ_AHEAD parts of a thread are loaded before their number is known.
constexpr int PXJ_AHEAD = 4;
template <typename TC, int NT>
__global__ __launch_bounds__(NT) void k_prefix_join(AttnPrefix args, PxPlan P) {
    constexpr int LANES = 32, GROUPS = NT / LANES;
    __shared__ __align__(16) float part[GROUPS][LANES * 4 + 4];
    __shared__ float gm[GROUPS], gl[GROUPS];
    const AttnPaged &p = args.a;
    const int n_parts = P.parts(), split_p = P.split_p, chunk_o = P.chunk_o;
    const int tid = threadIdx.x, d = p.kv.d_head, nq = d / 4, pieces = (nq + LANES - 1) / LANES;
    const int h = blockIdx.x / pieces, s = blockIdx.y;
    int first;
    const int gi = pa_find(args, s, first);
    const int grp = tid / LANES, e = (blockIdx.x - h * pieces) * LANES + tid % LANES;
    if (first < 0 || s < first || s - first >= args.max_group) return;  // (uniform; no difference past 31 bits)
    const int slot = gi * args.max_group + s - first;
    const int64_t at = ((int64_t)slot * p.n_q_head + h) * n_parts;
    const v4f *ov = reinterpret_cast<const v4f *>(p.ws) + at * nq + min(e, nq - 1);
    const float2 *mlp =
        reinterpret_cast<const float2 *>((const float *)p.ws + (int64_t)args.n_group * args.max_group * p.n_q_head * n_parts * d) + at;
    float2 t[PXJ_AHEAD];
    v4f x[PXJ_AHEAD];
    // part i of those that there are (np of the prefix): its place
    auto fetch = [&](int i0, int np, int n) {
#pragma unroll
        for (int k = 0; k < PXJ_AHEAD; ++k) {
            const int i = i0 + k * GROUPS, q = min(i < np ? i : split_p + i - np, n_parts - 1);
            if (i < n) {
                t[k] = mlp[q];
                x[k] = ov[(int64_t)q * nq];
            }
        }
    };
    fetch(grp, split_p, n_parts);  // (right where the prefix has all its parts)
    const PaGroup gr = pa_group(args, gi);
    const int64_t qrow = pa_row_of(p, s);
    if (s >= gr.first + gr.size || qrow < 0) return;  // (uniform)
    const PaRange own = pa_own(args, gr, s);
    const int np = (int)((own.first + P.chunk_p - 1) / P.chunk_p);  // (those that it sees something of)
    const int n = np + (own.len > own.begin ? (int)((own.len - own.begin + chunk_o - 1) / chunk_o) : 0);
    if (np < split_p) fetch(grp, np, n);
    v4f a = {0, 0, 0, 0};
    float M = -INFINITY, L = 0.0f, redo = NAN;
    const int ends = own.first < min(gr.len, (int64_t)np * P.chunk_p) ? np - 1 : -1;  // the chunk that it ends in
    for (int i0 = grp; i0 < n;) {
#pragma unroll
        for (int k = 0; k < PXJ_AHEAD; ++k) {
            if (i0 + k * GROUPS >= n) break;
            const float mn = fmaxf(M, t[k].x), base = mn == -INFINITY ? 0.0f : mn;
            const float f0 = __builtin_amdgcn_exp2f(M - base), f1 = __builtin_amdgcn_exp2f(t[k].x - base);
            L = fmaf(t[k].y, f1, L * f0);
            if (i0 + k * GROUPS == ends && !(fabsf(x[k][0]) + fabsf(x[k][1]) + fabsf(x[k][2]) + fabsf(x[k][3]) < INFINITY)) {
                redo = t[k].x;
                x[k] = v4f{0, 0, 0, 0};
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) a[c] = fmaf(x[k][c], f1, a[c] * f0);
            M = mn;
        }
        i0 += PXJ_AHEAD * GROUPS;
        fetch(i0, np, n);
    }
    if (__builtin_amdgcn_ballot_w64(redo == redo) != 0) {
        const int holder = pa_holder(p, gr);
        if (redo == redo) {
            const int share = p.n_q_head / p.kv.n_head, ec = min(e, nq - 1);
            const v4f y = px_seen_only<TC>(p, holder, h / share, (const TC *)p.q + qrow * p.ld_q + (int64_t)h * d, 4 * ec,
                                           (int64_t)ends * P.chunk_p, own.first, redo);
            const float f = __builtin_amdgcn_exp2f(redo - (M == -INFINITY ? 0.0f : M));
#pragma unroll
            for (int c = 0; c < 4; ++c) a[c] = fmaf(y[c], f, a[c]);
        }
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

static int64_t px_round(int64_t v, int64_t to, int64_t lo, int64_t hi) {
    v = v < lo ? lo : v > hi ? hi : v;
    return (v + to - 1) / to * to;
}
// Chunks of the prefixes for about 512 workgroups, what the card holds of k_attn_prefix
// at once (1 group of 64 on 32,001 tokens: for 256, 512, 1,024, 2,048 107, 97.5, 108, 132 us;
// 2 of 32 on 12,000: for 512 54, 1,024 59; 9 ragged ones 88, 70.7, 71.5).  Own tokens in
// chunks of 32, up to 128 where that is more than 4,096 waves (12 sequences of 16 heads with
// up to 60: 32 a chunk 11.9 us, 128 15.6; 140 of 8 with up to 900: 83 and 72.6), and at most
// 48 of them a sequence.  Columns of a wave: 16 up to 64 of a group, 32 from there (9 ragged
// groups with 16 83.4 us, with 32 73.0; 1 of 64: 112 and 97.7).
static PxPlan px_plan(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own, int64_t n_q_head,
                      int64_t n_kv_head, int64_t d_head) {
    PxPlan P;
    const int64_t share = n_q_head / n_kv_head, cols = share * max_group;
    P.nc = cols <= 16 ? 0 : cols > 64 && d_head <= 128 ? 2 : 1;
    P.tiles = P.nc ? (int)((cols + 64 * P.nc - 1) / (64 * P.nc)) : 1;
    const int64_t units = n_group * n_kv_head * P.tiles, most = 1 << 20;
    int64_t c = px_round(max_prefix * units / 512, 128, 128, most);
    if (units * ((max_prefix + c - 1) / c) > 1 << 22) c = px_round(max_prefix * units >> 21, 128, 128, 1 << 30);
    P.chunk_p = (int)c;
    P.split_p = (int)((max_prefix + c - 1) / c);
    P.wgs_p = P.split_p * units;
    const int64_t units_o = n_group * max_group * n_kv_head * ((share + 15) / 16), span = max_own + PA_ALIGN;
    c = px_round(span * units_o / 4096, 32, 32, 128);
    if (span > 48 * c) c = px_round(span / 48, 32, 128, (int64_t)1 << 30);
    P.chunk_o = (int)c;
    P.split_o = (int)((span + c - 1) / c);
    P.wgs_o = 0;  // (with the number of sequences)
    return P;
}
size_t attn_prefix_workspace(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own, int64_t n_q_head,
                             int64_t n_kv_head, int64_t d_head) {
    const PxPlan P = px_plan(n_group, max_group, max_prefix, max_own, n_q_head, n_kv_head, d_head);
    return (size_t)(n_group * max_group * n_q_head) * P.parts() * (d_head + 2) * 4;
}

template <typename TC, int DC, bool EXACT>
static hipError_t run_prefix(const AttnPrefix &p, hipStream_t stream) {
    constexpr int KT = DC > 4 ? 1 : 2;
    const int d = p.a.kv.d_head, share = p.a.n_q_head / p.a.kv.n_head;
    PxPlan P = px_plan(p.n_group, p.max_group, p.max_prefix, p.max_own, p.a.n_q_head, p.a.kv.n_head, d);
    P.wgs_o = ((int64_t)P.split_o * p.a.n_seq * p.a.kv.n_head * ((share + 15) / 16) + 31) / 32 * 8;
    if (P.wgs_o > 1 << 20) P.wgs_o = 1 << 20;  // (each takes several then; at most 2^21 x 49 parts in all)
    // LDS of the forms in the launch: pa_body's V tiles and sums of R columns, px_wide's tiles
    const int cols = share * p.max_group, R = cols < 16 ? cols : 16;
    const int v = 4 * KT * 16 * d * 2 + 64, o = 4 * R * (DC * 32 + 4) * 4;
    const int w = P.nc ? 2 * PX_TK * (2 * d + PX_PAD_K + PX_PAD_V) * 2 : 0;
    const int lds = w > v ? (w > o ? w : o) : (v > o ? v : o);
    auto kern = P.nc ? k_attn_prefix<TC, DC, EXACT, KT, true> : k_attn_prefix<TC, DC, EXACT, KT, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(P.wgs_p + P.wgs_o)), dim3(PX_NT), lds, stream, p, P);
    // (a wave a row and 128 values where rows are many, so that all are at work at once: 74
    // sequences of 32 heads and 2 parts 6.8 us, in four waves 8.5; few rows: four, for
    // their parts' sake)
    const bool many = (int64_t)p.a.n_seq * p.a.n_q_head >= 512;
    auto join = many ? k_prefix_join<TC, 64> : k_prefix_join<TC, 256>;
    hipLaunchKernelGGL(join, dim3(p.a.n_q_head * ((d + 127) / 128), p.a.n_seq), dim3(many ? 64 : 256), 0, stream, p, P);
    return hipGetLastError();
}
template <typename TC>
static hipError_t run_prefix_d(const AttnPrefix &p, hipStream_t stream) {
    const int d = p.a.kv.d_head;
    return d == 64    ? run_prefix<TC, 2, true>(p, stream)
           : d == 128 ? run_prefix<TC, 4, true>(p, stream)
           : d == 256 ? run_prefix<TC, 8, true>(p, stream)
           : d < 64   ? run_prefix<TC, 2, false>(p, stream)
           : d <= 96  ? run_prefix<TC, 3, false>(p, stream)
           : d <= 192 ? run_prefix<TC, 6, false>(p, stream)
                      : run_prefix<TC, 8, false>(p, stream);
}
hipError_t launch_attn_prefix(const AttnPrefix &p, hipStream_t stream) {
    return p.a.kv.type == TY_F16 ? run_prefix_d<_Float16>(p, stream) : run_prefix_d<__bf16>(p, stream);
}

}  // namespace s2x
