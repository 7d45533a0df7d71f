// s2x_beam.hip -- the best continuations of a beam search.
//
//   S[b, v] = score_b + logit[b, v] - log sum_u exp(logit[b, u])
//
// and the n_out largest of each request, over all its beams b and tokens v; of
// equal ones the lower beam, then the larger logit (S need not tell two small ones
// apart), then the lower token.  Within a beam that is the order of the logits, so
// that a part of a row knows its own.
//
// k_beam_rows: a workgroup's part of a row lies in registers, read once.  Its
// lanes' maxima serve twice: for the reference of a wave's sum of exponentials,
// and for a bound T, the n_out-th largest of the 256 maxima (found bit by bit, by
// counting the lanes at or above).  At least n_out values are >= T, so nothing
// below T is of use; less than n_out lanes hold values > T, so those fit a list in
// LDS whatever the logits are; of values equal to T the first n_out of each wave,
// in the order of tokens, are enough.  The list's members count the larger ones
// among them, which is their rank.
// Bound by the issue of instructions more than by the bytes (an fma, an exponential and
// an addition a logit): 434 live rows of 256,000 bf16 55.5 us = 4.0 TB/s; 4 rows of
// 32,000 f32 6.0 us, of which a launch is 2 to 3.
// k_beam_join: per request, the parts' sums, and the same over their candidates
// with S in f64: the order of two beams' candidates hangs on two sums of many
// terms, where f32 would make ties and swaps of its own.
#include "s2x_device.h"
#include "s2x_search.h"

namespace s2x {

constexpr int BM_NT = 256, BM_WAVES = BM_NT / WAVE;

template <typename T> struct Bm;
// per: values of a lane's 16-byte load; low: bits at the end of an f32 that a value
// of the type leaves 0; largest(): of a load's values, in pairs where the type has
// them, right if it is positive (always: exact)
template <> struct Bm<float> {
    static constexpr int per = 4, low = 0;
    static constexpr bool exact = true;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ float at(const v4u &r, int j) {
        const uint32_t u = r[j];  // (a cast of r[j] itself takes r[0])
        return __builtin_bit_cast(float, u);
    }
    static __device__ __forceinline__ float largest(const v4u &r) {
        return fmaxf(fmaxf(at(r, 0), at(r, 1)), fmaxf(at(r, 2), at(r, 3)));
    }
};
template <> struct Bm<_Float16> {
    static constexpr int per = 8, low = 13;
    static constexpr bool exact = true;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float at(const v4u &r, int j) {
        return f16_bits_to_f32((uint16_t)(j & 1 ? r[j / 2] >> 16 : r[j / 2]));
    }
    static __device__ __forceinline__ float largest(const v4u &r) {
        uint32_t m = r[0];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const uint32_t x = r[i];
            asm("v_pk_max_f16 %0, %0, %1" : "+v"(m) : "v"(x));  // (the builtin quiets its operands first)
        }
        const v2 h = __builtin_bit_cast(v2, m);
        return fmaxf((float)h[0], (float)h[1]);
    }
};
template <> struct Bm<__bf16> {
    static constexpr int per = 8, low = 16;
    static constexpr bool exact = false;
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
    typedef short v2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ float at(const v4u &r, int j) {
        return __builtin_bit_cast(float, j & 1 ? r[j / 2] & 0xffff0000u : r[j / 2] << 16);
    }
    // as integers: positive values in order, above all negative ones
    static __device__ __forceinline__ float largest(const v4u &r) {
        const uint32_t a = r[0], b = r[1], c = r[2], d = r[3];
        const v2 m = __builtin_elementwise_max(__builtin_elementwise_max(__builtin_bit_cast(v2, a), __builtin_bit_cast(v2, b)),
                                               __builtin_elementwise_max(__builtin_bit_cast(v2, c), __builtin_bit_cast(v2, d)));
        const uint32_t u = __builtin_bit_cast(uint32_t, m);
        return fmaxf(__builtin_bit_cast(float, u << 16), __builtin_bit_cast(float, u & 0xffff0000u));
    }
};

// Integers in the order of the values (-0 as +0).
__device__ __forceinline__ uint32_t bm_key(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bm_value(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t bm_key(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}
__device__ __forceinline__ double bm_value(uint64_t k) {
    return __builtin_bit_cast(double, k >> 63 ? k & ~(1ull << 63) : ~k);
}

// The K-th largest of 64 N keys, N of them in each lane of the wave, which are
// the same in every wave; its last `low` bits as its first bit tells.
template <typename U, int N>
__device__ __forceinline__ U bm_kth(const U (&k)[N], int K, int low) {
    U t = 0;
    for (int b = 8 * sizeof(U) - 1; b >= low; --b) {
        const U up = t | (U)1 << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __builtin_popcountll(__builtin_amdgcn_ballot_w64(k[i] >= up));
        if (n >= K) t = up;
    }
    if (!(t >> (8 * sizeof(U) - 1))) t |= ((U)1 << low) - 1;
    return t;
}

// what a sum relative to `from` counts relative to `to` >= from (-inf: an empty sum),
// off by the exponential's 2^-23 alone: what the argument's rounding takes is made up for
__device__ __forceinline__ double bm_scale(float from, float to) {
    if (from == -INFINITY) return 0.0;
    const double x = fmax(((double)from - (double)to) * 1.4426950408889634, -200.0);  // (2^-200: 0)
    const float r = (float)x;
    return (double)__builtin_amdgcn_exp2f(r) * fma(x - (double)r, 0.6931471805599453, 1.0);
}

// How many of a list's C members are ahead of member e, counted by a quad (its lanes
// have the same e); ahead(q): whether member q is.
template <typename F>
__device__ __forceinline__ int bm_rank(int C, F ahead) {
    int n = 0;
#pragma unroll 4
    for (int q = threadIdx.x & 3; q < C; q += 4) n += ahead(q);
    n += dpp_i<0xb1>(n);
    return n + dpp_i<0x4e>(n);
}

// The wave's largest, in all lanes.
__device__ __forceinline__ float bm_wave_max(float v) {
    const int m = __builtin_bit_cast(int, group16_max(v));
    auto row = [&](int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(m, 16 * i)); };
    return fmaxf(fmaxf(row(0), row(1)), fmaxf(row(2), row(3)));
}
// f(0) + .. + f(N - 1) in pairs.
template <int N, typename F>
__device__ __forceinline__ float bm_pairs(F f) {
    if constexpr (N == 1) return f(0);
    else return bm_pairs<N / 2>(f) + bm_pairs<N / 2>([&](int j) { return f(j + N / 2); });
}

// Workspace: candidates [row][split][K] (value, token; token -1: none), then the
// sums [row][split] of 2^(x log2 e - top) and their tops.
struct BmCand {
    float   x;
    int32_t token;
};
struct BmSum {
    double sum;
    float  top;
    int    pad;
};
struct BmPlan {
    int loads, span, n_split;
};
// Parts of a row: up to 16 loads a lane, fewer where rows are few, as long as that
// takes no more than 512 workgroups and the join has a request's candidates in one
// round.  2, 4, 8, 16 loads, both launches, f32: 1 request of 4 beams of 32,000 12.5, 13.0,
// 13.8, 14.5 us; 14 of 5 of 56,284 20.6, 18.4, 17.7, 18.7; 60 of 2 of 30,000 17.8, 15.6,
// 14.9, 14.9; 1 of 8 of 100,000 (8 out) 24.9, 16.5, 16.9, 17.6; 13 of 12 of 50,000 (24 out)
// 42.2, 35.7, 28.6, 29.1; 1 of 32 of 32,000 (64 out) 86, 52, 36, 39; 64 of 8 of 256,000
// bf16 (16 out) 123, 94, 67, 64.
constexpr int BJ_PER = 8, BJ_TILE = BM_NT * BJ_PER;  // candidates of a round of 256 threads
static BmPlan bm_plan(int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out, int per) {
    auto parts = [&](int loads) { return (n_vocab + loads * BM_NT * per - 1) / (loads * BM_NT * per); };
    int loads = 16;
    while (loads > 2 && n_req * n_beam * parts(loads / 2) <= 512 && n_beam * n_out * parts(loads / 2) <= BJ_TILE) loads /= 2;
    const int64_t n = parts(loads);
    int64_t span = (n_vocab + n - 1) / n;
    span = (span + per - 1) / per * per;
    return BmPlan{loads, (int)span, (int)((n_vocab + span - 1) / span)};
}
static int64_t bm_most_splits(int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out) {  // whatever the type
    const int a = bm_plan(n_req, n_beam, n_vocab, n_out, 4).n_split, b = bm_plan(n_req, n_beam, n_vocab, n_out, 8).n_split;
    return a > b ? a : b;
}
size_t beam_select_workspace(int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out) {
    const int64_t parts = n_req * n_beam * bm_most_splits(n_req, n_beam, n_vocab, n_out);
    return (size_t)parts * (sizeof(BmSum) + n_out * sizeof(BmCand));
}
__device__ __forceinline__ BmSum *bm_sums(const BeamSelect &p) { return (BmSum *)p.ws; }
__device__ __forceinline__ BmCand *bm_cands(const BeamSelect &p, int n_split) {
    return (BmCand *)(bm_sums(p) + (int64_t)p.n_req * p.n_beam * n_split);
}
// 0: no beam, 1: a beam, 2: one that has ended
__device__ __forceinline__ int bm_state(const BeamSelect &p, int row) {
    const float s = p.scores[row];
    return !(fabsf(s) < INFINITY) ? 0 : p.done && p.done[row] ? 2 : 1;
}

template <typename T, int NL>
__global__ __launch_bounds__(BM_NT) void k_beam_rows(BeamSelect p, int span, int n_split, int cap) {
    constexpr int PER = Bm<T>::per, STEP = BM_NT * PER;
    extern __shared__ __align__(16) uint8_t lds[];
    uint64_t *list = reinterpret_cast<uint64_t *>(lds);  // key | ~place, `cap` entries
    __shared__ float tops[BM_NT];
    __shared__ double wsum[BM_WAVES];
    __shared__ float wtop[BM_WAVES];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y, split = blockIdx.x;
    // (few loads a lane: latency counts, and they do not wait for the beam's state)
    if (NL > 4 && bm_state(p, row) != 1) return;  // (uniform)
    const int from = split * span, n = min(span, p.n_vocab - from), K = p.n_out;
    const T *x = (const T *)p.logits + (int64_t)row * p.ld + from;
    if (tid == 0) count = 0;

    v4u r[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int c = i * STEP + tid * PER;
        if (c + PER <= n) {
            r[i] = __builtin_bit_cast(v4u, *reinterpret_cast<const typename Bm<T>::vec *>(x + c));
        } else {
            T t[PER];
#pragma unroll
            for (int j = 0; j < PER; ++j) t[j] = c + j < n ? x[c + j] : (T)-INFINITY;
            __builtin_memcpy(&r[i], t, 16);
        }
    }
    if (NL <= 4 && bm_state(p, row) != 1) return;  // (uniform)
    float mi[NL], top = -INFINITY;
    auto each_value = [&]() {  // mi and top from the values one by one
        top = -INFINITY;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            mi[i] = Bm<T>::at(r[i], 0);
#pragma unroll
            for (int j = 1; j < PER; ++j) mi[i] = fmaxf(mi[i], Bm<T>::at(r[i], j));
            top = fmaxf(top, mi[i]);
        }
    };
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        mi[i] = Bm<T>::largest(r[i]);
        top = fmaxf(top, mi[i]);
    }
    if (!Bm<T>::exact && __builtin_amdgcn_ballot_w64(!(top > 0.0f)) != 0) each_value();
    tops[tid] = top;
    // the sum relative to the wave's largest, of 2^(x L - c), c the rounded top L.  With
    // log2(e) = L + LT the exponent is (x - top) (L + LT) = (x L - c) + (c - top L) +
    // (x - top) LT: the second part is the same for all, a factor of the sum (at most
    // 2^-12 from 1: its series), and the third is left out, 2^-26 of x - top.  Past 4,096
    // c lacks too much: there by differences.  A load's values are added in f32, in
    // pairs, and those sums in f64: all one after the other in f32, values that repeat
    // were off by up to 36 2^-24, this way by 3 (434 rows of 256,000 bf16 0.7 us slower).
    const float wt = bm_wave_max(top), L = 1.44269502e+00f, c = wt * L;
    double sum = 0.0;
    if (__builtin_amdgcn_ballot_w64(fabsf(wt) > 4096.0f && wt != -INFINITY) == 0) {  // (by a ballot: 8 registers fewer)
        const float ref = wt == -INFINITY ? 0.0f : c;
#pragma unroll
        for (int i = 0; i < NL; ++i)
            sum = sum + (double)bm_pairs<PER>([&](int j) { return __builtin_amdgcn_exp2f(fmaf(Bm<T>::at(r[i], j), L, -ref)); });
        const double t = wt == -INFINITY ? 0.0 : (double)fmaf(-wt, L, c) * 0.6931471805599453;
        sum = wave_dsum(sum) * fma(t, fma(t, 0.5, 1.0), 1.0);
    } else {
#pragma unroll
        for (int i = 0; i < NL; ++i)
            sum = sum + (double)bm_pairs<PER>([&](int j) { return __builtin_amdgcn_exp2f((Bm<T>::at(r[i], j) - wt) * L); });
        sum = wave_dsum(sum);
    }
    if (lane == 0) {
        wsum[wave] = sum;
        wtop[wave] = wt;
    }
    __syncthreads();
    uint32_t k4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k4[i] = bm_key(tops[i * WAVE + lane]);
    const float bound = bm_value(bm_kth(k4, K, Bm<T>::low));

    // values above the bound, then the wave's first K equal to it
    if (!Bm<T>::exact && !(bound > 0.0f)) each_value();  // (uniform)
    auto put = [&](float v, int c, int at) { list[at] = (uint64_t)bm_key(v) << 32 | (uint32_t)~c; };
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        if (__builtin_amdgcn_ballot_w64(mi[i] > bound) == 0) continue;
        if (mi[i] > bound) {
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                const float v = Bm<T>::at(r[i], j);
                if (v > bound) put(v, i * STEP + tid * PER + j, atomicAdd(&count, 1));
            }
        }
    }
    if (bound > -INFINITY) {
        int taken = 0;  // (uniform over the wave)
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            if (taken >= K || __builtin_amdgcn_ballot_w64(mi[i] >= bound) == 0) continue;
            int here = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) here += Bm<T>::at(r[i], j) == bound;
            int in = here;
#pragma unroll
            for (int o = 1; o < WAVE; o <<= 1) {
                const int t = __shfl_up(in, o);
                if (lane >= o) in += t;
            }
            int rank = taken + in - here;
            taken += __shfl(in, WAVE - 1);
#pragma unroll
            for (int j = 0; j < PER; ++j) {
                if (Bm<T>::at(r[i], j) == bound && rank++ < K) put(bound, i * STEP + tid * PER + j, atomicAdd(&count, 1));
            }
        }
    }
    __syncthreads();
    const int C = min(count, cap);
    const int64_t part = (int64_t)row * n_split + split;
    BmCand *out = bm_cands(p, n_split) + part * K;
    for (int e = tid >> 2; e < C; e += BM_NT / 4) {
        const uint64_t k = list[e];
        const int rank = bm_rank(C, [&](int q) { return list[q] > k; });
        if (rank < K && (tid & 3) == 0) out[rank] = BmCand{bm_value((uint32_t)(k >> 32)), from + (int)~(uint32_t)k};
    }
    for (int e = C + tid; e < K; e += BM_NT) out[e] = BmCand{-INFINITY, -1};
    if (tid < BM_WAVES) {  // (a quad)
        static_assert(BM_WAVES == 4, "a lane a wave");
        const float t = wtop[tid];
        float wt = fmaxf(t, dpp_f<0xb1>(t));
        wt = fmaxf(wt, dpp_f<0x4e>(wt));
        double s = wsum[tid] * bm_scale(t, wt);
        s = s + dpp_d<0xb1>(s);
        s = s + dpp_d<0x4e>(s);
        if (tid == 0) bm_sums(p)[part] = BmSum{s, wt, 0};
    }
}

constexpr int BJ_SUMS = 1024;  // sums kept in LDS

template <int NT>
__global__ __launch_bounds__(NT) void k_beam_join(BeamSelect p, int n_split) {
    constexpr int WAVES = NT / WAVE, TILE = NT * BJ_PER, BJ_CAP = NT == 256 ? 1024 : 2048;  // members of a list
    static_assert((BEAM_MAX_OUT - 1) * (BJ_PER + 1) + WAVES * BEAM_MAX_OUT <= BJ_CAP, "the list's largest length");
    __shared__ double add[BEAM_MAX_OUT];  // score - lse of the beams; -inf: none
    __shared__ uint8_t state[BEAM_MAX_OUT];
    // a member's key, what orders equal ones (63 - beam, the logit's key, ~place: 6, 32
    // and 14 bits) and its token
    static_assert(BEAM_MAX_OUT <= 64 && NT * (BJ_PER + 1) <= 1 << 14, "beam and place in their bits");
    __shared__ uint64_t tops[NT], lk[BJ_CAP], lo[BJ_CAP];
    __shared__ int32_t lt[BJ_CAP];
    __shared__ uint64_t bk[BEAM_MAX_OUT], bo[BEAM_MAX_OUT];  // the best so far, in order
    __shared__ int32_t bt[BEAM_MAX_OUT];
    __shared__ BmSum ls[BJ_SUMS];
    __shared__ int count, ties;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, req = blockIdx.x, K = p.n_out;
    const BmSum *sums = bm_sums(p) + (int64_t)req * p.n_beam * n_split;
    const BmCand *cands = bm_cands(p, n_split) + (int64_t)req * p.n_beam * n_split * K;
    const int per_beam = n_split * K, all = p.n_beam * per_beam, n_sum = p.n_beam * n_split;
    // all loads that wait for nothing: the sums (of beams that have none: whatever
    // is there, not used), the first round's candidates
    const bool kept = n_sum <= BJ_SUMS;
    if (kept)
        for (int i = tid; i < n_sum; i += NT) ls[i] = sums[i];
    BmCand first[BJ_PER];
#pragma unroll
    for (int i = 0; i < BJ_PER; ++i) first[i] = cands[min(i * NT + tid, all - 1)];
    if (tid < p.n_beam) state[tid] = bm_state(p, req * p.n_beam + tid);
    if (tid < K) {
        bk[tid] = bm_key(-(double)INFINITY);
        bo[tid] = 0;
        bt[tid] = -1;
    }
    __syncthreads();
    for (int b = wave; b < p.n_beam; b += WAVES) {
        const int st = state[b];
        const BmSum *from = kept ? ls + b * n_split : sums + (int64_t)b * n_split;
        float top = -INFINITY;
        double s = 0.0;
        if (st == 1) {
            for (int i = lane; i < n_split; i += WAVE) top = fmaxf(top, from[i].top);
            top = bm_wave_max(top);
            for (int i = lane; i < n_split; i += WAVE) {
                const BmSum q = from[i];
                s += q.sum * bm_scale(q.top, top);
            }
            s = wave_dsum(s);
        }
        if (lane == 0) {
            // (no finite sum, from a NaN or an infinity, and no value at all: no candidates)
            const double score = (double)p.scores[req * p.n_beam + b], lse = log(s) + (double)top;
            add[b] = st == 2 ? score : st == 1 && fabs(lse) < INFINITY ? score - lse : -INFINITY;
        }
    }
    const int step_b = NT / per_beam, step_r = NT - step_b * per_beam;
    for (int e0 = 0; e0 < all; e0 += TILE) {
        __syncthreads();
        if (tid == 0) count = ties = 0;
        // this round's candidates, and the best of those before as places below
        // all of them
        const uint64_t none = bm_key(-(double)INFINITY);
        uint64_t key[BJ_PER + 1], beams = 0;  // (63 - beam in 6 bits each)
        uint32_t logit[BJ_PER + 1];
        int32_t tok[BJ_PER + 1];
        key[0] = none;
        logit[0] = 0;
        tok[0] = -1;
        if (tid < K) {
            key[0] = bk[tid];
            logit[0] = (uint32_t)(bo[tid] >> 14);
            beams = bo[tid] >> 46;
            tok[0] = bt[tid];
        }
        auto ord = [&](int i) { return (beams >> 6 * i & 63) << 32 | logit[i]; };
        int b = (e0 + tid) / per_beam, rest = e0 + tid - b * per_beam;
#pragma unroll
        for (int i = 1; i <= BJ_PER; ++i) {
            if (i > 1) {
                b += step_b;
                rest += step_r;
                if (rest >= per_beam) {
                    rest -= per_beam;
                    ++b;
                }
            }
            key[i] = none;
            logit[i] = 0;
            tok[i] = -1;
            const int e = e0 + (i - 1) * NT + tid;
            if (e >= all) continue;
            beams |= (uint64_t)(63 - b) << 6 * i;
            if (state[b] == 2) {
                if (rest == 0) {
                    key[i] = bm_key(add[b]);
                    tok[i] = p.done_token;
                }
            } else if (add[b] > -INFINITY) {
                const BmCand c = e0 ? cands[e] : first[i - 1];
                if (c.token >= 0) key[i] = bm_key(add[b] + (double)c.x);
                logit[i] = bm_key(c.x);
                tok[i] = c.token;
            }
        }
        uint64_t top = key[0];
#pragma unroll
        for (int i = 1; i <= BJ_PER; ++i) top = max(top, key[i]);
        tops[tid] = top;
        __syncthreads();
        // a bound by the upper halves of the keys first: enough unless more keys
        // than the list takes share the bound's (many equal scores), then by whole keys
        uint32_t h4[WAVES];
#pragma unroll
        for (int i = 0; i < WAVES; ++i) h4[i] = (uint32_t)(tops[i * WAVE + lane] >> 32);
        const uint32_t hb = bm_kth(h4, K, 0);
        auto put = [&](int i) {
            const int at = atomicAdd(&count, 1);
            lk[at] = key[i];
            lo[at] = ord(i) << 14 | (uint64_t)((1 << 14) - 1 - (i * NT + tid));
            lt[at] = tok[i];
        };
        int eq = 0;
#pragma unroll
        for (int i = 0; i <= BJ_PER; ++i) eq += (uint32_t)(key[i] >> 32) == hb && key[i] > none;
        eq = group_isum<64>(eq);
        if (lane == 0 && eq) atomicAdd(&ties, eq);
        __syncthreads();
        if (ties <= BJ_CAP - (BEAM_MAX_OUT - 1) * (BJ_PER + 1)) {  // (uniform)
#pragma unroll
            for (int i = 0; i <= BJ_PER; ++i)
                if ((uint32_t)(key[i] >> 32) >= hb && key[i] > none) put(i);
        } else {
            // and of those equal to the bound by their order, in the same way: lanes
            // whose largest is above the bound are above all of them
            uint64_t k4[WAVES];
#pragma unroll
            for (int i = 0; i < WAVES; ++i) k4[i] = tops[i * WAVE + lane];
            const uint64_t bound = bm_kth(k4, K, 0);
            __syncthreads();
            uint64_t first_of = top > bound ? ~0ull : 0;
#pragma unroll
            for (int i = 0; i <= BJ_PER; ++i)
                if (key[i] == bound) first_of = max(first_of, ord(i));
            tops[tid] = first_of;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < WAVES; ++i) k4[i] = tops[i * WAVE + lane];
            const uint64_t bound_o = bm_kth(k4, K, 0);
            int taken = 0;
#pragma unroll
            for (int i = 0; i <= BJ_PER; ++i) {
                const bool at = key[i] == bound && bound > none;
                if (key[i] > bound || (at && ord(i) > bound_o)) put(i);
                const bool is = at && ord(i) == bound_o;
                const uint64_t m = __builtin_amdgcn_ballot_w64(is);
                if (is && taken + __builtin_popcountll(m & ((1ull << lane) - 1)) < K) put(i);
                taken += __builtin_popcountll(m);
            }
        }
        __syncthreads();
        const int C = min(count, BJ_CAP);
        for (int e = tid >> 2; e < C; e += NT / 4) {
            const uint64_t k = lk[e], o = lo[e];
            const int rank = bm_rank(C, [&](int q) { return lk[q] > k || (lk[q] == k && lo[q] > o); });
            if (rank < K && (tid & 3) == 0) {
                bk[rank] = k;
                bo[rank] = o;
                bt[rank] = lt[e];
            }
        }
        for (int e = C + tid; e < K; e += NT) {
            bk[e] = none;
            bo[e] = 0;
            bt[e] = -1;
        }
    }
    __syncthreads();
    if (tid < K) {
        const bool there = bk[tid] > bm_key(-(double)INFINITY);
        const int64_t at = (int64_t)req * K + tid;
        p.parent[at] = there ? req * p.n_beam + 63 - (int)(bo[tid] >> 46) : -1;
        p.token[at] = there ? bt[tid] : -1;
        p.score[at] = there ? (float)bm_value(bk[tid]) : -INFINITY;
    }
}

template <typename T>
static hipError_t run_beam(const BeamSelect &p, hipStream_t stream) {
    const int rows = p.n_req * p.n_beam;
    const BmPlan P = bm_plan(p.n_req, p.n_beam, p.n_vocab, p.n_out, Bm<T>::per);
    const int cap = (p.n_out - 1) * P.loads * Bm<T>::per + BM_WAVES * p.n_out;
    auto kern = P.loads == 16 ? k_beam_rows<T, 16> : P.loads == 8 ? k_beam_rows<T, 8> : P.loads == 4 ? k_beam_rows<T, 4>
                                                                                                     : k_beam_rows<T, 2>;
    hipLaunchKernelGGL(kern, dim3(P.n_split, rows), dim3(BM_NT), (size_t)cap * 8, stream, p, P.span, P.n_split, cap);
    // (1,024 threads where 256 need more than a round: 7 requests of 32 beams of 4 parts of
    // 64 candidates 50.5 us, both launches, 74.9 with 256; 64 of 8 of 8 of 16 73.9 and 65.2)
    const bool wide = (int64_t)p.n_beam * P.n_split * p.n_out > BJ_TILE;
    hipLaunchKernelGGL(wide ? k_beam_join<1024> : k_beam_join<256>, dim3(p.n_req), dim3(wide ? 1024 : 256), 0, stream, p, P.n_split);
    return hipGetLastError();
}
hipError_t launch_beam_select(const BeamSelect &p, hipStream_t stream) {
    switch (p.type) {
    case TY_F32: return run_beam<float>(p, stream);
    case TY_F16: return run_beam<_Float16>(p, stream);
    default: return run_beam<__bf16>(p, stream);
    }
}

}  // namespace s2x
