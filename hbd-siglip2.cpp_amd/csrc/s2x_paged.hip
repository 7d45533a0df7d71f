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
#include "s2x_paged.h"

namespace s2x {

constexpr int PJ_NT = 256;  // threads of the join

// PACKED: rows by tok_start
template <typename TC, int DC, bool EXACT, int KT, int NW, bool PACKED>
__global__ __launch_bounds__(NW * WAVE) void k_attn_paged(AttnPaged p, int chunk, int n_split) {
    const PaWork w = pa_work(blockIdx.x, p.n_seq, n_split, p.kv.n_head * ((p.n_q_head / p.kv.n_head + 15) / 16));
    pa_body<TC, DC, EXACT, KT, NW, PACKED ? PA_PACKED : PA_ROWS>(p, w, chunk, n_split, n_split, 0);
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
