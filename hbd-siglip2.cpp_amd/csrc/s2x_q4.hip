// s2x_q4.hip -- Q4_0 weights: the repack and the products of few rows.
#include "s2x_decode.h"
#include "s2x_device.h"

namespace s2x {

// One thread per 16-byte piece of a tile: lane l's values of 4 blocks.
__global__ __launch_bounds__(256) void k_repack_q4_0(const uint8_t *__restrict__ raw, int64_t n_piece,
                                                     int64_t KB, int64_t N, int64_t tiles_k,
                                                     uint8_t *__restrict__ qs, uint16_t *__restrict__ d) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n_piece) return;
    const int64_t tile = i / 64;
    const int l = (int)(i % 64), g = l / 16;
    const int64_t tn = tile / tiles_k, tk = tile - tn * tiles_k, n = tn * 16 + l % 16;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t kb = tk * 4 + j;
        if (n >= N || kb >= KB) continue;
        // values 16 (g & 1) + 8 (g >> 1) ..: a half of 8 bytes
        const uint8_t *b = raw + (n * KB + kb) * 18 + 2 + 8 * (g >> 1);
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = g & 1 ? b[k] >> 4 : b[k] & 15, hi = g & 1 ? b[4 + k] >> 4 : b[4 + k] & 15;
            w[j] |= ((lo | hi << 4) ^ 0x88) << (8 * k);
        }
    }
    reinterpret_cast<uint4 *>(qs)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    // scale l of the tile: column l % 16, block g
    const int64_t kb = tk * 4 + g;
    uint16_t v = 0;
    if (n < N && kb < KB) {
        const uint8_t *b = raw + (n * KB + kb) * 18;
        v = (uint16_t)(b[0] | b[1] << 8);
    }
    d[i] = v;
}
hipError_t launch_repack_q4_0(const void *raw, const Q4View &w, hipStream_t stream) {
    const int64_t n = w.tiles_n() * w.tiles_k() * 64;
    hipLaunchKernelGGL(k_repack_q4_0, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream,
                       (const uint8_t *)raw, n, w.K / QK, w.N, w.tiles_k(), const_cast<uint8_t *>(w.qs),
                       const_cast<uint16_t *>(w.d));
    return hipGetLastError();
}

// The weight as the Q8_0 planes of the int8 GEMM, for more rows: exact, a block
// keeps its scale.  A wave a tile: 16 bytes in, 8 values of each of 4 blocks;
// the halves of blocks that lie 32 lanes apart change places
// (v_permlane32_swap), so that a lane stores 16 bytes of one block and a row
// gets 64 bytes a store.  Columns past N (to the plane's whole 128) get zero
// scales alone.
__global__ __launch_bounds__(256) void k_expand_q4(const uint8_t *__restrict__ qs, const uint16_t *__restrict__ d,
                                                   int64_t n_tile, int KB, int64_t N, int tiles_k,
                                                   int8_t *__restrict__ out, int64_t ld_qs,
                                                   uint16_t *__restrict__ dT, int64_t ldT) {
    const int64_t tile = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / WAVE;
    if (tile >= n_tile) return;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int64_t n = tile / tiles_k * 16 + c;
    const int tk = (int)(tile % tiles_k);
    if (4 * tk + g < KB)  // (the position of column n's scale in a dT row: WeightView)
        dT[(4 * tk + g) * ldT + ((n & ~(int64_t)63) | ((n & 31) << 1) | ((n >> 5) & 1))] =
            n < N ? d[tile * 64 + lane] : (uint16_t)0;
    if (n - c >= N) return;  // (uniform)
    const v4u w = *reinterpret_cast<const v4u *>(qs + tile * 1024 + lane * 16);
    uint32_t o[4][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        // a nibble v of two's complement: (v ^ 8) - 8 in each byte, borrows kept apart
        const uint32_t lo = (w[j] & 0x0f0f0f0fu) ^ 0x08080808u, hi = ((w[j] >> 4) & 0x0f0f0f0fu) ^ 0x08080808u;
        o[j][0] = ((lo | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
        o[j][1] = ((hi | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        // lanes 0 - 31: 16 (g & 1) .. + 7 of block 2 h, and its next 8 from the lane 32 on; 32 - 63: of 2 h + 1
        const auto p0 = __builtin_amdgcn_permlane32_swap(o[2 * h][0], o[2 * h + 1][0], false, false);
        const auto p1 = __builtin_amdgcn_permlane32_swap(o[2 * h][1], o[2 * h + 1][1], false, false);
        const int kb = 4 * tk + 2 * h + (g >> 1);
        if (n < N && kb < KB)
            *reinterpret_cast<uint4 *>(out + n * ld_qs + (int64_t)kb * QK + 16 * (g & 1)) =
                make_uint4(p0[0], p1[0], p0[1], p1[1]);
    }
}
hipError_t launch_expand_q4(const Q4View &w, const WeightView &dst, hipStream_t stream) {
    const int64_t n = dst.ldT / 16 * w.tiles_k();
    hipLaunchKernelGGL(k_expand_q4, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, stream, w.qs, w.d, n,
                       (int)(w.K / QK), w.N, (int)w.tiles_k(), const_cast<int8_t *>(dst.qs), dst.ld_qs,
                       const_cast<uint16_t *>(dst.dT), dst.ldT);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Products of few rows: the weight is read as it lies.
//
// v_mfma_i32_16x16x32_i8 takes a block of 32 values at 16 columns (A) and 16
// rows (B) and leaves lane l columns 4 g + i (g = l / 16) of row l % 16.
//  * A: a nibble in the high half of a byte is 16 (v - 8) as int8, so two
//    operations make 8 operand bytes of a word: w << 4 and w, both
//    & 0xf0f0f0f0; the sums carry the 16 to the end.
//  * B: a lane loads 16 bytes, half a block: lanes 0 - 31 of the tile's even
//    block, 32 - 63 of its odd one; v_permlane32_swap gives every lane 8 bytes
//    of both, those from 16 (g & 1) + 8 (g >> 1) on.
//  * the blocks' scales d_w d_x by v_mfma_f32_16x16x16_f16: lane group g holds
//    block g's d_w and d_x in the first of its four slots of k, and A is zeroed
//    but for the block wanted: one exact product per output.
// So acc = fmaf((float)I, d_w d_x, acc) is 8 VALU operations on 4 outputs, and a
// tile's 1,152 bytes of weight come with 5 load instructions.  What bounds it:
//  * one group of 16 rows: the weight's bytes, once the loads' lanes (64 bytes a
//    clock and CU) are few.  With the scales multiplied on the VALU and loaded
//    as each lane needs them there were 11 loads a tile, and 1 x 1152 x 256000
//    took 53 us against 34.5 (4.8 TB/s, a copy's rate).
//  * more rows: the L1.  Lanes next to each other that load from different rows
//    are a cache access each (counted: 233 a wave and tile, the L1 busy 70 % of
//    the time); QUAD has four lanes load 64 bytes of a row and exchanges them
//    through LDS: 64 x 4096 x 14336 31 -> 25 us.  (32 rows a wave on the 32 x 32
//    MFMAs, half the instructions, took as long as the form without QUAD.)
//  * loads of the next tiles ahead of a tile's products: no faster, the waves of
//    the other workgroups on a CU cover each other's.
//
// A wave takes 16 rows and NT groups of 16 columns over a range of K, wk waves
// of a workgroup share their columns' K and join in LDS in order.  Further rows
// are further workgroups, next to each other on one XCD, so that the weight
// comes out of its L2 again (more rows a wave: slower at every size up to 64).
// ---------------------------------------------------------------------------
constexpr int Q4_NW = 8, Q4_NT = Q4_NW * WAVE;

struct Q4Grid {
    int wk, lwk;  // waves along K (a power of two) and its logarithm
    int tiles_k, KB, M, N, row_groups;
};

// QUAD: the activation loaded four lanes a row.
template <int NT, bool QUAD>
__global__ __launch_bounds__(Q4_NT) void k_mul_mat_q4(const uint8_t *__restrict__ wq, const uint16_t *__restrict__ wd,
                                                      Q4Grid G, const int8_t *__restrict__ xq,
                                                      const uint32_t *__restrict__ xds, float *y, int64_t ldy,
                                                      EpiParams epi) {
    constexpr int COLS = NT * 16, P = COLS + 4;
    __shared__ __align__(16) float part[Q4_NW][16][P];  // [wave][row][column]
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = wave & (G.wk - 1), wn = wave >> G.lwk;  // this wave's part of K, column group
    const int groups = Q4_NW >> G.lwk;                     // column groups of the workgroup
    const int id = xcd_linear(blockIdx.x, gridDim.x), col = id / G.row_groups;
    const int m0 = (id - col * G.row_groups) * 16, tn0 = (col * groups + wn) * NT;
    const int tiles_n = (G.N + 15) / 16, per = (G.tiles_k + G.wk - 1) >> G.lwk;
    const int k0 = wk * per, k1 = min(k0 + per, G.tiles_k);

    // the activation as it is loaded: row lr, piece lg of 64 bytes
    const int lr = QUAD ? lane >> 2 : r, lg = QUAD ? lane & 3 : g;
    const int64_t m = min(m0 + lr, G.M - 1);  // (rows past M: computed, not stored)
    const int8_t *xr = xq + m * G.KB * QK + 16 * (lg & 1);
    const uint32_t *dr = xds + m * G.KB;
    const uint8_t *wp[NT];
    const uint16_t *dp[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) {
        const int64_t t = (int64_t)min(tn0 + b, tiles_n - 1) * G.tiles_k;
        wp[b] = wq + t * 1024 + lane * 16;
        dp[b] = wd + t * 64 + lane;
    }
    v4f acc[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b) acc[b] = v4f{0, 0, 0, 0};

    for (int t = k0; t < k1; ++t) {
        v4u w[NT], x[2];
        uint32_t d[NT];
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            w[b] = *reinterpret_cast<const v4u *>(wp[b] + (int64_t)t * 1024);
            d[b] = dp[b][(int64_t)t * 64];
        }
        // blocks past K: the last one again, against zero nibbles and scales
        const int kb = 4 * t + (lg >> 1), last = G.KB - 1;
        x[0] = *reinterpret_cast<const v4u *>(xr + min(kb, last) * QK);
        x[1] = *reinterpret_cast<const v4u *>(xr + min(kb + 2, last) * QK);
        uint32_t dx0 = dr[min(4 * t + lg, last)] & 0xffffu;
        if constexpr (QUAD) {  // row r, piece g to lane 16 g + r
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c) x[h][c] = __shfl(x[h][c], 4 * r + g);
            dx0 = __shfl(dx0, 4 * r + g);
        }
        const v2i dx = {(int)dx0, 0};
        // x[h]: 16 bytes of block 2 h + (g >> 1) -> xb[j]: 8 of block j
        v2i xb[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const auto p = __builtin_amdgcn_permlane32_swap(x[h][c], x[h][c + 2], false, false);
                xb[2 * h][c] = (int)p[0];
                xb[2 * h + 1][c] = (int)p[1];
            }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int b = 0; b < NT; ++b) {
                const v2i wv = {(int)((w[b][j] << 4) & 0xf0f0f0f0u), (int)(w[b][j] & 0xf0f0f0f0u)};
                const v2i dw = {g == j ? (int)d[b] : 0, 0};
                const v4i I = __builtin_amdgcn_mfma_i32_16x16x32_i8(
                    __builtin_bit_cast(long, wv), __builtin_bit_cast(long, xb[j]), v4i{0, 0, 0, 0}, 0, 0, 0);
                const v4f s = __builtin_amdgcn_mfma_f32_16x16x16f16(
                    __builtin_bit_cast(v4h, dw), __builtin_bit_cast(v4h, dx), v4f{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][i] = fmaf((float)I[i], s[i], acc[b][i]);
            }
    }

#pragma unroll
    for (int b = 0; b < NT; ++b) *reinterpret_cast<v4f *>(&part[wave][r][16 * b + 4 * g]) = acc[b] * 0.0625f;
    __syncthreads();
    const int cols = COLS * groups, rows = min(16, G.M - m0);
    for (int i = tid; i < rows * cols; i += Q4_NT) {
        const int row = i / cols, c = i - row * cols, grp = c / COLS;
        const int64_t mr = m0 + row, n = (int64_t)col * cols + c;
        if (n >= G.N) continue;
        float v = part[grp << G.lwk][row][c % COLS];
        for (int k = 1; k < G.wk; ++k) v = v + part[(grp << G.lwk) + k][row][c % COLS];
        if (epi.kind != EPI_NONE) v = v + epi.bias[n];
        if (epi.kind == EPI_BIAS_GELU) v = gelu_tanh(v);
        if (epi.kind == EPI_BIAS_RESID)
            v = v + epi.resid[(epi.resid_rows > 0 ? mr % epi.resid_rows : mr) * epi.ld_resid + n];
        y[mr * ldy + n] = v;
    }
}

hipError_t launch_mul_mat_q4(const Q4View &w, const int8_t *xq, const uint32_t *xds, int64_t M, float *y,
                             int64_t ldy, const EpiParams &epi, hipStream_t stream) {
    // Parts of K: until the column groups' waves are 14 a CU (4096 x 14336, one
    // row: 10.5 us in 8 parts, 10.1 in 4, 10.4 in 2, 17 in 1).  From the weight's
    // shape alone, so that a row's sums are grouped the same whatever M is.
    int wk = 1, lwk = 0;
    for (; wk < Q4_NW && wk < w.tiles_k() && w.tiles_n() * wk < 3584; ++lwk) wk *= 2;
    const int64_t rg = (M + 15) / 16;
    // The rows four lanes a row and exchanged, from 5 rows on: 16 x 4096 x 14336
    // 9.7 us (a lane a row 15.1), 8 x 4096 x 4096 4.8 (4.9), 4 x 11040 x 1152 7.7
    // (7.3).  Two column groups a wave where that leaves a workgroup for half of
    // the CUs, one read of the rows for both: 1 x 1152 x 256000 34.5 us (one group
    // 36.8), 4 x 4096 x 4096 5.1 (4.0); with the exchange only past two groups of
    // rows: 64 x 4096 x 4096 8.7 (9.5), 16 x 4096 x 14336 11.5 (9.7).
    const bool quad = M > 4, two = w.tiles_n() * rg * wk / Q4_NW > 256 && (!quad || M > 32);
    const int nt = two ? 2 : 1;
    const int64_t per_wg = (int64_t)(Q4_NW / wk) * nt;
    const Q4Grid G{wk, lwk, (int)w.tiles_k(), (int)(w.K / QK), (int)M, (int)w.N, (int)rg};
    auto kern = two ? (quad ? k_mul_mat_q4<2, true> : k_mul_mat_q4<2, false>)
                    : (quad ? k_mul_mat_q4<1, true> : k_mul_mat_q4<1, false>);
    hipLaunchKernelGGL(kern, dim3((unsigned)((w.tiles_n() + per_wg - 1) / per_wg * rg)), dim3(Q4_NT), 0, stream, w.qs,
                       w.d, G, xq, xds, y, ldy, epi);
    return hipGetLastError();
}

}  // namespace s2x
