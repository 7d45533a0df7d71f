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
//  * more rows: the L1, then the operations.  Lanes next to each other that load
//    from different rows are a cache access each (counted: 233 a wave and tile,
//    the L1 busy 70 % of the time); QUAD has four lanes load 64 bytes of a row
//    and exchanges them through LDS: 64 x 4096 x 14336 31 -> 24.6 us, and with 32
//    rows a wave (below) 19.6.
//  * loads of the next tiles ahead of a tile's products: no faster, the waves of
//    the other workgroups on a CU cover each other's.
//
// A wave takes 16 rows and NT groups of 16 columns over a range of K, wk waves
// of a workgroup share their columns' K and join in LDS in order.  Further rows
// are further workgroups, next to each other on one XCD, so that the weight
// comes out of its L2 again.
// ---------------------------------------------------------------------------
constexpr int Q4_NW = 8, Q4_NT = Q4_NW * WAVE;

struct Q4Grid {
    int wk, lwk;  // waves along K (a power of two) and its logarithm
    int tiles_k, KB, M, N, row_groups;
    int64_t resid0;  // the residual's row of row 0 (before resid_rows wraps it)
};

// The waves' sums [wave][ROWS][P] joined in the order of K, the epilogue, and out.
template <int COLS, int P, int ROWS>
__device__ __forceinline__ void q4_join(const float *part, const Q4Grid &G, int col, int m0, int groups, float *y,
                                        int64_t ldy, const EpiParams &epi) {
    const int cols = COLS * groups, rows = min(ROWS, G.M - m0);
    for (int i = threadIdx.x; i < rows * cols; i += Q4_NT) {
        const int row = i / cols, c = i - row * cols, grp = c / COLS;
        const int64_t mr = m0 + row, rr = G.resid0 + mr, n = (int64_t)col * cols + c;
        if (n >= G.N) continue;
        const float *p = part + ((grp << G.lwk) * ROWS + row) * P + c % COLS;
        float v = p[0];
        for (int k = 1; k < G.wk; ++k) v = v + p[k * ROWS * P];
        if (epi.kind != EPI_NONE) v = v + epi.bias[n];
        if (epi.kind == EPI_BIAS_GELU) v = gelu_tanh(v);
        if (epi.kind == EPI_BIAS_RESID)
            v = v + epi.resid[(epi.resid_rows > 0 ? rr % epi.resid_rows : rr) * epi.ld_resid + n];
        y[mr * ldy + n] = v;
    }
}

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
    q4_join<COLS, P, 16>(&part[0][0][0], G, col, m0, groups, y, ldy, epi);
}

// The same for 32 rows and 32 columns a wave, on the 32 x 32 MFMAs: half the
// instructions an output of the 16 x 16 ones, and the conversion of the block
// dots on the matrix pipe too.  A 32-value block is one
// v_mfma_i32_32x32x32_i8 whose accumulator begins at the bits of c0 = 1/2pi, a
// float whose ulp is 2^-26: its result read as a float is c0 + 16 I 2^-26 exactly
// (|16 I| <= 32 * 128 * 128 = 2^19 stays in c0's binade); one f16 product adds
// -c0 as three exact terms, another makes the scales d_w d_x, and the VALU is left
// with one fma an output.  The sums are those of the 16-row form times 2^-22, a
// power of two: the same bits (no term is below 2^-74 of that scale).  A tile's
// rows, 128 bytes each, go through a part of LDS that is the wave's own: loaded
// four lanes to 64 bytes of a row, read 16 bytes of a block a lane.  (64 columns a
// wave: 64 x 4096 x 14336 18.6 us against 19.6, 64 x 4096 x 4096 10.8 against 8.1.)
constexpr int Q4_XROW = 32 * 128, Q4_XW = Q4_XROW + 32 * 16;  // a wave's quants and scale words in LDS

__global__ __launch_bounds__(Q4_NT) void k_mul_mat_q4_32(const uint8_t *__restrict__ wq,
                                                         const uint16_t *__restrict__ wd, Q4Grid G,
                                                         const int8_t *__restrict__ xq,
                                                         const uint32_t *__restrict__ xds, float *y, int64_t ldy,
                                                         EpiParams epi) {
    constexpr int COLS = 32, P = COLS + 4;
    // rows of the waves, then their sums [wave][32][P]
    constexpr int ROWS = Q4_NW * Q4_XW, SUMS = Q4_NW * 32 * P * 4;
    __shared__ __align__(16) uint8_t lds32[ROWS > SUMS ? ROWS : SUMS];
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wk = wave & (G.wk - 1), wn = wave >> G.lwk;
    const int groups = Q4_NW >> G.lwk;
    const int id = xcd_linear(blockIdx.x, gridDim.x), col = id / G.row_groups;
    const int m0 = (id - col * G.row_groups) * 32, tn0 = (col * groups + wn) * 2;
    const int tiles_n = (G.N + 15) / 16, per = (G.tiles_k + G.wk - 1) >> G.lwk;
    const int k0 = wk * per, k1 = min(k0 + per, G.tiles_k);

    // as loaded: rows 16 a + lane / 4, piece lane % 4 of 64 bytes
    const int8_t *xr[2];
    const uint32_t *dr[2];
    uint8_t *xl = lds32 + wave * Q4_XW;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        const int64_t m = min(m0 + 16 * a + (lane >> 2), G.M - 1);  // (rows past M: computed, not stored)
        xr[a] = xq + m * G.KB * QK + 16 * (lane & 1);
        dr[a] = xds + m * G.KB;
    }
    // piece c of row w at place c ^ (w & 7) of the row's 8: 8 lanes' reads of one
    // piece lie in 8 bank groups
    uint8_t *xs[2][2];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int w = 16 * a + (lane >> 2), c = 4 * q + (lane & 3);
            xs[a][q] = xl + w * 128 + 16 * (c ^ (w & 7));
        }
    const int64_t tile = (int64_t)min(tn0 + (r >> 4), tiles_n - 1) * G.tiles_k;
    const uint8_t *wp = wq + tile * 1024 + (16 * h + (r & 15)) * 16;  // values 16 h .. + 7 of its 4 blocks; + 512: the next 8
    const uint16_t *dp = wd + tile * 64 + 16 * h + (r & 15);          // block h; + 32: block 2 + h
    v16f acc = {};
    // f16 (-0.125, -1119/256, -387/8192, 0) x (1, 2^-7, 2^-13, 0) = -c0, lanes
    // 32 .. 63 zero
    const v2i cA = {h ? 0 : (int)0xC45FB000u, h ? 0 : 0xAA0C};
    const v2i cB = {h ? 0 : 0x20003C00, h ? 0 : 0x0800};

    for (int t = k0; t < k1; ++t) {
        v4u w[2], xg[2][2];
        uint32_t d[2], dg[2];
        const int kb = 4 * t + ((lane & 3) >> 1), last = G.KB - 1;  // (blocks past K: the last, against zeros)
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            xg[a][0] = *reinterpret_cast<const v4u *>(xr[a] + min(kb, last) * QK);
            xg[a][1] = *reinterpret_cast<const v4u *>(xr[a] + min(kb + 2, last) * QK);
            dg[a] = dr[a][min(4 * t + (lane & 3), last)] & 0xffffu;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            w[j] = *reinterpret_cast<const v4u *>(wp + (int64_t)t * 1024 + 512 * j);
            d[j] = dp[(int64_t)t * 64 + 32 * j];
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            *reinterpret_cast<v4u *>(xs[a][0]) = xg[a][0];
            *reinterpret_cast<v4u *>(xs[a][1]) = xg[a][1];
            reinterpret_cast<uint32_t *>(xl + Q4_XROW)[64 * a + lane] = dg[a];  // [row][block]
        }
        __builtin_amdgcn_wave_barrier();
        v4i x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            x[j] = *reinterpret_cast<const v4i *>(xl + r * 128 + 16 * ((2 * j + h) ^ (r & 7)));
        v2i dx[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            dx[j] = v2i{(int)reinterpret_cast<const uint32_t *>(xl + Q4_XROW)[4 * r + 2 * j + h], 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __builtin_amdgcn_sched_barrier(0);  // (blocks apart: 121 registers, 4 waves a SIMD; mixed 134)
            const v4i wv = {(int)((w[0][j] << 4) & 0xf0f0f0f0u), (int)(w[0][j] & 0xf0f0f0f0u),
                            (int)((w[1][j] << 4) & 0xf0f0f0f0u), (int)(w[1][j] & 0xf0f0f0f0u)};
            const v2i dw = {h == (j & 1) ? (int)d[j / 2] : 0, 0};
            const v16i magic = 0x3E22F983;
            v16f I = __builtin_bit_cast(v16f, __builtin_amdgcn_mfma_i32_32x32x32_i8(wv, x[j], magic, 0, 0, 0));
            I = __builtin_amdgcn_mfma_f32_32x32x8f16(__builtin_bit_cast(v4h, cA), __builtin_bit_cast(v4h, cB), I, 0, 0, 0);
            const v16f s = __builtin_amdgcn_mfma_f32_32x32x8f16(__builtin_bit_cast(v4h, dw), __builtin_bit_cast(v4h, dx[j / 2]),
                                                                v16f{}, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[i] = fmaf(I[i], s[i], acc[i]);
        }
    }

    // acc[4 q + i]: column 8 q + 4 h + i of row r
    float *part = reinterpret_cast<float *>(lds32);
    float *mine = part + (wave * 32 + r) * P + 4 * h;
    __syncthreads();  // (the sums lie over the waves' rows)
#pragma unroll
    for (int q = 0; q < 4; ++q)
        *reinterpret_cast<v4f *>(mine + 8 * q) =
            v4f{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]} * 0x1p22f;
    __syncthreads();
    q4_join<COLS, P, 32>(part, G, col, m0, groups, y, ldy, epi);
}

static hipError_t run_q4(const Q4View &w, const int8_t *xq, const uint32_t *xds, int64_t M, float *y, int64_t ldy,
                         const EpiParams &epi, int64_t resid0, hipStream_t stream) {
    // Parts of K: until the column groups' waves are 14 a CU (4096 x 14336, one
    // row: 10.5 us in 8 parts, 10.1 in 4, 10.4 in 2, 17 in 1).  From the weight's
    // shape alone, so that a row's sums are grouped the same whatever M is.
    int wk = 1, lwk = 0;
    for (; wk < Q4_NW && wk < w.tiles_k() && w.tiles_n() * wk < 3584; ++lwk) wk *= 2;
    Q4Grid G{wk, lwk, (int)w.tiles_k(), (int)(w.K / QK), (int)M, (int)w.N, (int)((M + 31) / 32), resid0};
    const int groups = Q4_NW / wk;
    const auto launch = [&](auto kern, int tiles) {  // column tiles of a wave
        const int64_t per_wg = (int64_t)groups * tiles;
        hipLaunchKernelGGL(kern, dim3((unsigned)((w.tiles_n() + per_wg - 1) / per_wg * G.row_groups)), dim3(Q4_NT), 0,
                           stream, w.qs, w.d, G, xq, xds, y, ldy, epi);
        return hipGetLastError();
    };
    // 32 rows a wave past 16, where that makes 160 workgroups: 24 x 4096 x 14336
    // (224) 12.3 us, 16 rows a wave 14.7, 64 x 4096 x 14336 (448) 19.6 (24.6), 160
    // x 4320 x 1152 (180) 8.5 (9.3); 32 x 4096 x 4096 (128) 8.0 (6.1), 43 x 4320 x
    // 1152 (72) 7.3 (4.6)
    if (M > 16 && (w.tiles_n() + 1) / 2 * G.row_groups * wk / Q4_NW >= 160) return launch(k_mul_mat_q4_32, 2);
    G.row_groups = (int)((M + 15) / 16);
    // The rows four lanes a row and exchanged, from 5 rows on: 16 x 4096 x 14336
    // 9.7 us (a lane a row 15.1), 8 x 4096 x 4096 4.8 (4.9), 4 x 11040 x 1152 7.7
    // (7.3).  Below, two column groups a wave where that leaves a workgroup for
    // half of the CUs, one read of the rows for both: 1 x 1152 x 256000 34.5 us
    // (one group 36.8), 4 x 4096 x 4096 5.1 (4.0); with the exchange one group
    // is as fast or faster: 16 x 4096 x 14336 9.7 (two 11.5).
    if (M > 4) return launch(k_mul_mat_q4<1, true>, 1);
    if (w.tiles_n() * wk / Q4_NW > 256) return launch(k_mul_mat_q4<2, false>, 2);
    return launch(k_mul_mat_q4<1, false>, 1);
}

// Any M.  2,048 rows a launch: at the widest weight (2^24 columns, 2^16
// workgroups a row group of 32) that is 2^22 workgroups, 2^31 threads.
hipError_t launch_mul_mat_q4(const Q4View &w, const int8_t *xq, const uint32_t *xds, int64_t M, float *y,
                             int64_t ldy, const EpiParams &epi, hipStream_t stream) {
    hipError_t e = hipSuccess;
    for (int64_t m = 0; m < M && e == hipSuccess; m += 2048)
        e = run_q4(w, xq + m * w.K, xds + m * (w.K / QK), M - m < 2048 ? M - m : 2048, y + m * ldy, ldy, epi, m, stream);
    return e;
}

}  // namespace s2x
