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
        const uint8_t *b = raw + (n * KB + kb) * 18 + 2 + (g & 1) * 8;  // bytes of values 8 (g & 1) ..
        for (int k = 0; k < 4; ++k) {
            const uint32_t lo = g < 2 ? b[k] & 15 : b[k] >> 4, hi = g < 2 ? b[4 + k] & 15 : b[4 + k] >> 4;
            w[j] |= ((lo | hi << 4) ^ 0x88) << (8 * k);
        }
    }
    reinterpret_cast<uint4 *>(qs)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    // scale l of the tile: column 4 (l / 16) + l % 4, block l % 16 / 4
    const int64_t ns = tn * 16 + 4 * g + l % 4, kb = tk * 4 + l % 16 / 4;
    uint16_t v = 0;
    if (ns < N && kb < KB) {
        const uint8_t *b = raw + (ns * KB + kb) * 18;
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

__global__ __launch_bounds__(256) void k_expand_q4(const uint8_t *__restrict__ qs, const uint16_t *__restrict__ d,
                                                   int64_t n_block, int64_t KB, int64_t N, int64_t tiles_k,
                                                   int8_t *__restrict__ out, int64_t ld_qs,
                                                   uint16_t *__restrict__ dT, int64_t ldT) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n_block) return;
    const int64_t n = i / KB, kb = i - n * KB;
    const int64_t tile = n / 16 * tiles_k + kb / 4;
    const int c = (int)(n % 16), j = (int)(kb % 4);
    uint32_t o[8];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(qs + tile * 1024 + (16 * g + c) * 16 + 4 * j);
        // a nibble v of two's complement: (v ^ 8) - 8 in each byte, borrows kept apart
        const uint32_t lo = (w & 0x0f0f0f0fu) ^ 0x08080808u, hi = ((w >> 4) & 0x0f0f0f0fu) ^ 0x08080808u;
        o[2 * g] = ((lo | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
        o[2 * g + 1] = ((hi | 0x80808080u) - 0x08080808u) ^ 0x80808080u;
    }
    uint4 *dst = reinterpret_cast<uint4 *>(out + n * ld_qs + kb * QK);
    dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
    dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    // (the position of column n's scale in a dT row: WeightView)
    dT[kb * ldT + ((n & ~(int64_t)63) | ((n & 31) << 1) | ((n >> 5) & 1))] = d[tile * 64 + c / 4 * 16 + j * 4 + c % 4];
}
hipError_t launch_expand_q4(const Q4View &w, const WeightView &dst, hipStream_t stream) {
    const int64_t nb = w.N * (w.K / QK);
    uint16_t *dT = const_cast<uint16_t *>(dst.dT);
    hipError_t e = launch_fill_zero(dT, (size_t)(w.K / QK * dst.ldT) * 2, stream);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_expand_q4, dim3((unsigned)((nb + 255) / 256)), dim3(256), 0, stream, w.qs, w.d, nb,
                       w.K / QK, w.N, w.tiles_k(), const_cast<int8_t *>(dst.qs), dst.ld_qs, dT, dst.ldT);
    return hipGetLastError();
}

// One thread per output, blocks in order.
__global__ __launch_bounds__(256) void k_mul_mat_q4(Q4View w, int64_t tiles_k, const int8_t *__restrict__ xq,
                                                    const uint32_t *__restrict__ xds, int64_t M, float *y,
                                                    int64_t ldy, EpiParams epi) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= M * w.N) return;
    const int64_t m = i / w.N, n = i - m * w.N, KB = w.K / QK;
    const int c = (int)(n % 16);
    float acc = 0.0f;
    for (int64_t kb = 0; kb < KB; ++kb) {
        const int64_t tile = n / 16 * tiles_k + kb / 4;
        const int j = (int)(kb % 4);
        int dot = 0;
        for (int g = 0; g < 4; ++g) {
            const uint8_t *b = w.qs + tile * 1024 + (16 * g + c) * 16 + 4 * j;
            const int8_t *x = xq + m * w.K + kb * QK + 8 * g;
            for (int k = 0; k < 4; ++k)
                dot += ((int)((b[k] & 15) ^ 8) - 8) * x[k] + ((int)((b[k] >> 4) ^ 8) - 8) * x[4 + k];
        }
        const float dw = f16_bits_to_f32(w.d[tile * 64 + c / 4 * 16 + j * 4 + c % 4]);
        acc = fmaf((float)dot, dw * f16_bits_to_f32((uint16_t)(xds[m * KB + kb] & 0xffff)), acc);
    }
    if (epi.kind != EPI_NONE) acc = acc + epi.bias[n];
    if (epi.kind == EPI_BIAS_GELU) acc = gelu_tanh(acc);
    if (epi.kind == EPI_BIAS_RESID)
        acc = acc + epi.resid[(epi.resid_rows > 0 ? m % epi.resid_rows : m) * epi.ld_resid + n];
    y[m * ldy + n] = acc;
}
hipError_t launch_mul_mat_q4(const Q4View &w, const int8_t *xq, const uint32_t *xds, int64_t M, float *y,
                             int64_t ldy, const EpiParams &epi, hipStream_t stream) {
    hipLaunchKernelGGL(k_mul_mat_q4, dim3((unsigned)((M * w.N + 255) / 256)), dim3(256), 0, stream, w,
                       w.tiles_k(), xq, xds, M, y, ldy, epi);
    return hipGetLastError();
}

}  // namespace s2x
