// s2x_norm.hip -- residual addition, RMS norm and Q8_1 quantization in one pass.
//
//   h = x + resid,   y = (h * inv) * w,   inv = 1 / sqrt(mean(h^2) + eps)
//
// A row lies in the registers of its waves, 8 columns a lane and piece, from its
// load to its last store: each input is read once and each output written once.
// Bound by the bytes: 8,191 rows of 4,096, all bf16, 52 us = 5.2 TB/s, what a large
// copy reaches; 8,191 of 2,048 in f32 to Q8_1 41 us = 5.3; one row of 1,152 3.2 us, an
// empty launch about 2.  Rows of more than 16,384 columns, 32 a lane, spill: 500 of 32,768
// f32 76 us = 2.8.
// The mean is a sum in f64 (a row's f32 sum would be off by some 2^-21, and
// overflow from |h| = 2^64 on), inv is rounded once to f32.  A Q8_1 block is a
// quad's 32 columns.
#include "s2x_device.h"
#include "s2x_search.h"

namespace s2x {

// 8 elements at any address that their type allows (the vector memory path takes
// 16-byte accesses at any byte)
template <typename T> struct V8;
template <> struct V8<float> {
    typedef float vec __attribute__((ext_vector_type(8), aligned(4)));
};
template <> struct V8<_Float16> {
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
};
template <> struct V8<__bf16> {
    typedef __bf16 vec __attribute__((ext_vector_type(8), aligned(2)));
};

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T *p, int c, int H) {
    if (c + 8 <= H) {
        const auto t = *reinterpret_cast<const typename V8<T>::vec *>(p + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < H ? (float)p[c + i] : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8], int c, int H) {
    if (c + 8 <= H) {
        typename V8<T>::vec t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (T)f32_materialize(v[i]);
        *reinterpret_cast<typename V8<T>::vec *>(p + c) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c + i < H) p[c + i] = (T)f32_materialize(v[i]);
    }
}

// Q8_1 of a quad's 32 values, the bits of s2x_quantize_q8_1 (as in k_layernorm:
// amax on the bit patterns, the short division where it is exact)
__device__ __forceinline__ void quantize8(const AddRmsNorm &p, int64_t row, const float (&v)[8], int c) {
    uint32_t ab = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) ab = max(ab, __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu);
    ab = max(ab, (uint32_t)dpp_i<0xb1>((int)ab));
    ab = max(ab, (uint32_t)dpp_i<0x4e>((int)ab));
    float a = __builtin_bit_cast(float, ab), d, inv;
    int q[8];
    if (__builtin_amdgcn_ballot_w64(!q8_scales_ok(a)) == 0) {
        q8_scales(a, d, inv);
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = q8_round_fast(v[i], inv);
    } else {
        a = 0.0f;  // (a NaN is passed over)
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(v[i]));
        a = fmaxf(a, dpp_f<0xb1>(a));
        a = fmaxf(a, dpp_f<0x4e>(a));
        d = a / 127.0f;
        inv = a != 0.0f ? 127.0f / a : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = q8_round(v[i], inv);
    }
    int s = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = s + (int8_t)q[i];
    s = s + dpp_i<0xb1>(s);
    s = s + dpp_i<0x4e>(s);
    *reinterpret_cast<uint2 *>(p.qs + row * p.K_pad + c) =
        make_uint2(pack4_i8(q[0], q[1], q[2], q[3]), pack4_i8(q[4], q[5], q[6], q[7]));
    if ((threadIdx.x & 3) == 0)
        p.ds[row * (p.K_pad / QK) + c / QK] =
            (uint32_t)f32_to_f16_bits(d) | ((uint32_t)f32_to_f16_bits((float)s * d) << 16);
}

// NW waves a row, NV pieces of 8 columns a lane.  One wave a row: four rows a
// workgroup; LN < 64: LN lanes a row.
template <typename TX, typename TR, int NV, int NW, int LN = WAVE>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * WAVE) void k_add_rmsnorm(AddRmsNorm p) {
    __shared__ double part[2][NW];
    constexpr int LANES = NW * LN, ROWS = NW == 1 ? 256 / LN : 1;
    const int lane = NW == 1 ? threadIdx.x % LN : threadIdx.x, wave = threadIdx.x >> 6;
    const int H = p.H, cols = p.qs ? p.K_pad : H;
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * ROWS + (NW == 1 ? threadIdx.x / LN : 0); row < p.M; row += step, turn ^= 1) {
        float h[NV][8], w[NV][8];
        const TX *x = (const TX *)p.x + row * p.ld_x;
        const TR *r = (const TR *)p.resid + row * p.ld_resid;
#pragma unroll
        for (int n = 0; n < NV; ++n) load8(h[n], x, 8 * (n * LANES + lane), H);
        if (p.resid) {
            float t[NV][8];
#pragma unroll
            for (int n = 0; n < NV; ++n) load8(t[n], r, 8 * (n * LANES + lane), H);
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) h[n][i] = h[n][i] + t[n][i];
        }
        double s = 0.0;
#pragma unroll
        for (int n = 0; n < NV; ++n)
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fma((double)h[n][i], (double)h[n][i], s);
        if (p.w) {
#pragma unroll
            for (int n = 0; n < NV; ++n) load8(w[n], p.w, 8 * (n * LANES + lane), H);
        }
        s = LN == WAVE ? wave_dsum(s) : group_dsum<LN>(s);
        if constexpr (NW > 1) {
            if ((threadIdx.x & 63) == 0) part[turn][wave] = s;
            __syncthreads();  // (the other half is written next: one barrier a row)
            s = part[turn][0];
#pragma unroll
            for (int i = 1; i < NW; ++i) s = s + part[turn][i];
        }
        const float inv = (float)(1.0 / sqrt(s / (double)H + (double)p.eps));
        if (p.h_out) {
            TR *ho = (TR *)p.h_out + row * p.ld_h;
#pragma unroll
            for (int n = 0; n < NV; ++n) store8(ho, h[n], 8 * (n * LANES + lane), H);
        }
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int c = 8 * (n * LANES + lane);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[n][i] = h[n][i] * inv;
                if (p.w) h[n][i] = h[n][i] * w[n][i];
                if (c + i >= H) h[n][i] = 0.0f;  // (zeros past H also where inv is no number)
            }
            if (p.y) {
                if (p.y_type == TY_F32) store8((float *)p.y + row * p.ld_y, h[n], c, H);
                else if (p.y_type == TY_F16) store8((_Float16 *)p.y + row * p.ld_y, h[n], c, H);
                else store8((__bf16 *)p.y + row * p.ld_y, h[n], c, H);
            }
            if (p.qs && c < cols) quantize8(p, row, h[n], c);  // (quads leave together)
        }
    }
}

template <typename TX, typename TR, int NV, int NW, int LN = WAVE>
static hipError_t run_rms(const AddRmsNorm &p, hipStream_t stream) {
    constexpr int ROWS = 256 / LN;
    const int64_t wgs = NW == 1 ? (p.M + ROWS - 1) / ROWS : p.M, most = 1 << 20;
    auto kern = k_add_rmsnorm<TX, TR, NV, NW, LN>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(wgs < most ? wgs : most)), dim3(NW == 1 ? 256 : NW * WAVE), 0, stream, p);
    return hipGetLastError();
}
// 8 columns a lane up to 4,096, in as much of a wave or as many as that takes, 16 above:
// workgroups of which several fit a CU, so that some load while others are at their
// barrier.  bf16, 8,191 rows of 4,096: 8 waves of 8 columns 57.2 us, 4 of 16 58.8; 4,000
// of 5,120: 8 of 16 45.0, 16 of 8 55.7, 4 of 32 66.7; 1,000 of 16,384: 16 of 16 28.2, 8 of 32 32.2; 30,000 of 480: a wave 23.6, two 34.6;
// 60,000 of 256: half a wave 21.9, a wave 31.8; 100,000 of 128: a quarter 19.2, a wave 48.1;
// 300,000 of 64: an eighth 32.2, a wave 147.
template <typename TX, typename TR>
static hipError_t run_rms_h(const AddRmsNorm &p, hipStream_t stream) {
    const int cols = p.qs ? p.K_pad : p.H;
    if (cols <= 64) return run_rms<TX, TR, 1, 1, 8>(p, stream);
    if (cols <= 128) return run_rms<TX, TR, 1, 1, 16>(p, stream);
    if (cols <= 256) return run_rms<TX, TR, 1, 1, 32>(p, stream);
    if (cols <= 512) return run_rms<TX, TR, 1, 1>(p, stream);
    if (cols <= 1024) return run_rms<TX, TR, 1, 2>(p, stream);
    if (cols <= 2048) return run_rms<TX, TR, 1, 4>(p, stream);
    if (cols <= 4096) return run_rms<TX, TR, 1, 8>(p, stream);
    if (cols <= 8192) return run_rms<TX, TR, 2, 8>(p, stream);
    if (cols <= 16384) return run_rms<TX, TR, 2, 16>(p, stream);
    return run_rms<TX, TR, 4, 16>(p, stream);
}
hipError_t launch_add_rmsnorm(const AddRmsNorm &p, hipStream_t stream) {
    if (p.x_type == TY_F32) return run_rms_h<float, float>(p, stream);
    if (p.x_type == TY_F16)
        return p.r_type == TY_F32 ? run_rms_h<_Float16, float>(p, stream) : run_rms_h<_Float16, _Float16>(p, stream);
    return p.r_type == TY_F32 ? run_rms_h<__bf16, float>(p, stream) : run_rms_h<__bf16, __bf16>(p, stream);
}

}  // namespace s2x
