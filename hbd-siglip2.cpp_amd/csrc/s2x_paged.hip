// s2x_paged.hip -- attention of one new token per sequence over a paged cache.
//
// out = sum_t softmax_t(q . k_t * scale) v_t for up to 16 query heads that
// share a key head, one pass over the keys with the running maximum and sum.
// Each key and value is read once and used for 4 R flops (R query heads a key
// head), far below the matrix pipe's rate: the bytes of the cache bound it.
//
// A wave takes tiles of 32 keys, each by itself (no barrier in the loop):
//  * S^T = K Q^T by v_mfma_f32_16x16x32: K's rows are the A operand, which a
//    lane loads straight into its registers, 16 bytes of key lane % 16; the
//    16 query heads (zeros past R) are B, loaded once.
//  * S^T leaves that product with lane l holding head l % 16 and keys 4 g + i
//    (g = l / 16) -- the layout B wants of P^T in the second product, O^T =
//    V^T P^T, if its 8 values of k are taken as keys 4 g .. 4 g + 3 of the
//    tile's two halves.  So the probabilities never cross lanes.
//  * V^T as the A operand of that order is 4 consecutive keys of one value
//    index a lane: the transposing read of LDS (ds_read_b64_tr_b16) of V's
//    rows as they lie, staged in a part of LDS that is the wave's own.
//  * The next tile's keys and values are loaded once the scores have freed
//    the registers, and the page ids of the one after.
// A workgroup's four waves join in LDS; a sequence's chunks, where there is
// more than one, in k_attn_join.
#include "s2x_decode.h"
#include "s2x_device.h"

namespace s2x {

constexpr int PA_NT = 256, PA_NW = PA_NT / WAVE;
constexpr int PA_TILE = 32;             // keys of a wave's tile
constexpr int PA_STEP = PA_NW * PA_TILE;  // ... of a workgroup's

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

template <typename T> struct Pa;
// Terms of the cache's type that a probability enters the second product as:
// f16 11 bits each, bf16 8.  f16 takes p * 2^15 (p <= 1), which keeps the
// second term's 2^-25 of the largest above the subnormal range.
template <> struct Pa<_Float16> {
    typedef v8h vec;
    static constexpr float up = 32768.0f, down = 1.0f / 32768.0f;
    static __device__ __forceinline__ v4f mfma(vec a, vec b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Pa<__bf16> {
    typedef v8bf vec;
    static constexpr float up = 1.0f, down = 1.0f;
    static __device__ __forceinline__ v4f mfma(vec a, vec b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
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
    r.begin = r.first & ~(int64_t)(PA_TILE - 1);
    return r;
}

constexpr int pa_lds_bytes(int DC) {
    const int v = PA_NW * PA_TILE * DC * 64 + 64, o = PA_NW * 16 * (DC * 32 + 4) * 4;
    return v > o ? v : o;
}

// Values 4 e .. 4 e + 3 of head h: the sums over its keys by the sum of the
// exponentials (nothing seen: zeros, and lse = -inf by itself).
template <typename TC>
__device__ __forceinline__ void pa_write(const AttnPaged &p, int s, int h, int d, int e, v4f a, float M, float L) {
    typedef TC vec4 __attribute__((ext_vector_type(4)));
    const int64_t at = s * p.ld_out + (int64_t)h * d + 4 * e;
    v4f y;
    vec4 t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = L == 0.0f ? 0.0f : a[i] * Pa<TC>::down / L;
        t[i] = (TC)f32_materialize(y[i]);
    }
    if (p.out_f32) *reinterpret_cast<v4f *>((float *)p.out + at) = y;
    else *reinterpret_cast<vec4 *>((TC *)p.out + at) = t;
    if (e == 0 && p.lse) p.lse[(int64_t)s * p.n_q_head + h] = (M + log2f(L)) * 0.693147180559945309f;
}

// DC: 32-value chunks of a head; EXACT: d_head = 32 DC; NP: terms of P.
template <typename TC, int DC, bool EXACT, int NP>
__global__ __launch_bounds__(PA_NT) void k_attn_paged(AttnPaged p, int chunk, int n_split) {
    typedef typename Pa<TC>::vec vec;
    constexpr int DP = 32 * DC, DT = 2 * DC;
    __shared__ __align__(16) uint8_t lds[pa_lds_bytes(DC)];
    __shared__ float ml[PA_NW][2][16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const int split = blockIdx.x, s = blockIdx.z, d = EXACT ? DP : p.kv.d_head, nch = d / 8;
    const int group = p.n_q_head / p.kv.n_head, parts = (group + 15) / 16;
    const int hk = blockIdx.y / parts, h0 = hk * group + (blockIdx.y - hk * parts) * 16;
    const int R = min(16, (hk + 1) * group - h0);
    const PaRange kr = pa_range(p, s);
    const int64_t start = kr.begin + (int64_t)split * chunk, end = min(start + chunk, kr.len);
    if (start >= end && (n_split > 1)) return;  // (uniform; the only chunk writes zeros)

    const TC *kp = (const TC *)p.kv.k + hk * p.kv.ld_head, *vp = (const TC *)p.kv.v + hk * p.kv.ld_head;
    const int32_t *row = p.table + s * p.ld_table;
    const uint32_t pmask = (1u << p.kv.page_shift) - 1, ldp = (uint32_t)p.kv.ld_page, ldt = (uint32_t)p.kv.ld_tok;
    TC *vl = reinterpret_cast<TC *>(lds) + wave * PA_TILE * d;

    vec q[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) {
        q[c] = vec{};
        if (r < R && (EXACT || 32 * c + 8 * g < d))
            q[c] = *reinterpret_cast<const vec *>((const TC *)p.q + s * p.ld_q + (int64_t)(h0 + r) * d + 32 * c + 8 * g);
    }

    // page of key t0 + lane % 32, -1 unseen
    auto page_of = [&](int64_t t0) {
        const int64_t t = t0 + (lane & 31);
        int32_t id = -1;
        if (t >= kr.first && t < end) {
            id = row[t >> p.kv.page_shift];
            if (id >= p.kv.n_pages) id = -1;
        }
        return id;
    };
    vec k[2][DC], v[DT];
    const uint32_t magic = (65536u + nch - 1) / nch;  // f / nch for f < 1,024
    uint32_t seen = 0;
    auto load = [&](int64_t t0, int32_t id) {
        seen = (uint32_t)__builtin_amdgcn_ballot_w64(id >= 0);
        const bool all = EXACT && seen == ~0u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int key = 16 * j + r;
            const uint32_t pid = (uint32_t)__shfl(id, key);
            const TC *src = kp + ((uint64_t)pid * ldp + (((uint32_t)t0 + key) & pmask) * (uint64_t)ldt + 8 * g);
            const bool ok = all || (int32_t)pid >= 0;
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                k[j][c] = vec{};
                if (ok && (EXACT || 32 * c + 8 * g < d)) k[j][c] = *reinterpret_cast<const vec *>(src + 32 * c);
            }
        }
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            const uint32_t f = i * WAVE + lane, key = EXACT ? f / (DP / 8) : f * magic >> 16;
            const uint32_t pid = (uint32_t)__shfl(id, (int)(key & 31));
            const TC *src = vp + ((uint64_t)pid * ldp + (((uint32_t)t0 + key) & pmask) * (uint64_t)ldt + 8 * (f - key * nch));
            v[i] = vec{};
            if (all || (key < PA_TILE && (int32_t)pid >= 0)) v[i] = *reinterpret_cast<const vec *>(src);
        }
    };

    float m = -INFINITY, l = 0.0f;
    v4f o[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = v4f{0, 0, 0, 0};
    const float sc = p.scale * 1.44269504088896341f;  // log2(e)

    int64_t t0 = start + wave * PA_TILE;
    int32_t id_next = -1;
    if (t0 < end) {
        load(t0, page_of(t0));
        id_next = page_of(t0 + PA_STEP);
    }
    for (; t0 < end; t0 += PA_STEP) {
        const uint32_t mask = seen;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
            if (EXACT || i * WAVE + lane < PA_TILE * nch)
                *reinterpret_cast<vec *>(vl + (i * WAVE + lane) * 8) = v[i];
        }
        v4f st[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            st[j] = v4f{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < DC; ++c) st[j] = Pa<TC>::mfma(k[j][c], q[c], st[j]);
        }
        if (t0 + PA_STEP < end) {
            load(t0 + PA_STEP, id_next);
            id_next = page_of(t0 + 2 * PA_STEP);
        }
        // the softmax of head r over keys 4 g + i, 16 + 4 g + i
        float mt = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                st[j][i] = st[j][i] * sc;
                if (mask != ~0u && !(mask >> (16 * j + 4 * g + i) & 1)) st[j][i] = -INFINITY;
                mt = fmaxf(mt, st[j][i]);
            }
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float mn = fmaxf(m, mt), base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l = l * alpha;
        vec pt[NP];
#pragma unroll
        for (int j = 0; j < 2; ++j)
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
            v8s a;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                TC *src = vl + (16 * j + 4 * g + (r >> 2)) * d + 16 * i + (r & 3) * 4;
                const v4s t = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) v4s *)src);
#pragma unroll
                for (int n = 0; n < 4; ++n) a[4 * j + n] = t[n];
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) o[i] = Pa<TC>::mfma(__builtin_bit_cast(vec, a), pt[n], o[i]);
        }
        __builtin_amdgcn_wave_barrier();
    }

    // join the waves: o[i] is values 16 i + 4 g .. + 3 of head r
    l = l + __shfl_xor(l, 16);
    l = l + __shfl_xor(l, 32);
    float *ol = reinterpret_cast<float *>(lds);  // [wave][head][DP + 4]
    __syncthreads();
    if (r < R) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
            *reinterpret_cast<v4f *>(ol + (wave * 16 + r) * (DP + 4) + 16 * i + 4 * g) = o[i];
        if (g == 0) {
            ml[wave][0][r] = m;
            ml[wave][1][r] = l;
        }
    }
    __syncthreads();
    for (int i = tid; i < R * nch * 2; i += PA_NT) {
        const int h = i / (nch * 2), e = i - h * (nch * 2);
        float M = ml[0][0][h];
#pragma unroll
        for (int w = 1; w < PA_NW; ++w) M = fmaxf(M, ml[w][0][h]);
        const float base = M == -INFINITY ? 0.0f : M;
        v4f a = {0, 0, 0, 0};
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < PA_NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[w][0][h] - base);
            L = fmaf(ml[w][1][h], f, L);
            const v4f x = *reinterpret_cast<const v4f *>(ol + (w * 16 + h) * (DP + 4) + 4 * e);
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
            pa_write<TC>(p, s, h0 + h, d, e, a, M, L);
        }
    }
}

// Chunks of a sequence joined, one workgroup per sequence and query head: the
// chunks in PA_NT / (d / 4) groups, a thread 4 values of one.
template <typename TC>
__global__ __launch_bounds__(PA_NT) void k_attn_join(AttnPaged p, int chunk, int n_split) {
    __shared__ __align__(16) float part[PA_NT * 4];
    __shared__ float red[PA_NW], lsum[PA_NT];
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, d = p.kv.d_head, nq = d / 4;
    const PaRange kr = pa_range(p, s);
    const int n = kr.len > kr.begin ? (int)((kr.len - kr.begin + chunk - 1) / chunk) : 0;
    const int64_t at = ((int64_t)s * p.n_q_head + h) * n_split;
    const float *ws = (const float *)p.ws;
    const float2 *mlp = reinterpret_cast<const float2 *>(ws + (int64_t)p.n_seq * p.n_q_head * n_split * d) + at;
    float M = -INFINITY;
    for (int i = tid; i < n; i += PA_NT) M = fmaxf(M, mlp[i].x);
    M = group_max<64>(M);
    if ((tid & 63) == 0) red[tid >> 6] = M;
    __syncthreads();
    M = red[0];
#pragma unroll
    for (int w = 1; w < PA_NW; ++w) M = fmaxf(M, red[w]);
    const float base = M == -INFINITY ? 0.0f : M;
    const int groups = PA_NT / nq, grp = tid / nq, e = tid - grp * nq;
    v4f a = {0, 0, 0, 0};
    float L = 0.0f;
    if (grp < groups) {
        for (int i = grp; i < n; i += groups) {
            const float2 t = mlp[i];
            const float f = __builtin_amdgcn_exp2f(t.x - base);
            L = fmaf(t.y, f, L);
            const v4f x = reinterpret_cast<const v4f *>(ws)[(at + i) * nq + e];
#pragma unroll
            for (int c = 0; c < 4; ++c) a[c] = fmaf(x[c], f, a[c]);
        }
        reinterpret_cast<v4f *>(part)[tid] = a;
        lsum[tid] = L;
    }
    __syncthreads();
    if (grp == 0) {
        for (int i = 1; i < groups; ++i) {
            L = L + lsum[i * nq + e];
            a = a + reinterpret_cast<const v4f *>(part)[i * nq + e];
        }
        pa_write<TC>(p, s, h, d, e, a, M, L);
    }
}

// Chunk length and their number for a launch: about 4 workgroups a CU where
// the lengths allow it, whole steps of a workgroup's four waves.
static void pa_plan(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head, int &chunk, int &n_split) {
    const int64_t units = n_seq * n_kv_head * ((n_q_head / n_kv_head + 15) / 16);
    const int64_t span = max_len + PA_TILE;  // (the first tile may begin before a window)
    int64_t c = (span * units + 1023) / 1024;
    c = (c + PA_STEP - 1) / PA_STEP * PA_STEP;
    if (c < 2 * PA_STEP) c = 2 * PA_STEP;
    if (c > 4096) c = 4096;
    chunk = (int)c;
    n_split = (int)((span + c - 1) / c);
}

size_t attn_paged_workspace(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head, int64_t d_head) {
    int chunk, n_split;
    pa_plan(n_seq, max_len, n_q_head, n_kv_head, chunk, n_split);
    return n_split > 1 ? (size_t)(n_seq * n_q_head) * n_split * (d_head + 2) * 4 : 0;
}

template <typename TC, int DC, bool EXACT>
static void run_paged(const AttnPaged &p, int chunk, int n_split, hipStream_t stream) {
    const int group = p.n_q_head / p.kv.n_head;
    const dim3 grid(n_split, p.kv.n_head * ((group + 15) / 16), p.n_seq);
    constexpr int NP = sizeof(TC) == 2 && Pa<TC>::up == 1.0f ? 3 : 2;
    if (NP == 3 && p.out_f32)
        hipLaunchKernelGGL((k_attn_paged<TC, DC, EXACT, NP>), grid, dim3(PA_NT), 0, stream, p, chunk, n_split);
    else
        hipLaunchKernelGGL((k_attn_paged<TC, DC, EXACT, 2>), grid, dim3(PA_NT), 0, stream, p, chunk, n_split);
}
template <typename TC>
static hipError_t run_paged_d(const AttnPaged &p, hipStream_t stream) {
    int chunk, n_split;
    pa_plan(p.n_seq, p.max_len, p.n_q_head, p.kv.n_head, chunk, n_split);
    const int d = p.kv.d_head;
    if (d == 64) run_paged<TC, 2, true>(p, chunk, n_split, stream);
    else if (d == 128) run_paged<TC, 4, true>(p, chunk, n_split, stream);
    else if (d == 256) run_paged<TC, 8, true>(p, chunk, n_split, stream);
    else if (d < 64) run_paged<TC, 2, false>(p, chunk, n_split, stream);
    else if (d <= 96) run_paged<TC, 3, false>(p, chunk, n_split, stream);
    else if (d <= 192) run_paged<TC, 6, false>(p, chunk, n_split, stream);
    else run_paged<TC, 8, false>(p, chunk, n_split, stream);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || n_split == 1) return e;
    hipLaunchKernelGGL(k_attn_join<TC>, dim3(p.n_q_head, p.n_seq), dim3(PA_NT), 0, stream, p, chunk, n_split);
    return hipGetLastError();
}
hipError_t launch_attn_paged(const AttnPaged &p, hipStream_t stream) {
    return p.kv.type == TY_F16 ? run_paged_d<_Float16>(p, stream) : run_paged_d<__bf16>(p, stream);
}

}  // namespace s2x
