// s2x_paged.hip -- attention of one new token per sequence over a paged cache.
#include "s2x_decode.h"
#include "s2x_device.h"

namespace s2x {

// One workgroup per sequence and query head, 256 keys at a time: a thread's
// score per key, the running maximum and sum, then a thread per output value.
constexpr int PA_NT = 256;

template <typename TC>
__global__ __launch_bounds__(PA_NT) void k_attn_paged(AttnPaged p) {
    __shared__ float prob[PA_NT], red[2][PA_NT / WAVE], qf[256];
    __shared__ int64_t at[PA_NT];  // places of the keys in the cache, -1 unseen
    const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x, wave = tid >> 6;
    const int d = p.kv.d_head, hk = h / (p.n_q_head / p.kv.n_head);
    const TC *k = (const TC *)p.kv.k + hk * p.kv.ld_head, *v = (const TC *)p.kv.v + hk * p.kv.ld_head;
    int64_t len = min(max(p.kv_len[s], 0), p.max_len);
    len = min(len, p.ld_table << p.kv.page_shift);
    const int64_t first = p.window > 0 ? max(len - p.window, (int64_t)0) : 0;
    if (tid < d) qf[tid] = (float)((const TC *)p.q)[s * p.ld_q + (int64_t)h * d + tid];
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    for (int64_t c = first; c < len; c += PA_NT) {
        const int64_t t = c + tid;
        float sc = -INFINITY;
        int64_t place = -1;
        if (t < len) {
            const int32_t id = p.table[s * p.ld_table + (t >> p.kv.page_shift)];
            if (id >= 0 && id < p.kv.n_pages) {
                place = id * p.kv.ld_page + (t & ((1 << p.kv.page_shift) - 1)) * p.kv.ld_tok;
                float a = 0.0f;
                for (int i = 0; i < d; ++i) a = fmaf(qf[i], (float)k[place + i], a);
                sc = a * p.scale;
            }
        }
        at[tid] = place;
        float mx = group_max<64>(sc);
        if ((tid & 63) == 0) red[0][wave] = mx;
        __syncthreads();
        mx = m;
        for (int w = 0; w < PA_NT / WAVE; ++w) mx = fmaxf(mx, red[0][w]);
        const float base = mx == -INFINITY ? 0.0f : mx;
        const float e = expf(sc - base), f = expf(m - base);
        prob[tid] = e;
        const float sum = group_sum<64>(e);
        if ((tid & 63) == 0) red[1][wave] = sum;
        __syncthreads();
        l = l * f;
        for (int w = 0; w < PA_NT / WAVE; ++w) l = l + red[1][w];
        m = mx;
        if (tid < d) {
            acc = acc * f;
            for (int j = 0; j < PA_NT; ++j)
                if (at[j] >= 0) acc = fmaf(prob[j], (float)v[at[j] + tid], acc);
        }
        __syncthreads();
    }
    if (tid < d) {
        const float o = l > 0.0f ? acc / l : l;
        const int64_t i = s * p.ld_out + (int64_t)h * d + tid;
        if (p.out_f32) ((float *)p.out)[i] = o;
        else ((TC *)p.out)[i] = (TC)o;
    }
    if (tid == 0 && p.lse) p.lse[(int64_t)s * p.n_q_head + h] = l > 0.0f ? logf(l) + m : l - INFINITY;
}

size_t attn_paged_workspace(int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_attn_paged(const AttnPaged &p, hipStream_t stream) {
    auto kern = p.kv.type == TY_F16 ? k_attn_paged<_Float16> : k_attn_paged<__bf16>;
    hipLaunchKernelGGL(kern, dim3(p.n_q_head, p.n_seq), dim3(PA_NT), 0, stream, p);
    return hipGetLastError();
}

}  // namespace s2x
