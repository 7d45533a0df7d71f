// s2x_tokens.hip -- the decode step around its products: block tables and slot
// maps from the lengths of a batch (k_kv_slots), and the projections' rows to
// queries and cache entries (k_qk_norm_rope).
#include "s2x_decode.h"
#include "s2x_device.h"

namespace s2x {

// ---------------------------------------------------------------------------
// Block tables and slot maps.  Sequence b's rows begin at the exclusive prefix
// sum of n_new, its new pages at the prefix sum of
//   ceil((len + n) / page) - ceil(len / page)
// in the free list.  One launch, no workspace: every workgroup sums all
// lengths itself (8 bytes a sequence out of the L2) into LDS, then finds the
// sequence of each of its rows and new pages by binary search there.  The
// launch's latency is what it costs; two launches with the prefix sums in
// memory would add one.
// ---------------------------------------------------------------------------
constexpr int KS_NT = 1024;

__device__ __forceinline__ int ks_upper(const int32_t *first, int n, int32_t t) {
    int lo = 0, hi = n;  // the last i with first[i] <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

__global__ __launch_bounds__(KS_NT) void k_kv_slots(KvSlots p) {
    __shared__ int32_t tok0[KV_MAX_SEQ], page0[KV_MAX_SEQ];  // saturated starts
    __shared__ int64_t wsum[2][KS_NT / WAVE], total[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int page_up = (1 << p.page_shift) - 1;
    auto counts = [&](int b, int64_t &len, int64_t &n, int64_t &have, int64_t &fresh) {
        len = max(p.kv_len[b], 0);
        n = max(p.n_new[b], 0);
        have = (len + page_up) >> p.page_shift;
        fresh = ((len + n + page_up) >> p.page_shift) - have;
    };

    // prefix sums: each thread a run of sequences, then the waves' sums
    const int per = (p.n_seq + KS_NT - 1) / KS_NT;
    const int b0 = min(tid * per, p.n_seq), b1 = min(b0 + per, p.n_seq);
    int64_t st = 0, sp = 0, len, n, have, fresh;
    for (int b = b0; b < b1; ++b) {
        counts(b, len, n, have, fresh);
        st += n;
        sp += fresh;
    }
    int64_t it = st, ip = sp;  // inclusive over the wave
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int64_t a = __shfl_up(it, o), b = __shfl_up(ip, o);
        if (lane >= o) {
            it += a;
            ip += b;
        }
    }
    if (lane == WAVE - 1) {
        wsum[0][wave] = it;
        wsum[1][wave] = ip;
    }
    __syncthreads();
    int64_t bt = 0, bp = 0;
#pragma unroll
    for (int w = 0; w < KS_NT / WAVE; ++w) {
        if (w < wave) {
            bt += wsum[0][w];
            bp += wsum[1][w];
        }
    }
    if (tid == KS_NT - 1) {
        total[0] = bt + it;
        total[1] = bp + ip;
    }
    int64_t t0 = bt + it - st, f0 = bp + ip - sp;  // of this thread's first sequence
    for (int b = b0; b < b1; ++b) {
        counts(b, len, n, have, fresh);
        // (starts past the last row or page any call can hold: as that)
        tok0[b] = (int32_t)min(t0, (int64_t)INT32_MAX);
        page0[b] = (int32_t)min(f0, (int64_t)INT32_MAX);
        if (blockIdx.x == 0) {
            p.len_out[b] = (int32_t)min(len + n, (int64_t)INT32_MAX);
            p.tok_start[b] = (int32_t)min(t0, p.max_tok);
        }
        t0 += n;
        f0 += fresh;
    }
    __syncthreads();
    const int64_t n_tok = total[0], n_fresh = total[1];
    if (blockIdx.x == 0 && tid == 0) {
        p.tok_start[p.n_seq] = (int32_t)min(n_tok, p.max_tok);
        p.used[0] = n_fresh;
        p.used[1] = n_tok;
    }

    const int64_t step = (int64_t)gridDim.x * KS_NT, first = (int64_t)blockIdx.x * KS_NT + tid;
    auto given = [&](int64_t f) {  // the f-th page taken from the free list
        if (f >= p.n_free) return -1;
        const int32_t id = p.free_pages[f];
        return id >= 0 && id < p.n_pages ? id : -1;
    };
    // the tables' new entries
    for (int64_t f = first; f < min(n_fresh, (int64_t)INT32_MAX); f += step) {
        const int b = ks_upper(page0, p.n_seq, (int32_t)f);
        counts(b, len, n, have, fresh);
        const int64_t i = have + f - page0[b];
        if (i < p.ld_table) p.table[b * p.ld_table + i] = given(f);
    }
    // the rows; entries of the table that this call writes are not read back
    for (int64_t t = first; t < p.max_tok; t += step) {
        int64_t pos = 0, slot = -1;
        if (t < n_tok) {
            const int b = ks_upper(tok0, p.n_seq, (int32_t)t);
            counts(b, len, n, have, fresh);
            pos = len + t - tok0[b];
            const int64_t i = pos >> p.page_shift;
            int32_t id = -1;
            if (i < p.ld_table) id = i < have ? p.table[b * p.ld_table + i] : given(page0[b] + i - have);
            if (id >= 0 && id < p.n_pages) slot = ((int64_t)id << p.page_shift) + (pos & page_up);
        }
        p.pos[t] = (int32_t)min(pos, (int64_t)INT32_MAX);
        p.slots[t] = slot;
    }
}

hipError_t launch_kv_slots(const KvSlots &p, hipStream_t stream) {
    const int64_t rows = p.max_tok > p.n_seq ? p.max_tok : p.n_seq;
    const int64_t wgs = (rows + KS_NT - 1) / KS_NT;
    hipLaunchKernelGGL(k_kv_slots, dim3((unsigned)(wgs < 1 ? 1 : wgs > 256 ? 256 : wgs)), dim3(KS_NT), 0,
                       stream, p);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Head norms, position rotation and the write into the cache, one pass.
//   y = h * (1/sqrt(mean(h^2) + eps)) * w,   (a, b) -> (a c - b s, b c + a s)
// with c, s of pos * freq[j]: the angle and its remainder by whole turns in
// f64 (at position 2^20 an f32 angle is off by up to 2^-4), cos and sin of the
// remainder in f32.  A head is a group of G lanes with 8 values each, pairs
// whole in one lane: lanes 0 .. ceil(d_rot / 8) - 1 hold 4 pairs, the lanes
// behind them 8 values that stay.
// ---------------------------------------------------------------------------
constexpr int QK_NT = 256;

template <typename T>
__device__ __forceinline__ void qk_load(const T *p, float (&v)[4]) {
    typedef T vec __attribute__((ext_vector_type(4)));
    const vec t = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)t[i];
}
template <typename T>
__device__ __forceinline__ void qk_store(T *p, const float (&v)[4]) {
    typedef T vec __attribute__((ext_vector_type(4)));
    vec t;
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = (T)f32_materialize(v[i]);
    *reinterpret_cast<vec *>(p) = t;
}

// One workgroup: n_t tokens from t0, of each the heads h0, h0 + dh, ...
template <typename TX, typename TC, int G>
__global__ __launch_bounds__(QK_NT) void k_qk_norm_rope(QkNormRope p, int n_t) {
    extern __shared__ float2 turn[];  // [n_t][pairs] cos, sin
    const int tid = threadIdx.x, half = p.d_rot / 2, d = p.kv.d_head;
    const int64_t t0 = (int64_t)blockIdx.x * n_t;
    const int nt = (int)min((int64_t)n_t, p.n_tok - t0);
    for (int i = tid; i < nt * half; i += QK_NT) {
        const int t = i / half, j = i - t * half;
        const double a = (double)p.pos[t0 + t] * p.freq[j];
        // whole turns off: 2 pi as a head and a tail, so that the product
        // with up to 2^40 turns keeps 2^-50 of a turn
        const double n = __builtin_rint(a * 0.15915494309189535);
        const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
        float s, c;
        sincosf((float)r, &s, &c);
        turn[i] = make_float2(c, s);
    }
    __syncthreads();

    const int lane = tid % G, n_rot = (p.d_rot + 7) / 8;
    const int heads = p.n_q_head + 2 * p.kv.n_head;
    const bool vec = p.d_rot % 8 == 0;  // pairs in whole lanes: 16-byte pieces
    // this lane's values: element e0 + i (i < 4) and e1 + i - 4, those below
    // their ends
    int e0, e1, end0, end1;
    const bool turns = lane < n_rot;
    if (turns && !p.pairs) {
        e0 = 4 * lane, e1 = half + 4 * lane;
        end0 = half, end1 = p.d_rot;
    } else {
        e0 = turns ? 8 * lane : p.d_rot + 8 * (lane - n_rot);
        e1 = e0 + 4;
        end0 = end1 = turns ? p.d_rot : d;
    }
    const bool live = e0 < end0;
    for (int i = blockIdx.y * (QK_NT / G) + tid / G; i < nt * heads; i += gridDim.y * (QK_NT / G)) {
        const int t = i / heads, h = i - t * heads;
        const int64_t row = t0 + t;
        const TX *src = reinterpret_cast<const TX *>(p.x) + row * p.ld_x + (int64_t)h * d;
        float a[4] = {0, 0, 0, 0}, b[4] = {0, 0, 0, 0};
        if (live) {
            if (vec) {
                qk_load(src + e0, a);
                qk_load(src + e1, b);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (e0 + k < end0) a[k] = (float)src[e0 + k];
                    if (e1 + k < end1) b[k] = (float)src[e1 + k];
                }
            }
        }
        const bool value = h >= p.n_q_head + p.kv.n_head;
        const float *w = h < p.n_q_head ? p.q_norm : value ? nullptr : p.k_norm;
        if (w) {  // (uniform over the group of lanes)
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) ss = fmaf(b[k], b[k], fmaf(a[k], a[k], ss));
            const float inv = 1.0f / sqrtf(group_sum<G>(ss) / (float)d + p.eps);
            if (live) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    a[k] = a[k] * inv * (e0 + k < end0 ? w[e0 + k] : 0.0f);
                    b[k] = b[k] * inv * (e1 + k < end1 ? w[e1 + k] : 0.0f);
                }
            }
        }
        if (!value && turns) {
            // (a lane's last pairs may be past the rotated part: theirs are
            // zeros, turned by some other pair's angle)
            const float2 *ct = turn + t * half;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 cs = ct[min(4 * lane + k, half - 1)];
                if (p.pairs) {
                    float &u = k < 2 ? a[2 * k] : b[2 * k - 4], &v = k < 2 ? a[2 * k + 1] : b[2 * k - 3];
                    const float u0 = u;
                    u = fmaf(u0, cs.x, -(v * cs.y));
                    v = fmaf(v, cs.x, u0 * cs.y);
                } else {
                    const float u0 = a[k];
                    a[k] = fmaf(u0, cs.x, -(b[k] * cs.y));
                    b[k] = fmaf(b[k], cs.x, u0 * cs.y);
                }
            }
        }
        TC *dst;
        if (h < p.n_q_head) {
            dst = reinterpret_cast<TC *>(p.q) + row * p.ld_q + (int64_t)h * d;
        } else {
            const int64_t slot = p.slots[row], page = slot >> p.kv.page_shift;
            if (slot < 0 || page >= p.kv.n_pages) continue;
            const int hk = value ? h - p.n_q_head - p.kv.n_head : h - p.n_q_head;
            dst = reinterpret_cast<TC *>(value ? p.kv.v : p.kv.k) + page * p.kv.ld_page + hk * p.kv.ld_head +
                  (slot & ((1 << p.kv.page_shift) - 1)) * p.kv.ld_tok;
        }
        if (!live) continue;
        if (vec) {
            qk_store(dst + e0, a);
            qk_store(dst + e1, b);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (e0 + k < end0) dst[e0 + k] = (TC)f32_materialize(a[k]);
                if (e1 + k < end1) dst[e1 + k] = (TC)f32_materialize(b[k]);
            }
        }
    }
}

template <typename TX, typename TC, int G>
static hipError_t run_qk(const QkNormRope &p, hipStream_t stream) {
    const int heads = p.n_q_head + 2 * p.kv.n_head, per_wg = QK_NT / G;
    const int half = p.d_rot / 2;
    int n_t = 1, parts = 1;
    if (p.n_tok < 1024) {
        parts = (heads + per_wg - 1) / per_wg;
    } else {
        n_t = half ? QK_NT / half : 4;
        n_t = n_t < 1 ? 1 : n_t > 4 ? 4 : n_t;
    }
    const int64_t wgs = (p.n_tok + n_t - 1) / n_t;
    hipLaunchKernelGGL((k_qk_norm_rope<TX, TC, G>), dim3((unsigned)wgs, (unsigned)parts), dim3(QK_NT),
                       (unsigned)(sizeof(float2) * n_t * (half ? half : 1)), stream, p, n_t);
    return hipGetLastError();
}
template <typename TX, typename TC>
static hipError_t run_qk_g(const QkNormRope &p, hipStream_t stream) {
    // lanes with pairs, then lanes with the values that stay
    const int lanes = (p.d_rot + 7) / 8 + (p.kv.d_head - p.d_rot + 7) / 8;
    if (lanes <= 8) return run_qk<TX, TC, 8>(p, stream);
    if (lanes <= 16) return run_qk<TX, TC, 16>(p, stream);
    if (lanes <= 32) return run_qk<TX, TC, 32>(p, stream);
    return run_qk<TX, TC, 64>(p, stream);
}
template <typename TX>
static hipError_t run_qk_c(const QkNormRope &p, hipStream_t stream) {
    return p.kv.type == TY_F16 ? run_qk_g<TX, _Float16>(p, stream) : run_qk_g<TX, __bf16>(p, stream);
}
hipError_t launch_qk_norm_rope_kv(const QkNormRope &p, hipStream_t stream) {
    switch (p.x_type) {
    case TY_F32: return run_qk_c<float>(p, stream);
    case TY_F16: return run_qk_c<_Float16>(p, stream);
    default: return run_qk_c<__bf16>(p, stream);
    }
}

}  // namespace s2x
