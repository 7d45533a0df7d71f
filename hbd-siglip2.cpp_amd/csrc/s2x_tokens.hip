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
// sequence of each of its rows and new pages by binary search there.  Its
// latencies are what it costs (lengths in, sums, search, table, rows out: 5.1
// us for 200 sequences with one row each, 6.5 for 700 with 86,000); two
// launches with the sums in memory would add one.
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

// PER: most sequences of a thread.
template <int PER>
__global__ __launch_bounds__(KS_NT) void k_kv_slots(KvSlots p) {
    __shared__ int32_t tok0[PER * KS_NT], page0[PER * KS_NT], held[PER * KS_NT];  // saturated starts, lengths
    __shared__ int64_t wsum[2][KS_NT / WAVE];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int page_up = (1 << p.page_shift) - 1;
    auto pages = [&](int64_t len) { return (len + page_up) >> p.page_shift; };

    // prefix sums: each thread a run of sequences, then the waves' sums
    const int per = PER == 1 ? 1 : (p.n_seq + KS_NT - 1) / KS_NT, b0 = tid * per;
    int32_t len[PER], n[PER];
    int64_t st = 0, sp = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool in = i < per && b0 + i < p.n_seq;
        len[i] = in ? max(p.kv_len[b0 + i], 0) : 0;
        n[i] = in ? max(p.n_new[b0 + i], 0) : 0;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        st += n[i];
        sp += pages((int64_t)len[i] + n[i]) - pages(len[i]);
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
    int64_t t0 = it - st, f0 = ip - sp, n_tok = 0, n_fresh = 0;
#pragma unroll
    for (int w = 0; w < KS_NT / WAVE; ++w) {
        if (w < wave) {
            t0 += wsum[0][w];
            f0 += wsum[1][w];
        }
        n_tok += wsum[0][w];
        n_fresh += wsum[1][w];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int b = b0 + i;
        if (i < per && b < p.n_seq) {
            // (starts past the last row or page any call can hold: as that)
            tok0[b] = (int32_t)min(t0, (int64_t)INT32_MAX);
            page0[b] = (int32_t)min(f0, (int64_t)INT32_MAX);
            held[b] = len[i];
            if (blockIdx.x == 0) {
                p.len_out[b] = (int32_t)min((int64_t)len[i] + n[i], (int64_t)INT32_MAX);
                p.tok_start[b] = (int32_t)min(t0, p.max_tok);
            }
            t0 += n[i];
            f0 += pages((int64_t)len[i] + n[i]) - pages(len[i]);
        }
    }
    if (blockIdx.x == 0 && tid == 0) {
        p.tok_start[p.n_seq] = (int32_t)min(n_tok, p.max_tok);
        p.used[0] = n_fresh;
        p.used[1] = n_tok;
    }
    __syncthreads();

    const int64_t step = (int64_t)gridDim.x * KS_NT, first = (int64_t)blockIdx.x * KS_NT + tid;
    auto given = [&](int64_t f) {  // the f-th page taken from the free list
        if (f >= p.n_free) return -1;
        const int32_t id = p.free_pages[f];
        return id >= 0 && id < p.n_pages ? id : -1;
    };
    // the rows; entries of the table that this call writes are not read back
    for (int64_t t = first; t < p.max_tok; t += step) {
        int64_t pos = 0, slot = -1;
        if (t < n_tok) {
            const int b = ks_upper(tok0, p.n_seq, (int32_t)t);
            pos = (int64_t)held[b] + t - tok0[b];
            const int64_t i = pos >> p.page_shift, have = pages(held[b]);
            int32_t id = -1;
            if (i < p.ld_table) id = i < have ? p.table[b * p.ld_table + i] : given(page0[b] + i - have);
            if (id >= 0 && id < p.n_pages) slot = ((int64_t)id << p.page_shift) + (pos & page_up);
        }
        p.pos[t] = (int32_t)min(pos, (int64_t)INT32_MAX);
        p.slots[t] = slot;
    }
    // the tables' new entries; past a row's end on to the next sequence's pages, so
    // that the rounds are the table's, not those of lengths that no table holds
    // (up to 2^31 pages)
    for (int64_t f = first; f < min(n_fresh, (int64_t)INT32_MAX); f += step) {
        const int b = ks_upper(page0, p.n_seq, (int32_t)f);
        const int64_t i = pages(held[b]) + f - page0[b];
        if (i < p.ld_table) {
            p.table[b * p.ld_table + i] = given(f);
        } else {
            if (b + 1 >= p.n_seq) break;
            f += (uint32_t)(page0[b + 1] - (int32_t)f - 1) / (uint32_t)step * step;  // (page0[b + 1] > f)
        }
    }
}

hipError_t launch_kv_slots(const KvSlots &p, hipStream_t stream) {
    const int64_t rows = p.max_tok > p.n_seq ? p.max_tok : p.n_seq;
    const int64_t wgs = (rows + KS_NT - 1) / KS_NT;
    auto kern = p.n_seq <= KS_NT ? k_kv_slots<1> : k_kv_slots<KV_MAX_SEQ / KS_NT>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(wgs < 1 ? 1 : wgs > 256 ? 256 : wgs)), dim3(KS_NT), 0, stream, p);
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

template <typename T>
struct Qk4 {
    typedef T vec __attribute__((ext_vector_type(4)));
};

// One workgroup: a token's heads (those of its part, where tokens are few), NT / G
// at a time.  VEC: d_rot % 8 == 0, so that a lane's values are two whole
// pieces of four.  cos and sin are evaluated once a token and pair, into LDS; a
// lane's weights stay in its registers; the next head's values are loaded
// before the present one's are used.  Bound by its bytes: 8,191 rows of 32 + 2 x
// 8 heads of 128, bf16 to bf16, 39.5 us = 5.1 TB/s, a large copy's rate (4.9 to
// 5.3).  Several tokens a workgroup, their number at run time, were slower there
// (43 us with 2, 47 with 4); two were faster where heads are few, since threads
// idle there and a token's weights, angles and barrier are paid for few bytes
// (20,000 rows of 8 + 2 heads of 128 28.6 us against 32.4, of 4 + 8 heads of 64
// 16.8 against 19.8): given up for the wide rows, not tried at compile time.  NT
// and the loop left to run time were 42, the weights as single floats and an IEEE
// square root and division 55.  Not VEC: single elements, 8,191 rows of 16 + 32
// heads of 72 in bf16, 36 turned, 89 us, with 72 turned 34.
template <typename TX, typename TC, int G, bool VEC, int NT>
__global__ __launch_bounds__(NT) void k_qk_norm_rope(QkNormRope p) {
    typedef typename Qk4<TX>::vec xvec;
    typedef typename Qk4<TC>::vec cvec;
    __shared__ float2 turn[128];  // cos, sin of the token's pairs
    const int tid = threadIdx.x, half = p.d_rot / 2, d = p.kv.d_head;
    const int64_t row = blockIdx.x;
    const int lane = tid % G, n_rot = (p.d_rot + 7) / 8;
    const int nq = p.n_q_head, nk = p.kv.n_head, heads = nq + 2 * nk, step = gridDim.y * (NT / G);
    // this lane's values: element e0 + i and e1 + i (i < 4), those below their ends
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
    const int a0 = live ? e0 : 0, a1 = live ? e1 : 4;  // (idle lanes read, and drop, a live place)

    struct Head {
        xvec a, b;
    };
    auto load = [&](int h) {
        const TX *src = reinterpret_cast<const TX *>(p.x) + row * p.ld_x + (int64_t)h * d;
        Head v;
        if constexpr (VEC) {
            v.a = *reinterpret_cast<const xvec *>(src + a0);
            v.b = *reinterpret_cast<const xvec *>(src + a1);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v.a[k] = e0 + k < end0 ? src[e0 + k] : (TX)0.0f;
                v.b[k] = e1 + k < end1 ? src[e1 + k] : (TX)0.0f;
            }
        }
        return v;
    };
    int h = blockIdx.y * (NT / G) + tid / G;
    Head next = {};
    if (h < heads) next = load(h);
    // the weights of this lane's values (a kind of head without a norm takes no
    // factor at all)
    typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
    float wq[8], wk[8];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const float *w = c ? p.k_norm : p.q_norm;
        float *to = c ? wk : wq;
#pragma unroll
        for (int k = 0; k < 8; ++k) to[k] = 0.0f;
        if (!w) continue;
        if constexpr (VEC) {
            const f4 u = *reinterpret_cast<const f4 *>(w + a0), v = *reinterpret_cast<const f4 *>(w + a1);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                to[k] = u[k];
                to[4 + k] = v[k];
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                to[k] = e0 + k < end0 ? w[e0 + k] : 0.0f;
                to[4 + k] = e1 + k < end1 ? w[e1 + k] : 0.0f;
            }
        }
    }
    const int64_t slot = p.slots[row], page = slot >> p.kv.page_shift;
    const bool cached = slot >= 0 && page < p.kv.n_pages;
    const int64_t place = page * p.kv.ld_page + (slot & ((1 << p.kv.page_shift) - 1)) * p.kv.ld_tok;
    if (tid < half) {  // (half <= NT: 3 heads or more of G lanes, half <= 4 G)
        const double a = (double)p.pos[row] * p.freq[tid];
        // whole turns off: 2 pi as a head and a tail, so that the product
        // with up to 2^40 turns keeps 2^-50 of a turn
        const double n = __builtin_rint(a * 0.15915494309189535);
        const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, a));
        float s, c;
        sincosf((float)r, &s, &c);
        turn[tid] = make_float2(c, s);
    }
    __syncthreads();

    const float inv_d = 1.0f / (float)d;
    for (; h < heads; h += step) {
        const Head cur = next;
        if (h + step < heads) next = load(h + step);
        float a[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a[k] = live ? (float)cur.a[k] : 0.0f;
            b[k] = live ? (float)cur.b[k] : 0.0f;
        }
        const bool query = h < nq, value = h >= nq + nk;
        if (query ? p.q_norm != nullptr : !value && p.k_norm != nullptr) {  // (uniform over the group of lanes)
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) ss = fmaf(b[k], b[k], fmaf(a[k], a[k], ss));
            // v_rsq_f32 (1 ulp) where its argument is a normal number
            const float var = fmaf(group_sum<G>(ss), inv_d, p.eps);
            const float inv = var >= 0x1p-126f ? __builtin_amdgcn_rsqf(var) : 1.0f / sqrtf(var);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                a[k] = a[k] * inv * (query ? wq[k] : wk[k]);
                b[k] = b[k] * inv * (query ? wq[4 + k] : wk[4 + k]);
            }
        }
        if (!value && turns) {
            // (a lane's last pairs may be past the rotated part: theirs are
            // zeros, turned by some other pair's angle)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 cs = turn[VEC ? 4 * lane + k : min(4 * lane + k, half - 1)];
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
        if (!live || (!query && !cached)) continue;
        TC *dst;
        if (query) dst = reinterpret_cast<TC *>(p.q) + row * p.ld_q + (int64_t)h * d;
        else if (value) dst = reinterpret_cast<TC *>(p.kv.v) + place + (h - nq - nk) * p.kv.ld_head;
        else dst = reinterpret_cast<TC *>(p.kv.k) + place + (h - nq) * p.kv.ld_head;
        if constexpr (VEC) {
            cvec u, v;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u[k] = (TC)f32_materialize(a[k]);
                v[k] = (TC)f32_materialize(b[k]);
            }
            *reinterpret_cast<cvec *>(dst + e0) = u;
            *reinterpret_cast<cvec *>(dst + e1) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (e0 + k < end0) dst[e0 + k] = (TC)f32_materialize(a[k]);
                if (e1 + k < end1) dst[e1 + k] = (TC)f32_materialize(b[k]);
            }
        }
    }
}

template <typename TX, typename TC, int G, int NT>
static hipError_t run_qk_nt(const QkNormRope &p, hipStream_t stream) {
    const int heads = p.n_q_head + 2 * p.kv.n_head, per_wg = NT / G, rounds = (heads + per_wg - 1) / per_wg;
    // 8 workgroups a CU: fewer tokens than that share a token's heads among
    // workgroups (64 of 48 heads: 3 parts 3.6 us, 2 parts 4.3; 2,000: one part
    // 12.8, 2 parts 13.0, 3 parts 14.8)
    const int64_t most = 2048 / p.n_tok;
    const int parts = most < 1 ? 1 : most > rounds ? rounds : (int)most;
    auto kern = p.d_rot % 8 ? k_qk_norm_rope<TX, TC, G, false, NT> : k_qk_norm_rope<TX, TC, G, true, NT>;
    hipLaunchKernelGGL(kern, dim3((unsigned)p.n_tok, (unsigned)parts), dim3(NT), 0, stream, p);
    return hipGetLastError();
}
template <typename TX, typename TC, int G>
static hipError_t run_qk(const QkNormRope &p, hipStream_t stream) {
    // no more waves than a token's heads fill: 21,445 rows of 1 + 2 heads of 96
    // 12.9 us, in 256 threads 21.4
    const int want = (p.n_q_head + 2 * p.kv.n_head) * G;
    if constexpr (3 * G <= 64)
        if (want <= 64) return run_qk_nt<TX, TC, G, 64>(p, stream);
    if constexpr (3 * G <= 128)
        if (want <= 128) return run_qk_nt<TX, TC, G, 128>(p, stream);
    return run_qk_nt<TX, TC, G, 256>(p, stream);
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
