// s2x_prefix.hip -- attention of one new token per sequence where groups of
// sequences share their first tokens.
//
//   out = (sum over the prefix + sum over the own tokens), each with its running
//   maximum and sum, joined by e^(maximum - the larger one)
//
// The prefix's keys and values are read once for all query heads of the group that
// share a key head (its columns).  Up to 16 columns take the kernel of the decode
// step's attention, a wave a tile (s2x_paged.h), and so do the own tokens.  More
// columns: k_attn_prefix, whose waves share tiles of 64 keys in LDS and have 16 or
// 32 columns each.  All leave sums in the workspace; k_prefix_join adds them.
#include "s2x_paged.h"

namespace s2x {

template <typename TC, int DC, bool EXACT, int KT, int NW, PaMode MODE>
__global__ __launch_bounds__(NW * WAVE) void k_attn_group(AttnPrefix p, int chunk, int n_split, int n_parts, int part0) {
    pa_body<TC, DC, EXACT, KT, NW, MODE>(p, chunk, n_split, n_parts, part0);
}

constexpr int PX_TK = 64;  // keys of a tile
constexpr int PX_PAD_K = 8, PX_PAD_V = 16;  // rows in LDS end with these: reads of 16 rows spread over the banks

// DC, EXACT as in s2x_paged.h; NC: 16-column parts of a wave; NW: waves.
// A step: the next tile's pieces into registers, the products of this one, the
// pieces into the other half of LDS, one barrier.  S^T and O^T as in s2x_paged.h.
template <typename TC, int DC, bool EXACT, int NC, int NW>
__global__ __launch_bounds__(NW * WAVE) void k_attn_prefix(AttnPrefix args, int chunk, int n_split, int n_parts, int tiles) {
    typedef typename Pa<TC>::vec vec;
    constexpr int DP = 32 * DC, DT = 2 * DC, NT = NW * WAVE, NP = Pa<TC>::terms;
    constexpr int PER = (PX_TK * (DP / 8) + NT - 1) / NT;  // pieces of a thread
    extern __shared__ __align__(16) uint8_t lds[];
    const AttnPaged &p = args.a;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = EXACT ? DP : p.kv.d_head, nch = d / 8, sk = d + PX_PAD_K, sv = d + PX_PAD_V;
    const int share = p.n_q_head / p.kv.n_head;
    // the tiles of columns, then the heads, of one chunk follow each other on one XCD
    int u = xcd_linear(blockIdx.x, gridDim.x);
    const int tile = u % tiles;
    u /= tiles;
    const int hk = u % p.kv.n_head;
    u /= p.kv.n_head;
    const int gi = u % args.n_group, split = u / args.n_group;
    const PaGroup gr = pa_group(args, gi);
    const int cols = gr.size * share, c0 = tile * (16 * NC * NW);
    const int64_t start = (int64_t)split * chunk, end = min(start + chunk, gr.len);
    if (c0 >= cols || start >= end) return;  // (uniform)

    const TC *kp = (const TC *)p.kv.k + hk * p.kv.ld_head, *vp = (const TC *)p.kv.v + hk * p.kv.ld_head;
    const int32_t *row = p.table + (int64_t)gr.first * p.ld_table;
    const uint32_t pmask = (1u << p.kv.page_shift) - 1, ldp = (uint32_t)p.kv.ld_page, ldt = (uint32_t)p.kv.ld_tok;
    TC *kl = reinterpret_cast<TC *>(lds), *vl = kl + 2 * PX_TK * sk;

    const int w0 = c0 + wave * 16 * NC;
    const bool live = w0 < cols;
    vec q[NC][DC];
    int64_t lim[NC];
    bool ragged = false;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int c = w0 + 16 * n + r, i = min(c, cols - 1) / share, s = gr.first + i;
        const int64_t qrow = pa_row_of(p, s);
        lim[n] = pa_len(p, s);
        ragged |= __builtin_amdgcn_ballot_w64(lim[n] < end) != 0;
#pragma unroll
        for (int k = 0; k < DC; ++k) {
            q[n][k] = vec{};
            if (c < cols && qrow >= 0 && (EXACT || 32 * k + 8 * g < d))
                q[n][k] = *reinterpret_cast<const vec *>((const TC *)p.q + qrow * p.ld_q + (int64_t)(hk * share + c - i * share) * d +
                                                         32 * k + 8 * g);
        }
    }

    auto entry_of = [&](int64_t t0) { return row[min((t0 + lane) >> p.kv.page_shift, p.ld_table - 1)]; };
    const uint32_t magic = (65536u + nch - 1) / nch;  // f / nch for f < 2,048
    vec kr[PER], vr[PER];
    uint64_t seen = 0;
    auto load = [&](int64_t t0, int32_t entry) {
        seen = __builtin_amdgcn_ballot_w64(t0 + lane < end && (uint32_t)entry < (uint32_t)p.kv.n_pages);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t f = i * NT + tid, key = EXACT ? f / (DP / 8) : f * magic >> 16;
            const uint32_t pid = (uint32_t)__shfl(entry, (int)(key & 63));
            kr[i] = vr[i] = vec{};
            if (f < (uint32_t)(PX_TK * nch) && (seen >> (key & 63) & 1)) {
                const uint64_t at = (uint64_t)pid * ldp + (((uint32_t)t0 + key) & pmask) * (uint64_t)ldt + 8 * (f - key * nch);
                kr[i] = *reinterpret_cast<const vec *>(kp + at);
                vr[i] = *reinterpret_cast<const vec *>(vp + at);
            }
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t f = i * NT + tid, key = EXACT ? f / (DP / 8) : f * magic >> 16;
            if (f < (uint32_t)(PX_TK * nch)) {
                *reinterpret_cast<vec *>(kl + (buf * PX_TK + key) * sk + 8 * (f - key * nch)) = kr[i];
                *reinterpret_cast<vec *>(vl + (buf * PX_TK + key) * sv + 8 * (f - key * nch)) = vr[i];
            }
        }
    };

    float m[NC], l[NC];
    v4f o[NC][DT];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[n][i] = v4f{0, 0, 0, 0};
    }
    const float sc = p.scale * 1.44269504088896341f;  // log2(e)

    load(start, entry_of(start));
    int32_t next = entry_of(start + PX_TK);
    store(0);
    uint64_t mask = seen;
    __syncthreads();
    int buf = 0;
    for (int64_t t0 = start; t0 < end; t0 += PX_TK, buf ^= 1) {
        const bool more = t0 + PX_TK < end;  // (uniform)
        if (more) {
            load(t0 + PX_TK, next);
            next = entry_of(t0 + 2 * PX_TK);
        }
        if (live) {
            const TC *kt = kl + buf * PX_TK * sk;
            TC *vt = vl + buf * PX_TK * sv;
            v4f st[NC][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int n = 0; n < NC; ++n) st[n][j] = v4f{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < DC; ++k) {
                    vec kk = vec{};
                    if (EXACT || 32 * k + 8 * g < d) kk = *reinterpret_cast<const vec *>(kt + (16 * j + r) * sk + 32 * k + 8 * g);
#pragma unroll
                    for (int n = 0; n < NC; ++n) st[n][j] = Pa<TC>::mfma(kk, q[n][k], st[n][j]);
                }
            }
            vec pt[NC][NP][2];
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                float mt = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        st[n][j][i] = st[n][j][i] * sc;
                    }
                if (mask != ~0ull || ragged) {  // (uniform)
                    const int left = (int)min(max(lim[n] - t0, (int64_t)0), (int64_t)PX_TK);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = 16 * j + 4 * g + i;
                            if (!(mask >> key & 1) || key >= left) st[n][j][i] = -INFINITY;
                        }
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mt = fmaxf(mt, st[n][j][i]);
                mt = fmaxf(mt, __shfl_xor(mt, 16));
                mt = fmaxf(mt, __shfl_xor(mt, 32));
                if (__builtin_amdgcn_ballot_w64(mt > m[n]) != 0) {
                    const float mn = fmaxf(m[n], mt), b = mn == -INFINITY ? 0.0f : mn;
                    const float alpha = __builtin_amdgcn_exp2f(m[n] - b);
                    m[n] = mn;
                    l[n] = l[n] * alpha;
#pragma unroll
                    for (int i = 0; i < DT; ++i) o[n][i] = o[n][i] * alpha;
                }
                const float base = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float e = __builtin_amdgcn_exp2f(st[n][j][i] - base);
                        l[n] = l[n] + e;
                        float x = e * Pa<TC>::up;
#pragma unroll
                        for (int t = 0; t < NP; ++t) {
                            pt[n][t][j >> 1][4 * (j & 1) + i] = (TC)x;
                            x = x - (float)pt[n][t][j >> 1][4 * (j & 1) + i];
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                if (!EXACT && 16 * i >= d) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v4s a[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        TC *src = vt + (32 * h + 16 * j + 4 * g + (r >> 2)) * sv + 16 * i + (r & 3) * 4;
                        a[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)src);
                    }
                    const vec a8 = __builtin_bit_cast(vec, __builtin_shufflevector(a[0], a[1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                    for (int n = 0; n < NC; ++n)
#pragma unroll
                        for (int t = 0; t < NP; ++t) o[n][i] = Pa<TC>::mfma(a8, pt[n][t][h], o[n][i]);
                }
            }
        }
        if (more) store(buf ^ 1);
        mask = seen;
        __syncthreads();
    }

    // o[n][i] is values 16 i + 4 g .. + 3 of column w0 + 16 n + r
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        l[n] = l[n] + __shfl_xor(l[n], 16);
        l[n] = l[n] + __shfl_xor(l[n], 32);
        const int c = w0 + 16 * n + r;
        if (c >= cols) continue;
        const int i = c / share;
        const int64_t at = ((int64_t)(gi * args.max_group + i) * p.n_q_head + hk * share + c - i * share) * n_parts + split;
        v4f *ov = reinterpret_cast<v4f *>(p.ws) + at * (d / 4);
#pragma unroll
        for (int k = 0; k < DT; ++k) {
            if (!EXACT && 16 * k + 4 * g >= d) break;
            ov[4 * k + g] = o[n][k];
        }
        if (g == 0)
            reinterpret_cast<float2 *>((float *)p.ws + (int64_t)args.n_group * args.max_group * p.n_q_head * n_parts * d)[at] =
                make_float2(m[n], l[n]);
    }
}

// The parts of a sequence's prefix and of its own tokens joined, as k_attn_join
// does the chunks: a workgroup per query head and 4 LANES values of it.
constexpr int PXJ_NT = 256;
template <typename TC, int LANES>
__global__ __launch_bounds__(PXJ_NT) void k_prefix_join(AttnPrefix args, int chunk_p, int split_p, int chunk_o, int n_parts) {
    constexpr int GROUPS = PXJ_NT / LANES;
    __shared__ __align__(16) float part[GROUPS][LANES * 4 + 4];
    __shared__ float gm[GROUPS], gl[GROUPS];
    const AttnPaged &p = args.a;
    const int tid = threadIdx.x, d = p.kv.d_head, nq = d / 4, pieces = (nq + LANES - 1) / LANES;
    const int h = blockIdx.x / pieces, slot = blockIdx.y, gi = slot / args.max_group;
    const int grp = tid / LANES, e = (blockIdx.x - h * pieces) * LANES + tid % LANES;
    const PaGroup gr = pa_group(args, gi);
    const int s = gr.first + slot - gi * args.max_group;
    if (s >= gr.first + gr.size) return;  // (uniform)
    const int64_t qrow = pa_row_of(p, s);
    if (qrow < 0) return;  // (uniform)
    const PaRange own = pa_own(args, gr, s);
    const int np = (int)((gr.len + chunk_p - 1) / chunk_p);
    const int n = np + (own.len > own.begin ? (int)((own.len - own.begin + chunk_o - 1) / chunk_o) : 0);
    const int64_t at = ((int64_t)slot * p.n_q_head + h) * n_parts;
    const v4f *ov = reinterpret_cast<const v4f *>(p.ws) + at * nq + min(e, nq - 1);
    const float2 *mlp =
        reinterpret_cast<const float2 *>((const float *)p.ws + (int64_t)args.n_group * args.max_group * p.n_q_head * n_parts * d) + at;
    v4f a = {0, 0, 0, 0};
    float M = -INFINITY, L = 0.0f;
    for (int i = grp; i < n; i += GROUPS) {
        const int k = i < np ? i : split_p + i - np;
        const float2 t = mlp[k];
        const v4f x = ov[(int64_t)k * nq];
        const float mn = fmaxf(M, t.x), base = mn == -INFINITY ? 0.0f : mn;
        const float f0 = __builtin_amdgcn_exp2f(M - base), f1 = __builtin_amdgcn_exp2f(t.x - base);
        L = fmaf(t.y, f1, L * f0);
#pragma unroll
        for (int c = 0; c < 4; ++c) a[c] = fmaf(x[c], f1, a[c] * f0);
        M = mn;
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

struct PxPlan {
    int nw, nc, tiles;             // of the prefix; nc 0: the form of up to 16 columns
    int chunk_p, split_p, chunk_o, split_o;
    int parts() const { return split_p + split_o; }
};
static int64_t px_round(int64_t v, int64_t to, int64_t lo, int64_t hi) {
    v = v < lo ? lo : v > hi ? hi : v;
    return (v + to - 1) / to * to;
}
static PxPlan px_plan(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own, int64_t n_q_head,
                      int64_t n_kv_head, int64_t d_head) {
    PxPlan P;
    const int64_t share = n_q_head / n_kv_head, cols = share * max_group;
    if (cols <= 16) {
        P.nc = 0, P.nw = 4, P.tiles = 1;
    } else {
        P.nc = cols > 64 && d_head <= 128 ? 2 : 1;
        P.nw = cols <= 32 ? 2 : cols <= 128 ? 4 : 8;
        P.tiles = (int)((cols + 16 * P.nc * P.nw - 1) / (16 * P.nc * P.nw));
    }
    const int64_t units = n_group * n_kv_head * P.tiles, most = 1 << 20;
    int64_t c = px_round(max_prefix * units / (P.nc == 2 ? 256 : 512), 128, 128, most);
    if (units * ((max_prefix + c - 1) / c) > 1 << 22) c = px_round(max_prefix * units >> 21, 128, 128, 1 << 30);
    P.chunk_p = (int)c;
    P.split_p = (int)((max_prefix + c - 1) / c);
    const int64_t units_o = n_group * max_group * n_kv_head * ((share + 15) / 16), span = max_own + PA_ALIGN;
    c = max_own <= 320 ? span : px_round(span * units_o / 1536, 128, 256, most);
    c = (c + 127) / 128 * 128;
    if (units_o * ((span + c - 1) / c) > 1 << 22) c = px_round(span * units_o >> 21, 128, 128, 1 << 30);
    P.chunk_o = (int)c;
    P.split_o = (int)((span + c - 1) / c);
    return P;
}
size_t attn_prefix_workspace(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own, int64_t n_q_head,
                             int64_t n_kv_head, int64_t d_head) {
    const PxPlan P = px_plan(n_group, max_group, max_prefix, max_own, n_q_head, n_kv_head, d_head);
    return (size_t)(n_group * max_group * n_q_head) * P.parts() * (d_head + 2) * 4;
}

template <typename TC, int DC, bool EXACT, PaMode MODE>
static hipError_t run_group(const AttnPrefix &p, const PxPlan &P, hipStream_t stream) {
    constexpr int KT = DC > 4 ? 1 : 2, NW = 4;
    const int share = p.a.n_q_head / p.a.kv.n_head, d = p.a.kv.d_head;
    const int R = MODE == PA_PREFIX ? share * p.max_group : share < 16 ? share : 16;
    const int n_split = MODE == PA_PREFIX ? P.split_p : P.split_o;
    const int64_t units = MODE == PA_PREFIX ? p.n_group : (int64_t)p.n_group * p.max_group * ((share + 15) / 16);
    const int v = NW * KT * 16 * d * 2 + 64, o = NW * R * (DC * 32 + 4) * 4, lds = v > o ? v : o;
    auto kern = k_attn_group<TC, DC, EXACT, KT, NW, MODE>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(units * p.a.kv.n_head * n_split)), dim3(NW * WAVE), lds, stream, p,
                       MODE == PA_PREFIX ? P.chunk_p : P.chunk_o, n_split, P.parts(), MODE == PA_PREFIX ? 0 : P.split_p);
    return hipGetLastError();
}
template <typename TC, int DC, bool EXACT, int NC, int NW>
static hipError_t run_wide_w(const AttnPrefix &p, const PxPlan &P, hipStream_t stream) {
    const int64_t wgs = (int64_t)P.split_p * p.n_group * p.a.kv.n_head * P.tiles;
    const int lds = 2 * PX_TK * (2 * p.a.kv.d_head + PX_PAD_K + PX_PAD_V) * 2;
    auto kern = k_attn_prefix<TC, DC, EXACT, NC, NW>;
    hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(NW * WAVE), lds, stream, p, P.chunk_p, P.split_p, P.parts(), P.tiles);
    return hipGetLastError();
}
template <typename TC, int DC, bool EXACT>
static hipError_t run_prefix(const AttnPrefix &p, hipStream_t stream) {
    const PxPlan P = px_plan(p.n_group, p.max_group, p.max_prefix, p.max_own, p.a.n_q_head, p.a.kv.n_head, p.a.kv.d_head);
    hipError_t e = hipSuccess;
    if (P.split_p) {
        if (P.nc == 0) {
            e = run_group<TC, DC, EXACT, PA_PREFIX>(p, P, stream);
        } else if constexpr (DC <= 4) {
            e = P.nc == 2 ? (P.nw == 8 ? run_wide_w<TC, DC, EXACT, 2, 8>(p, P, stream) : run_wide_w<TC, DC, EXACT, 2, 4>(p, P, stream))
                          : (P.nw == 4 ? run_wide_w<TC, DC, EXACT, 1, 4>(p, P, stream) : run_wide_w<TC, DC, EXACT, 1, 2>(p, P, stream));
        } else {
            e = P.nw == 8   ? run_wide_w<TC, DC, EXACT, 1, 8>(p, P, stream)
                : P.nw == 4 ? run_wide_w<TC, DC, EXACT, 1, 4>(p, P, stream)
                            : run_wide_w<TC, DC, EXACT, 1, 2>(p, P, stream);
        }
    }
    if (e != hipSuccess) return e;
    e = run_group<TC, DC, EXACT, PA_OWN>(p, P, stream);
    if (e != hipSuccess) return e;
    const bool few = P.parts() <= 16;
    const int width = few ? 128 : 32, d = p.a.kv.d_head;
    auto join = few ? k_prefix_join<TC, 32> : k_prefix_join<TC, 8>;
    hipLaunchKernelGGL(join, dim3(p.a.n_q_head * ((d + width - 1) / width), p.n_group * p.max_group), dim3(PXJ_NT), 0, stream, p,
                       P.chunk_p, P.split_p, P.chunk_o, P.parts());
    return hipGetLastError();
}
template <typename TC>
static hipError_t run_prefix_d(const AttnPrefix &p, hipStream_t stream) {
    const int d = p.a.kv.d_head;
    return d == 64    ? run_prefix<TC, 2, true>(p, stream)
           : d == 128 ? run_prefix<TC, 4, true>(p, stream)
           : d == 256 ? run_prefix<TC, 8, true>(p, stream)
           : d < 64   ? run_prefix<TC, 2, false>(p, stream)
           : d <= 96  ? run_prefix<TC, 3, false>(p, stream)
           : d <= 192 ? run_prefix<TC, 6, false>(p, stream)
                      : run_prefix<TC, 8, false>(p, stream);
}
hipError_t launch_attn_prefix(const AttnPrefix &p, hipStream_t stream) {
    return p.a.kv.type == TY_F16 ? run_prefix_d<_Float16>(p, stream) : run_prefix_d<__bf16>(p, stream);
}

}  // namespace s2x
