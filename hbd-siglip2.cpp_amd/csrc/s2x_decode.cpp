// s2x_decode.cpp -- the extern "C" boundary of the decode step (include/s2x.h):
// argument checks and status codes of the Q4_0 products, the paged cache's
// slots, the query/key norms with rotation and the paged attention.
#include "s2x_decode.h"

#include <climits>
#include <new>

#include "s2x.h"
#include "s2x_internal.h"

// The opaque Q4_0 weight handle: repacked planes in device memory.
struct s2x_weight_q4 {
    s2x::Q4View view;
    void *mem = nullptr;  // base of the planes
    bool owns = false;    // hipFree on destroy
};

namespace s2x {

// (the last bound keeps the repack's grid within 2^32 threads: 38 GB of weight)
static bool q4_shape_ok(int64_t K, int64_t N) {
    return K > 0 && N > 0 && K % QK_ == 0 && K <= (1 << 20) && N <= (1 << 24) &&
           round_up_i(K, 128) * round_up_i(N, 128) <= (int64_t)1 << 36;
}
// planes: tiles of 1,024 bytes, then 128 bytes of scales a tile
static Q4View q4_view(void *base, int64_t K, int64_t N) {
    Q4View v;
    v.K = K;
    v.N = N;
    v.qs = (const uint8_t *)base;
    v.d = (const uint16_t *)(v.qs + v.tiles_n() * v.tiles_k() * 1024);
    return v;
}
static size_t q4_bytes(int64_t K, int64_t N) {
    return (size_t)round_up_i(round_up_i(K, 128) / 128 * (round_up_i(N, 16) / 16) * (1024 + 128), 256);
}

static bool type_size(int32_t type, int64_t &size) {
    size = type == S2X_TYPE_F32 ? 4 : 2;
    return type == S2X_TYPE_F32 || type == S2X_TYPE_F16 || type == S2X_TYPE_BF16;
}
static int log2_page(int64_t page) {  // -1: no power of two up to 65,536
    for (int i = 0; i <= 16; ++i)
        if (page == (int64_t)1 << i) return i;
    return -1;
}

static int check_cache(const s2x_kv_cache *c, KvView &v, const char *who) {
    if (!c) return fail(S2X_ERR_INVALID_ARG, "%s: cache is null", who);
    if (c->type != S2X_TYPE_F16 && c->type != S2X_TYPE_BF16)
        return fail(S2X_ERR_UNSUPPORTED, "%s: cache type %d (F16 or BF16)", who, (int)c->type);
    const int shift = log2_page(c->page_size);
    if (shift < 0)
        return fail(S2X_ERR_UNSUPPORTED, "%s: page_size %d is no power of two up to 65,536", who,
                    (int)c->page_size);
    if (c->n_pages <= 0 || c->n_pages > INT32_MAX || c->n_head <= 0 || c->d_head <= 0)
        return fail(S2X_ERR_INVALID_ARG, "%s: cache of %lld pages, %lld heads of %lld", who,
                    (long long)c->n_pages, (long long)c->n_head, (long long)c->d_head);
    if (c->d_head % 8 || c->d_head > 256 || c->n_head > 1024)
        return fail(S2X_ERR_UNSUPPORTED, "%s: d_head %% 8 == 0, d_head <= 256, at most 1,024 heads", who);
    const int64_t most = INT32_MAX, ps = c->page_size;  // (32-bit strides, 64-bit offsets)
    if (c->ld_page < 8 || c->ld_head < 8 || c->ld_tok < 8 || c->ld_page % 8 || c->ld_head % 8 ||
        c->ld_tok % 8 || c->ld_page > most || c->ld_head > most || c->ld_tok > most)
        return fail(S2X_ERR_INVALID_ARG, "%s: cache strides must be positive multiples of 8 below 2^31", who);
    const int64_t heads = (c->n_head - 1) * c->ld_head, toks = (ps - 1) * c->ld_tok;
    const bool by_tok = (c->n_head == 1 || c->ld_head >= c->d_head) &&
                        (ps == 1 || c->ld_tok >= heads + c->d_head);
    const bool by_head = (ps == 1 || c->ld_tok >= c->d_head) &&
                         (c->n_head == 1 || c->ld_head >= toks + c->d_head);
    if ((!by_tok && !by_head) || (c->n_pages > 1 && c->ld_page < heads + toks + c->d_head))
        return fail(S2X_ERR_INVALID_ARG, "%s: cache rows overlap", who);
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16))
        return fail(S2X_ERR_INVALID_ARG, "%s: k / v null or not 16-byte aligned", who);
    v = KvView{c->k, c->v, c->type, shift, c->n_pages, c->ld_page, c->ld_head, c->ld_tok,
               (int)c->n_head, (int)c->d_head};
    return S2X_OK;
}

}  // namespace s2x

using namespace s2x;

extern "C" {

// ---------------------------------------------------------------------------
// Q4_0 weights and products
// ---------------------------------------------------------------------------
size_t s2x_weight_q4_0_bytes(int64_t K, int64_t N) { return q4_shape_ok(K, N) ? q4_bytes(K, N) : 0; }

int s2x_weight_q4_0_create_in(const void *raw_dev, int64_t K, int64_t N, void *dev_buf, void *stream,
                              s2x_weight_q4 **out) {
    if (!out) return fail(S2X_ERR_INVALID_ARG, "weight_q4_0_create_in: out is null");
    *out = nullptr;
    if (!q4_shape_ok(K, N))
        return fail(S2X_ERR_INVALID_ARG, "weight_q4_0_create_in: bad shape K=%lld N=%lld", (long long)K,
                    (long long)N);
    if (!raw_dev || !dev_buf || !aligned(raw_dev, 2) || !aligned(dev_buf, 256))
        return fail(S2X_ERR_INVALID_ARG,
                    "weight_q4_0_create_in: raw must be 2-byte and dev_buf 256-byte aligned");
    s2x_weight_q4 *w = new (std::nothrow) s2x_weight_q4();
    if (!w) return fail(S2X_ERR_OOM, "weight_q4_0_create_in: out of host memory");
    w->mem = dev_buf;
    w->view = q4_view(dev_buf, K, N);
    const hipError_t e = launch_repack_q4_0(raw_dev, w->view, (hipStream_t)stream);
    if (e != hipSuccess) {
        delete w;
        return hip_fail(e, "q4_0 repack launch");
    }
    *out = w;
    return S2X_OK;
}

int s2x_weight_q4_0_create(const void *raw, int raw_is_host, int64_t K, int64_t N, void *stream,
                           s2x_weight_q4 **out) {
    if (!out) return fail(S2X_ERR_INVALID_ARG, "weight_q4_0_create: out is null");
    *out = nullptr;
    if (!q4_shape_ok(K, N) || !raw)
        return fail(S2X_ERR_INVALID_ARG, "weight_q4_0_create: raw null or bad shape K=%lld N=%lld",
                    (long long)K, (long long)N);
    if (!raw_is_host && !aligned(raw, 2))
        return fail(S2X_ERR_INVALID_ARG, "weight_q4_0_create: raw must be 2-byte aligned");
    const size_t raw_bytes = (size_t)(N * (K / QK_)) * 18;
    void *tmp = nullptr, *mem = nullptr;
    hipError_t e = hipSuccess;
    if (raw_is_host) {
        if (hipMalloc(&tmp, raw_bytes) != hipSuccess)
            return fail(S2X_ERR_OOM, "weight_q4_0_create: hipMalloc(%zu) failed", raw_bytes);
        // (a copy from pageable memory: done when it returns)
        e = hipMemcpy(tmp, raw, raw_bytes, hipMemcpyHostToDevice);
    }
    int st = e == hipSuccess ? S2X_OK : hip_fail(e, "weight_q4_0_create copy");
    if (st == S2X_OK && hipMalloc(&mem, q4_bytes(K, N)) != hipSuccess)
        st = fail(S2X_ERR_OOM, "weight_q4_0_create: hipMalloc of the planes failed");
    if (st == S2X_OK)
        st = s2x_weight_q4_0_create_in(raw_is_host ? tmp : raw, K, N, mem, stream, out);
    if (st == S2X_OK) {
        (*out)->owns = true;
        e = hipStreamSynchronize((hipStream_t)stream);
        if (e != hipSuccess) {
            s2x_weight_q4_0_destroy(*out);
            *out = nullptr;
            mem = nullptr;
            st = hip_fail(e, "weight_q4_0_create sync");
        }
    }
    if (st != S2X_OK && mem) (void)hipFree(mem);
    if (tmp) (void)hipFree(tmp);
    return st;
}

void s2x_weight_q4_0_destroy(s2x_weight_q4 *w) {
    if (!w) return;
    if (w->owns && w->mem) (void)hipFree(w->mem);
    delete w;
}
int64_t s2x_weight_q4_0_k(const s2x_weight_q4 *w) { return w ? w->view.K : 0; }
int64_t s2x_weight_q4_0_n(const s2x_weight_q4 *w) { return w ? w->view.N : 0; }

size_t s2x_mul_mat_q4_0_workspace_size(int64_t K, int64_t N, int64_t M) {
    if (!q4_shape_ok(K, N) || M <= S2X_Q4_FEW_ROWS) return 0;
    if (!gemm_in_reach(K, gemm_ld_dw(N), N, EpiParams{})) return 0;
    return weight_planes_bytes(K, N, gemm_ld_q(K));
}

int s2x_mul_mat_q4_0_q8_1(const s2x_weight_q4 *w, const void *qs, const void *ds, int64_t M, float *y,
                          int64_t ldy, const s2x_epilogue *epi, void *workspace, size_t ws_bytes,
                          void *stream) {
    const char *who = "mul_mat_q4_0_q8_1";
    if (!w) return fail(S2X_ERR_INVALID_ARG, "%s: weight is null", who);
    int st = check_q81_planes(qs, ds, M, who);
    if (st != S2X_OK) return st;
    const Q4View &v = w->view;
    EpiParams p;
    st = check_epi(epi, v.N, p);
    if (st != S2X_OK) return st;
    if (p.kind == EPI_GELU_Q81 || p.kind == EPI_GELU_F16)
        return fail(S2X_ERR_UNSUPPORTED, "%s: epilogue NONE, BIAS, BIAS_GELU or BIAS_RESID", who);
    if (!y || ldy < v.N || !aligned(y, 4))
        return fail(S2X_ERR_INVALID_ARG, "%s: y null/misaligned or ldy=%lld < N=%lld", who, (long long)ldy,
                    (long long)v.N);
    const size_t need = s2x_mul_mat_q4_0_workspace_size(v.K, v.N, M);
    if (need && (!workspace || !aligned(workspace, 256)))
        return fail(S2X_ERR_INVALID_ARG, "%s: workspace null or not 256-byte aligned", who);
    if (ws_bytes < need) return fail(S2X_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    if (M == 0) return S2X_OK;
    hipStream_t s = (hipStream_t)stream;
    hipError_t e;
    // (the few-rows form, whose offsets have 64 bits, takes what the GEMM cannot reach)
    if (M <= S2X_Q4_FEW_ROWS || !gemm_in_reach(v.K, gemm_ld_dw(v.N), ldy, p)) {
        e = launch_mul_mat_q4(v, (const int8_t *)qs, (const uint32_t *)ds, M, y, ldy, p, s);
    } else {
        const WeightView d = planes_view(workspace, v.K, v.N, gemm_ld_q(v.K));
        e = launch_expand_q4(v, d, s);
        if (e == hipSuccess)
            e = launch_gemm(d, (const int8_t *)qs, (const uint32_t *)ds, v.K / QK_, M, y, ldy, p, s);
    }
    return e == hipSuccess ? S2X_OK : hip_fail(e, "q4_0 product launch");
}

// ---------------------------------------------------------------------------
// paged cache
// ---------------------------------------------------------------------------
int s2x_kv_slots(const int32_t *kv_len, const int32_t *n_new, int64_t n_seq, const int32_t *free_pages,
                 int64_t n_free, int64_t page_size, int64_t n_pages, int32_t *block_table,
                 int64_t ld_table, int64_t max_tok, int32_t *len_out, int32_t *tok_start, int32_t *pos,
                 int64_t *slots, int64_t *used, void *stream) {
    if (n_seq < 0 || n_free < 0 || n_pages < 0 || ld_table < 0 || max_tok < 0)
        return fail(S2X_ERR_INVALID_ARG, "kv_slots: negative size");
    const int shift = log2_page(page_size);
    if (shift < 0 || n_seq > KV_MAX_SEQ || max_tok >= INT32_MAX || n_pages > INT32_MAX ||
        n_free > INT32_MAX || ld_table > INT32_MAX)
        return fail(S2X_ERR_UNSUPPORTED,
                    "kv_slots: page_size=%lld (a power of two up to 65,536), n_seq=%lld (<= %lld), "
                    "max_tok=%lld (31 bits)", (long long)page_size, (long long)n_seq,
                    (long long)KV_MAX_SEQ, (long long)max_tok);
    if ((n_seq && (!kv_len || !n_new || !len_out)) || (n_free && !free_pages) ||
        (n_seq && ld_table && !block_table) || (max_tok && (!pos || !slots)) || !tok_start || !used)
        return fail(S2X_ERR_INVALID_ARG, "kv_slots: null pointer");
    if (!aligned(kv_len, 4) || !aligned(n_new, 4) || !aligned(free_pages, 4) || !aligned(block_table, 4) ||
        !aligned(len_out, 4) || !aligned(tok_start, 4) || !aligned(pos, 4) || !aligned(slots, 8) ||
        !aligned(used, 8))
        return fail(S2X_ERR_INVALID_ARG, "kv_slots: misaligned pointer");
    // the workgroups read the lengths, and the table, while others write: no
    // output over them
    struct Range { const void *p; int64_t bytes; };
    const Range in[] = {{kv_len, 4 * n_seq}, {n_new, 4 * n_seq}, {free_pages, 4 * n_free}};
    const Range out[] = {{block_table, 4 * n_seq * ld_table}, {len_out, 4 * n_seq}, {tok_start, 4 * n_seq + 4},
                         {pos, 4 * max_tok}, {slots, 8 * max_tok}, {used, 16}};
    const auto meet = [](const Range &a, const Range &b) {
        const uintptr_t x = (uintptr_t)a.p, z = (uintptr_t)b.p;
        return a.bytes && b.bytes && x < z + (uintptr_t)b.bytes && z < x + (uintptr_t)a.bytes;
    };
    for (const Range &b : out) {
        for (const Range &a : in)
            if (meet(a, b)) return fail(S2X_ERR_INVALID_ARG, "kv_slots: an output overlaps an input");
        for (const Range *a = out; a != &b; ++a)
            if (meet(*a, b)) return fail(S2X_ERR_INVALID_ARG, "kv_slots: two outputs overlap");
    }
    const KvSlots p{kv_len, n_new, (int)n_seq, free_pages, n_free, shift, n_pages, block_table, ld_table,
                    max_tok, len_out, tok_start, pos, slots, used};
    const hipError_t e = launch_kv_slots(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "kv_slots launch");
}

int s2x_qk_norm_rope_kv(const void *x, int32_t x_type, int64_t ld_x, int64_t n_tok, int64_t n_q_head,
                        const float *q_norm, const float *k_norm, float eps, const double *freq,
                        int64_t d_rot, int32_t rope_style, const int32_t *pos, const int64_t *slots,
                        void *q, int64_t ld_q, const s2x_kv_cache *cache, void *stream) {
    const char *who = "qk_norm_rope_kv";
    KvView v;
    int st = check_cache(cache, v, who);
    if (st != S2X_OK) return st;
    int64_t size;
    if (!type_size(x_type, size)) return fail(S2X_ERR_INVALID_ARG, "%s: x_type %d", who, (int)x_type);
    if (rope_style != S2X_ROPE_HALVES && rope_style != S2X_ROPE_PAIRS)
        return fail(S2X_ERR_INVALID_ARG, "%s: rope_style %d", who, (int)rope_style);
    if (n_tok < 0 || n_q_head <= 0 || d_rot < 0 || d_rot % 2 || d_rot > v.d_head)
        return fail(S2X_ERR_INVALID_ARG, "%s: n_tok=%lld n_q_head=%lld d_rot=%lld", who, (long long)n_tok,
                    (long long)n_q_head, (long long)d_rot);
    if (n_tok > (1 << 23) || n_q_head > 1024)
        return fail(S2X_ERR_UNSUPPORTED, "%s: at most 2^23 rows and 1,024 query heads", who);
    if (ld_x < (n_q_head + 2 * v.n_head) * v.d_head || ld_x % 8 || ld_q < n_q_head * v.d_head || ld_q % 8)
        return fail(S2X_ERR_INVALID_ARG, "%s: ld_x=%lld / ld_q=%lld below the row or no multiple of 8", who,
                    (long long)ld_x, (long long)ld_q);
    if (n_tok == 0) return S2X_OK;
    if (!x || !q || !slots || (d_rot && (!pos || !freq)))
        return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(x, 16) || !aligned(q, 16) || !aligned(q_norm, 4) || !aligned(k_norm, 4) ||
        !aligned(freq, 8) || !aligned(pos, 4) || !aligned(slots, 8))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    const QkNormRope p{x, x_type, ld_x, n_tok, (int)n_q_head, q_norm, k_norm, eps, freq, (int)d_rot,
                       rope_style == S2X_ROPE_PAIRS, pos, slots, q, ld_q, v};
    const hipError_t e = launch_qk_norm_rope_kv(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "qk_norm_rope_kv launch");
}

static int check_paged_shape(const char *who, int64_t n_seq, int64_t max_len, int64_t n_q_head,
                             int64_t n_kv_head, int64_t d_head) {
    if (n_seq < 0 || max_len < 0 || n_q_head <= 0 || n_kv_head <= 0 || n_q_head % n_kv_head || d_head <= 0)
        return fail(S2X_ERR_INVALID_ARG, "%s: n_seq=%lld max_len=%lld, %lld query heads on %lld", who,
                    (long long)n_seq, (long long)max_len, (long long)n_q_head, (long long)n_kv_head);
    if (n_seq > 65535 || max_len > (1 << 30) || n_q_head > 1024 || d_head % 8 || d_head > 256)
        return fail(S2X_ERR_UNSUPPORTED,
                    "%s: n_seq <= 65,535, max_len <= 2^30, n_q_head <= 1,024, d_head %% 8 == 0 up to 256", who);
    if (n_seq * n_kv_head * ((n_q_head / n_kv_head + 15) / 16) > (1 << 22))
        return fail(S2X_ERR_UNSUPPORTED, "%s: at most 2^22 sequences x key heads (in 16 query heads each)", who);
    return S2X_OK;
}

size_t s2x_attn_paged_workspace_size(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head,
                                     int64_t d_head) {
    if (check_paged_shape("attn_paged", n_seq, max_len, n_q_head, n_kv_head, d_head) != S2X_OK) return 0;
    return attn_paged_workspace(n_seq, max_len, n_q_head, n_kv_head, d_head);
}

// (tok_start null: row s of q is sequence s's)
static int attn_paged(const char *who, const void *q, int64_t ld_q, int64_t n_row, const int32_t *tok_start,
                      const s2x_kv_cache *cache, const int32_t *block_table, int64_t ld_table,
                      const int32_t *kv_len, int64_t n_seq, int64_t max_len, int64_t n_q_head, float scale,
                      int64_t window, void *out, int32_t out_type, int64_t ld_out, float *lse,
                      void *workspace, size_t ws_bytes, void *stream) {
    KvView v;
    int st = check_cache(cache, v, who);
    if (st != S2X_OK) return st;
    st = check_paged_shape(who, n_seq, max_len, n_q_head, v.n_head, v.d_head);
    if (st != S2X_OK) return st;
    if (out_type != S2X_TYPE_F32 && out_type != v.type)
        return fail(S2X_ERR_UNSUPPORTED, "%s: out_type %d (F32 or the cache's type)", who, (int)out_type);
    if (window < 0 || ld_table < 0 || ld_table > INT32_MAX)
        return fail(S2X_ERR_INVALID_ARG, "%s: window=%lld ld_table=%lld", who, (long long)window,
                    (long long)ld_table);
    const int64_t H = n_q_head * v.d_head;
    if (ld_q < H || ld_q % 8 || ld_out < H || ld_out % 8)
        return fail(S2X_ERR_INVALID_ARG, "%s: ld_q=%lld / ld_out=%lld below the row or no multiple of 8", who,
                    (long long)ld_q, (long long)ld_out);
    if (n_seq == 0 || n_row == 0) return S2X_OK;
    if (!q || !kv_len || !out || (ld_table && max_len && !block_table))
        return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(block_table, 4) || !aligned(kv_len, 4) ||
        !aligned(lse, 4) || !aligned(tok_start, 4))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    const size_t need = attn_paged_workspace(n_seq, max_len, n_q_head, v.n_head, v.d_head);
    if (need && (!workspace || !aligned(workspace, 256)))
        return fail(S2X_ERR_INVALID_ARG, "%s: workspace null or not 256-byte aligned", who);
    if (ws_bytes < need) return fail(S2X_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    const AttnPaged p{q, ld_q, v, block_table, ld_table, kv_len, (int)n_seq, (int)max_len, (int)n_q_head,
                      (int)(window > INT32_MAX ? 0 : window), scale, out, out_type == S2X_TYPE_F32, ld_out,
                      lse, workspace, tok_start, n_row};
    const hipError_t e = launch_attn_paged(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "attn_paged launch");
}

int s2x_attn_paged(const void *q, int64_t ld_q, const s2x_kv_cache *cache, const int32_t *block_table,
                   int64_t ld_table, const int32_t *kv_len, int64_t n_seq, int64_t max_len,
                   int64_t n_q_head, float scale, int64_t window, void *out, int32_t out_type,
                   int64_t ld_out, float *lse, void *workspace, size_t ws_bytes, void *stream) {
    return attn_paged("attn_paged", q, ld_q, n_seq, nullptr, cache, block_table, ld_table, kv_len, n_seq, max_len,
                      n_q_head, scale, window, out, out_type, ld_out, lse, workspace, ws_bytes, stream);
}

int s2x_attn_paged_rows(const void *q, int64_t ld_q, int64_t n_row, const int32_t *tok_start,
                        const s2x_kv_cache *cache, const int32_t *block_table, int64_t ld_table,
                        const int32_t *kv_len, int64_t n_seq, int64_t max_len, int64_t n_q_head, float scale,
                        int64_t window, void *out, int32_t out_type, int64_t ld_out, float *lse,
                        void *workspace, size_t ws_bytes, void *stream) {
    if (n_row < 0) return fail(S2X_ERR_INVALID_ARG, "attn_paged_rows: n_row=%lld", (long long)n_row);
    if (!tok_start && n_seq > 0 && n_row > 0) return fail(S2X_ERR_INVALID_ARG, "attn_paged_rows: tok_start is null");
    return attn_paged("attn_paged_rows", q, ld_q, n_row, tok_start, cache, block_table, ld_table, kv_len, n_seq,
                      max_len, n_q_head, scale, window, out, out_type, ld_out, lse, workspace, ws_bytes, stream);
}

}  // extern "C"
