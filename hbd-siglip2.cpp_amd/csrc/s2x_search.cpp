// s2x_search.cpp -- the extern "C" boundary of a beam search over a paged cache
// (include/s2x.h): argument checks and status codes of the residual RMS norm with
// Q8_1, the beam selection, the cache's pages and the attention over a prefix.
#include "s2x_search.h"

#include <climits>
#include <cmath>

#include "s2x.h"
#include "s2x_internal.h"

namespace s2x {

struct Span {
    const void *p;
    int64_t     bytes;
    int64_t     row = 0, pitch = 0;  // bytes of a row, and from one to the next (0: all one)
};
static bool meet(const Span &a, const Span &b) {
    const uintptr_t x = (uintptr_t)a.p, z = (uintptr_t)b.p;
    if (!a.p || !b.p || !a.bytes || !b.bytes || x >= z + (uintptr_t)b.bytes || z >= x + (uintptr_t)a.bytes) return false;
    if (a.pitch && a.pitch == b.pitch) {  // rows of one buffer: b's between a's
        const int64_t d = ((int64_t)(z - x) % a.pitch + a.pitch) % a.pitch;
        if (d >= a.row && d + b.row <= a.pitch) return false;
    }
    return true;
}
// rows `ld` apart of which `n` elements of `size` bytes count
static Span rows_of(const void *p, int64_t rows, int64_t ld, int64_t n, int64_t size) {
    return Span{p, rows > 0 ? ((rows - 1) * ld + n) * size : 0, n * size, rows > 1 ? ld * size : 0};
}
template <int NI, int NO>
static const char *overlap(const Span (&in)[NI], const Span (&out)[NO]) {
    for (const Span &o : out) {
        for (const Span &i : in)
            if (meet(i, o)) return "an output overlaps an input";
        for (const Span *q = out; q != &o; ++q)
            if (meet(*q, o)) return "two outputs overlap";
    }
    return nullptr;
}

}  // namespace s2x

using namespace s2x;

extern "C" {

// ---------------------------------------------------------------------------
// residual, RMS norm, Q8_1
// ---------------------------------------------------------------------------
int s2x_add_rmsnorm_quantize_q8_1(const void *x, int32_t x_type, int64_t ld_x, const void *resid,
                                  int32_t resid_type, int64_t ld_resid, int64_t H, int64_t M,
                                  const float *w, float eps, void *h_out, int64_t ld_h, int64_t K_pad,
                                  void *qs, void *ds, void *y, int32_t y_type, int64_t ld_y, void *stream) {
    const char *who = "add_rmsnorm_quantize_q8_1";
    int64_t sx, sr, sy;
    if (!type_size(x_type, sx) || !type_size(resid_type, sr) || !type_size(y_type, sy))
        return fail(S2X_ERR_INVALID_ARG, "%s: x_type %d, resid_type %d, y_type %d", who, (int)x_type, (int)resid_type,
                    (int)y_type);
    if (resid_type != S2X_TYPE_F32 && resid_type != x_type)
        return fail(S2X_ERR_UNSUPPORTED, "%s: resid_type %d (F32 or x's type)", who, (int)resid_type);
    if (H <= 0 || M < 0) return fail(S2X_ERR_INVALID_ARG, "%s: H=%lld M=%lld", who, (long long)H, (long long)M);
    if (H > RMS_MAX_H || M > (1 << 30))
        return fail(S2X_ERR_UNSUPPORTED, "%s: H <= %lld and M <= 2^30", who, (long long)RMS_MAX_H);
    if ((qs == nullptr) != (ds == nullptr) || (!qs && !y && M > 0))
        return fail(S2X_ERR_INVALID_ARG, "%s: qs and ds, y, or all three", who);
    if (qs && (K_pad % QK_ || K_pad < H || K_pad - H >= QK_))
        return fail(S2X_ERR_INVALID_ARG, "%s: K_pad=%lld for H=%lld", who, (long long)K_pad, (long long)H);
    if (ld_x < H || (resid && ld_resid < H) || (h_out && ld_h < H) || (y && ld_y < H))
        return fail(S2X_ERR_INVALID_ARG, "%s: a row stride below H=%lld", who, (long long)H);
    const int64_t far = (int64_t)1 << 32;  // (offsets then stay within 64 bits)
    if (ld_x > far || (resid && ld_resid > far) || (h_out && ld_h > far) || (y && ld_y > far))
        return fail(S2X_ERR_UNSUPPORTED, "%s: a row stride above 2^32", who);
    if (M == 0) return S2X_OK;
    if (!x) return fail(S2X_ERR_INVALID_ARG, "%s: x is null", who);
    if (!aligned(x, sx) || !aligned(resid, sr) || !aligned(h_out, sr) || !aligned(w, 4) || !aligned(y, sy) ||
        !aligned(qs, 16) || !aligned(ds, 4))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer (qs: 16 bytes)", who);
    // rows are read whole before they are written: h_out may be resid or x, row for row
    const Span rx = rows_of(x, M, ld_x, H, sx), rr = rows_of(resid, M, ld_resid, H, sr), rw{w, 4 * H};
    const Span oh = rows_of(h_out, M, ld_h, H, sr), oy = rows_of(y, M, ld_y, H, sy);
    const Span oq{qs, M * K_pad}, od{ds, M * (K_pad / QK_) * 4};
    const bool h_is_x = h_out == x && ld_h == ld_x && resid_type == x_type, h_is_r = h_out == resid && ld_h == ld_resid;
    const Span none{nullptr, 0};
    const Span in[] = {rx, rr, rw}, in_h[] = {h_is_x ? none : rx, h_is_r ? none : rr, rw};
    const Span out[] = {oy, oq, od}, out_h[] = {oh}, in_o[] = {oh};
    const char *bad = overlap(in, out);
    if (!bad) bad = overlap(in_h, out_h);
    if (!bad && overlap(in_o, out)) bad = "two outputs overlap";
    if (bad) return fail(S2X_ERR_INVALID_ARG, "%s: %s", who, bad);
    const AddRmsNorm p{x, resid, h_out, w, y, (int8_t *)qs, (uint32_t *)ds, ld_x, ld_resid, ld_h, ld_y, M,
                       x_type, resid_type, y_type, (int)H, (int)K_pad, eps};
    const hipError_t e = launch_add_rmsnorm(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "add_rmsnorm launch");
}

// ---------------------------------------------------------------------------
// beam selection
// ---------------------------------------------------------------------------
static int check_beam(const char *who, int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out) {
    if (n_req < 0 || n_beam <= 0 || n_vocab <= 0 || n_out <= 0)
        return fail(S2X_ERR_INVALID_ARG, "%s: n_req=%lld n_beam=%lld n_vocab=%lld n_out=%lld", who, (long long)n_req,
                    (long long)n_beam, (long long)n_vocab, (long long)n_out);
    if (n_beam > BEAM_MAX_OUT || n_out > BEAM_MAX_OUT || n_vocab > (1 << 24) || n_req > 65535 || n_req * n_beam > 65535)
        return fail(S2X_ERR_UNSUPPORTED, "%s: n_beam and n_out <= %d, n_req * n_beam <= 65,535, n_vocab <= 2^24", who,
                    BEAM_MAX_OUT);
    return S2X_OK;
}

size_t s2x_beam_select_workspace_size(int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out) {
    if (check_beam("beam_select", n_req, n_beam, n_vocab, n_out) != S2X_OK) return 0;
    return beam_select_workspace(n_req, n_beam, n_vocab, n_out);
}

int s2x_beam_select(const void *logits, int32_t type, int64_t ld, int64_t n_req, int64_t n_beam, int64_t n_vocab,
                    const float *scores, const uint8_t *done, int32_t done_token, int64_t n_out, int32_t *parent,
                    int32_t *token, float *score, void *workspace, size_t ws_bytes, void *stream) {
    const char *who = "beam_select";
    int st = check_beam(who, n_req, n_beam, n_vocab, n_out);
    if (st != S2X_OK) return st;
    int64_t size;
    if (!type_size(type, size)) return fail(S2X_ERR_INVALID_ARG, "%s: type %d", who, (int)type);
    if (ld < n_vocab || ld > (int64_t)1 << 32)
        return fail(S2X_ERR_INVALID_ARG, "%s: ld=%lld for n_vocab=%lld", who, (long long)ld, (long long)n_vocab);
    if (n_req == 0) return S2X_OK;
    if (!logits || !scores || !parent || !token || !score) return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(logits, size) || !aligned(scores, 4) || !aligned(parent, 4) || !aligned(token, 4) || !aligned(score, 4))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    const size_t need = beam_select_workspace(n_req, n_beam, n_vocab, n_out);
    if (!workspace || !aligned(workspace, 256))
        return fail(S2X_ERR_INVALID_ARG, "%s: workspace null or not 256-byte aligned", who);
    if (ws_bytes < need) return fail(S2X_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    const int64_t rows = n_req * n_beam;
    const Span in[] = {rows_of(logits, rows, ld, n_vocab, size), Span{scores, 4 * rows}, Span{done, rows}};
    const Span out[] = {Span{parent, 4 * n_req * n_out}, Span{token, 4 * n_req * n_out}, Span{score, 4 * n_req * n_out},
                        Span{workspace, (int64_t)need}};
    if (const char *bad = overlap(in, out)) return fail(S2X_ERR_INVALID_ARG, "%s: %s", who, bad);
    const BeamSelect p{logits, type, ld, (int)n_req, (int)n_beam, (int)n_vocab, scores, done, done_token, (int)n_out,
                       parent, token, score, workspace};
    const hipError_t e = launch_beam_select(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "beam_select launch");
}

// ---------------------------------------------------------------------------
// pages
// ---------------------------------------------------------------------------
static int check_pages(const char *who, int64_t n_out, int64_t n_seq, int64_t ld_table, int64_t page_size,
                       int64_t n_pages, int64_t ld_out, int &shift) {
    if (n_out < 0 || n_seq < 0 || ld_table < 0 || n_pages < 0 || ld_out < ld_table)
        return fail(S2X_ERR_INVALID_ARG, "%s: %lld of %lld sequences, ld_table=%lld, ld_out=%lld, %lld pages", who,
                    (long long)n_out, (long long)n_seq, (long long)ld_table, (long long)ld_out, (long long)n_pages);
    shift = log2_page(page_size);
    if (shift < 0 || n_out > KV_MAX_SEQ || n_seq > KV_MAX_SEQ || n_pages > (1 << 24) || ld_out > INT32_MAX)
        return fail(S2X_ERR_UNSUPPORTED,
                    "%s: page_size=%lld (a power of two up to 65,536), at most %lld sequences and 2^24 pages, table "
                    "rows of 31 bits", who, (long long)page_size, (long long)KV_MAX_SEQ);
    return S2X_OK;
}
static int check_pages_ws(const char *who, int64_t n_pages, const void *ws, size_t ws_bytes) {
    const size_t need = kv_pages_workspace(n_pages);
    if (!ws || !aligned(ws, 256)) return fail(S2X_ERR_INVALID_ARG, "%s: workspace null or not 256-byte aligned", who);
    if (ws_bytes < need) return fail(S2X_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    return S2X_OK;
}

size_t s2x_kv_pages_workspace_size(int64_t n_pages) {
    return n_pages >= 0 && n_pages <= (1 << 24) ? kv_pages_workspace(n_pages) : 0;
}

int s2x_kv_fork(const int32_t *parent, int64_t n_out, const int32_t *kv_len, const int32_t *block_table, int64_t n_seq,
                int64_t ld_table, int64_t page_size, int64_t n_pages, const uint8_t *pinned, int32_t *table_out,
                int64_t ld_out, int32_t *len_out, int32_t *copy_src, int32_t *copy_dst, int32_t *copy_tok,
                int32_t *free_out, int64_t *count, void *workspace, size_t ws_bytes, void *stream) {
    const char *who = "kv_fork";
    int shift, st = check_pages(who, n_out, n_seq, ld_table, page_size, n_pages, ld_out, shift);
    if (st != S2X_OK) return st;
    if ((n_out && (!parent || !len_out || !copy_src || !copy_dst || !copy_tok)) || (n_out && ld_out && !table_out) ||
        (n_seq && (!kv_len || (ld_table && !block_table))) || (n_pages && !free_out) || !count)
        return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(parent, 4) || !aligned(kv_len, 4) || !aligned(block_table, 4) || !aligned(table_out, 4) ||
        !aligned(len_out, 4) || !aligned(copy_src, 4) || !aligned(copy_dst, 4) || !aligned(copy_tok, 4) ||
        !aligned(free_out, 4) || !aligned(count, 8))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    st = check_pages_ws(who, n_pages, workspace, ws_bytes);
    if (st != S2X_OK) return st;
    const Span in[] = {Span{parent, 4 * n_out}, Span{kv_len, 4 * n_seq}, Span{block_table, 4 * n_seq * ld_table},
                       Span{pinned, n_pages}};
    const Span out[] = {Span{table_out, 4 * n_out * ld_out}, Span{len_out, 4 * n_out}, Span{copy_src, 4 * n_out},
                        Span{copy_dst, 4 * n_out}, Span{copy_tok, 4 * n_out}, Span{free_out, 4 * n_pages}, Span{count, 16},
                        Span{workspace, (int64_t)kv_pages_workspace(n_pages)}};
    if (const char *bad = overlap(in, out)) return fail(S2X_ERR_INVALID_ARG, "%s: %s", who, bad);
    const KvPages p{parent, pinned, kv_len, block_table, (int)n_out, (int)n_seq, ld_table, ld_out, shift, n_pages,
                    table_out, len_out, copy_src, copy_dst, copy_tok, free_out, count, workspace};
    const hipError_t e = launch_kv_fork(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "kv_fork launch");
}

int s2x_kv_compact(const int32_t *kv_len, const int32_t *block_table, int64_t n_seq, int64_t ld_table, int64_t page_size,
                   int64_t n_pages, int32_t *table_out, int64_t ld_out, int32_t *copy_src, int32_t *copy_dst,
                   int64_t *count, void *workspace, size_t ws_bytes, void *stream) {
    const char *who = "kv_compact";
    int shift, st = check_pages(who, n_seq, n_seq, ld_table, page_size, n_pages, ld_out, shift);
    if (st != S2X_OK) return st;
    if ((n_seq && (!kv_len || (ld_table && !block_table) || (ld_out && !table_out))) ||
        (n_pages > 1 && (!copy_src || !copy_dst)) || !count)
        return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(kv_len, 4) || !aligned(block_table, 4) || !aligned(table_out, 4) || !aligned(copy_src, 4) ||
        !aligned(copy_dst, 4) || !aligned(count, 8))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    st = check_pages_ws(who, n_pages, workspace, ws_bytes);
    if (st != S2X_OK) return st;
    const Span in[] = {Span{kv_len, 4 * n_seq}, Span{block_table, 4 * n_seq * ld_table}};
    const Span out[] = {Span{table_out, 4 * n_seq * ld_out}, Span{copy_src, 4 * (n_pages / 2)},
                        Span{copy_dst, 4 * (n_pages / 2)}, Span{count, 16},
                        Span{workspace, (int64_t)kv_pages_workspace(n_pages)}};
    if (const char *bad = overlap(in, out)) return fail(S2X_ERR_INVALID_ARG, "%s: %s", who, bad);
    const KvPages p{nullptr, nullptr, kv_len, block_table, (int)n_seq, (int)n_seq, ld_table, ld_out, shift, n_pages,
                    table_out, nullptr, copy_src, copy_dst, nullptr, nullptr, count, workspace};
    const hipError_t e = launch_kv_compact(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "kv_compact launch");
}

int s2x_kv_copy_pages(const s2x_kv_cache *caches, int64_t n_cache, const int32_t *src, const int32_t *dst,
                      const int32_t *n_tok, int64_t n, const int64_t *n_dev, void *stream) {
    const char *who = "kv_copy_pages";
    if (n_cache < 0 || n < 0)
        return fail(S2X_ERR_INVALID_ARG, "%s: n_cache=%lld n=%lld", who, (long long)n_cache, (long long)n);
    if (n > (1 << 24) || n_cache > (1 << 20))
        return fail(S2X_ERR_UNSUPPORTED, "%s: at most 2^24 pages and 2^20 caches", who);
    if (n_cache == 0) return S2X_OK;
    if (!caches) return fail(S2X_ERR_INVALID_ARG, "%s: caches is null", who);
    KvView v, u;
    int st = check_cache(caches, v, who);
    if (st != S2X_OK) return st;
    for (int64_t i = 1; i < n_cache; ++i) {
        st = check_cache(caches + i, u, who);
        if (st != S2X_OK) return st;
        if (u.type != v.type || u.page_shift != v.page_shift || u.n_pages != v.n_pages || u.n_head != v.n_head ||
            u.d_head != v.d_head || u.ld_page != v.ld_page || u.ld_head != v.ld_head || u.ld_tok != v.ld_tok)
            return fail(S2X_ERR_INVALID_ARG, "%s: cache %lld is laid out unlike the first", who, (long long)i);
    }
    if (n == 0) return S2X_OK;
    if (!src || !dst) return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(n_tok, 4) || !aligned(n_dev, 8))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    for (int64_t i = 0; i < n_cache; i += KV_COPY_CACHES) {
        KvCopy p{};
        p.n_cache = (int)(n_cache - i < KV_COPY_CACHES ? n_cache - i : KV_COPY_CACHES);
        for (int k = 0; k < p.n_cache; ++k) {
            p.c[k].k = caches[i + k].k;
            p.c[k].v = caches[i + k].v;
        }
        p.kv = v;
        p.src = src, p.dst = dst, p.n_tok = n_tok, p.n_dev = n_dev, p.n = n;
        const hipError_t e = launch_kv_copy(p, (hipStream_t)stream);
        if (e != hipSuccess) return hip_fail(e, "kv_copy_pages launch");
    }
    return S2X_OK;
}

// ---------------------------------------------------------------------------
// attention over a shared prefix
// ---------------------------------------------------------------------------
static int check_prefix(const char *who, int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own,
                        int64_t n_q_head, int64_t n_kv_head, int64_t d_head) {
    if (n_group < 0 || max_group < 0 || max_prefix < 0 || max_own < 0 || n_q_head <= 0 || n_kv_head <= 0 ||
        n_q_head % n_kv_head || d_head <= 0)
        return fail(S2X_ERR_INVALID_ARG, "%s: %lld groups of at most %lld, max_prefix=%lld max_own=%lld, %lld query heads on %lld",
                    who, (long long)n_group, (long long)max_group, (long long)max_prefix, (long long)max_own,
                    (long long)n_q_head, (long long)n_kv_head);
    if (n_group > 65535 || max_group > 65535 || n_group * max_group > 65535 || max_prefix > (1 << 30) ||
        max_own > (1 << 30) || n_q_head > 1024 || d_head % 8 || d_head > 256)
        return fail(S2X_ERR_UNSUPPORTED,
                    "%s: n_group * max_group <= 65,535, max_prefix and max_own <= 2^30, n_q_head <= 1,024, d_head %% 8 == 0 "
                    "up to 256", who);
    if (n_group * max_group * n_kv_head * ((n_q_head / n_kv_head + 15) / 16) > (1 << 21))
        return fail(S2X_ERR_UNSUPPORTED, "%s: at most 2^21 sequences x key heads (in 16 query heads each)", who);
    return S2X_OK;
}

size_t s2x_attn_paged_prefix_workspace_size(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own,
                                            int64_t n_q_head, int64_t n_kv_head, int64_t d_head) {
    if (check_prefix("attn_paged_prefix", n_group, max_group, max_prefix, max_own, n_q_head, n_kv_head, d_head) != S2X_OK ||
        n_group == 0 || max_group == 0)
        return 0;
    return attn_prefix_workspace(n_group, max_group, max_prefix, max_own, n_q_head, n_kv_head, d_head);
}

int s2x_attn_paged_prefix(const void *q, int64_t ld_q, int64_t n_row, const int32_t *tok_start, const s2x_kv_cache *cache,
                          const int32_t *block_table, int64_t ld_table, const int32_t *kv_len, int64_t n_seq,
                          const int32_t *group_start, const int32_t *prefix_len, int64_t n_group, int64_t max_group,
                          int64_t max_prefix, int64_t max_own, int64_t n_q_head, float scale, void *out, int32_t out_type,
                          int64_t ld_out, float *lse, void *workspace, size_t ws_bytes, void *stream) {
    const char *who = "attn_paged_prefix";
    KvView v;
    int st = check_cache(cache, v, who);
    if (st != S2X_OK) return st;
    st = check_prefix(who, n_group, max_group, max_prefix, max_own, n_q_head, v.n_head, v.d_head);
    if (st != S2X_OK) return st;
    if (n_seq < 0 || n_row < 0 || n_row > INT32_MAX)
        return fail(S2X_ERR_INVALID_ARG, "%s: n_seq=%lld n_row=%lld", who, (long long)n_seq, (long long)n_row);
    if (n_seq > 65535 || n_seq * v.n_head * ((n_q_head / v.n_head + 15) / 16) > (1 << 21))
        return fail(S2X_ERR_UNSUPPORTED, "%s: at most 65,535 sequences, 2^21 x key heads (in 16 query heads each)", who);
    if (out_type != S2X_TYPE_F32 && out_type != v.type)
        return fail(S2X_ERR_UNSUPPORTED, "%s: out_type %d (F32 or the cache's type)", who, (int)out_type);
    if (ld_table < 0 || ld_table > INT32_MAX)
        return fail(S2X_ERR_INVALID_ARG, "%s: ld_table=%lld", who, (long long)ld_table);
    const int64_t H = n_q_head * v.d_head;
    if (ld_q < H || ld_q % 8 || ld_out < H || ld_out % 8 || ld_q > INT32_MAX || ld_out > INT32_MAX)
        return fail(S2X_ERR_INVALID_ARG, "%s: ld_q=%lld / ld_out=%lld below the row or no multiple of 8 within 31 bits", who,
                    (long long)ld_q, (long long)ld_out);
    if (n_seq == 0 || n_row == 0 || n_group == 0 || max_group == 0) return S2X_OK;
    if (!q || !kv_len || !out || !group_start || !prefix_len || (ld_table && (max_prefix || max_own) && !block_table))
        return fail(S2X_ERR_INVALID_ARG, "%s: null pointer", who);
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(block_table, 4) || !aligned(kv_len, 4) || !aligned(lse, 4) ||
        !aligned(tok_start, 4) || !aligned(group_start, 4) || !aligned(prefix_len, 4))
        return fail(S2X_ERR_INVALID_ARG, "%s: misaligned pointer", who);
    const size_t need = attn_prefix_workspace(n_group, max_group, max_prefix, max_own, n_q_head, v.n_head, v.d_head);
    if (!workspace || !aligned(workspace, 256))
        return fail(S2X_ERR_INVALID_ARG, "%s: workspace null or not 256-byte aligned", who);
    if (ws_bytes < need) return fail(S2X_ERR_WORKSPACE, "%s: workspace %zu < %zu bytes", who, ws_bytes, need);
    AttnPrefix p{};
    p.a = AttnPaged{q, ld_q, v, block_table, ld_table, kv_len, (int)n_seq, 0, (int)n_q_head, 0, scale, out,
                    out_type == S2X_TYPE_F32, ld_out, lse, workspace, tok_start, n_row};
    p.group_start = group_start, p.prefix_len = prefix_len;
    p.n_group = (int)n_group, p.max_group = (int)max_group, p.max_prefix = (int)max_prefix, p.max_own = (int)max_own;
    const hipError_t e = launch_attn_prefix(p, (hipStream_t)stream);
    return e == hipSuccess ? S2X_OK : hip_fail(e, "attn_paged_prefix launch");
}

}  // extern "C"
