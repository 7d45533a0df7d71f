// s2x_search.h -- host-side launchers of the kernels of a beam search over a
// paged cache (internal).
//
// As in s2x_kernels.h: asynchronous on `stream`, nothing validated here (the
// C-ABI layer in s2x_search.cpp does).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "s2x_decode.h"

namespace s2x {

// h = x + resid, y = h / sqrt(mean(h^2) + eps) * w, y to Q8_1 and / or rows.
struct AddRmsNorm {
    const void  *x;
    const void  *resid;  // may be null
    void        *h_out;  // may be null; resid's type
    const float *w;      // may be null
    void        *y;      // may be null
    int8_t      *qs;     // null: no Q8_1
    uint32_t    *ds;
    int64_t      ld_x, ld_resid, ld_h, ld_y, M;
    int          x_type, r_type, y_type, H, K_pad;
    float        eps;
};
constexpr int64_t RMS_MAX_H = 32768;
hipError_t launch_add_rmsnorm(const AddRmsNorm &p, hipStream_t stream);

// The n_out best continuations of each request's beams.
struct BeamSelect {
    const void    *logits;
    int            type;
    int64_t        ld;
    int            n_req, n_beam, n_vocab;
    const float   *scores;
    const uint8_t *done;  // may be null
    int            done_token, n_out;
    int32_t       *parent, *token;
    float         *score;
    void          *ws;
};
constexpr int BEAM_MAX_OUT = 64;
size_t beam_select_workspace(int64_t n_req, int64_t n_beam, int64_t n_vocab, int64_t n_out);
hipError_t launch_beam_select(const BeamSelect &p, hipStream_t stream);

// Block tables in a new order, with copies of open pages that several hold.
struct KvPages {
    const int32_t *parent;  // fork
    const uint8_t *pinned;  // fork; may be null
    const int32_t *kv_len, *table;
    int            n_out, n_seq;  // rows of table_out and of table (compact: the same)
    int64_t        ld_table, ld_out;
    int            page_shift;
    int64_t        n_pages;
    int32_t       *table_out, *len_out, *copy_src, *copy_dst, *copy_tok, *free_out;
    int64_t       *count;
    void          *ws;
};
size_t kv_pages_workspace(int64_t n_pages);
hipError_t launch_kv_fork(const KvPages &p, hipStream_t stream);
hipError_t launch_kv_compact(const KvPages &p, hipStream_t stream);

// Pages copied within each of several caches of one layout.
constexpr int KV_COPY_CACHES = 64;  // of one launch
struct KvCopy {
    struct { void *k, *v; } c[KV_COPY_CACHES];
    int            n_cache;
    KvView         kv;  // the layout
    const int32_t *src, *dst, *n_tok;  // n_tok may be null: whole pages
    const int64_t *n_dev;              // may be null: n
    int64_t        n;
};
hipError_t launch_kv_copy(const KvCopy &p, hipStream_t stream);

// Attention of sequences in groups that share their first tokens.
struct AttnPrefix {
    AttnPaged      a;  // (window 0; a.max_len is not used)
    const int32_t *group_start, *prefix_len;
    int            n_group, max_group, max_prefix, max_own;
};
size_t attn_prefix_workspace(int64_t n_group, int64_t max_group, int64_t max_prefix, int64_t max_own,
                             int64_t n_q_head, int64_t n_kv_head, int64_t d_head);
hipError_t launch_attn_prefix(const AttnPrefix &p, hipStream_t stream);

}  // namespace s2x
