// s2x_decode.h -- host-side launchers of the decode step's kernels (internal).
//
// As in s2x_kernels.h: asynchronous on `stream`, nothing validated here (the
// C-ABI layer in s2x_decode.cpp does).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "s2x_kernels.h"

namespace s2x {

// element types (s2x_type)
enum ElemType { TY_F32 = 0, TY_F16 = 1, TY_BF16 = 2 };

// Most sequences of one slots call: its workgroups each hold the starts of
// all of them, 8 bytes a sequence, in LDS.
constexpr int64_t KV_MAX_SEQ = 8192;

struct KvSlots {
    const int32_t *kv_len, *n_new;
    int            n_seq;
    const int32_t *free_pages;
    int64_t        n_free;
    int            page_shift;  // log2 of the page size
    int64_t        n_pages;
    int32_t       *table;
    int64_t        ld_table, max_tok;
    int32_t       *len_out, *tok_start, *pos;
    int64_t       *slots, *used;
};
hipError_t launch_kv_slots(const KvSlots &p, hipStream_t stream);

// A paged cache as the kernels see it (elements, page size as its log2).
struct KvView {
    void   *k, *v;
    int     type, page_shift;
    int64_t n_pages, ld_page, ld_head, ld_tok;
    int     n_head, d_head;
};

struct QkNormRope {
    const void    *x;
    int            x_type;
    int64_t        ld_x, n_tok;
    int            n_q_head;
    const float   *q_norm, *k_norm;
    float          eps;
    const double  *freq;
    int            d_rot;
    bool           pairs;
    const int32_t *pos;
    const int64_t *slots;
    void          *q;
    int64_t        ld_q;
    KvView         kv;
};
hipError_t launch_qk_norm_rope_kv(const QkNormRope &p, hipStream_t stream);

// Attention of one query row per sequence over a paged cache.
struct AttnPaged {
    const void    *q;
    int64_t        ld_q;
    KvView         kv;
    const int32_t *table;
    int64_t        ld_table;
    const int32_t *kv_len;
    int            n_seq, max_len, n_q_head, window;  // window 0: all
    float          scale;
    void          *out;
    bool           out_f32;  // else the cache's type
    int64_t        ld_out;
    float         *lse;      // may be null
    void          *ws;
    const int32_t *tok_start;  // null: row s of q is sequence s's
    int64_t        n_row;      // rows of q, with tok_start
};
size_t attn_paged_workspace(int64_t n_seq, int64_t max_len, int64_t n_q_head, int64_t n_kv_head,
                            int64_t d_head);
hipError_t launch_attn_paged(const AttnPaged &p, hipStream_t stream);

// A Q4_0 weight (K, N) repacked for the int8 MFMA.  A tile is 16 columns n by
// 128 values of K (4 blocks), 1,024 bytes: lane l = 16 g + n % 16 has the 16
// bytes at 16 l, word j of them 8 values of the tile's block j, from 16 (g & 1)
// + 8 (g >> 1) on, the first 4 in the low halves of its bytes, the others in
// the high ones, nibbles in two's complement (v - 8).  Tiles of one column group follow each other along
// K.  Scales: per tile 64 halves, [j][c] of block j and column c.
// Columns past N and blocks past K / 32 are zeros.
struct Q4View {
    const uint8_t  *qs;
    const uint16_t *d;
    int64_t         K, N;
    int64_t tiles_k() const { return (K + 127) / 128; }
    int64_t tiles_n() const { return (N + 15) / 16; }
};
hipError_t launch_repack_q4_0(const void *raw, const Q4View &w, hipStream_t stream);
// y = epilogue (NONE, BIAS, BIAS_GELU, BIAS_RESID), xq [M][K], xds [M][K / 32];
// any M, made for few rows
hipError_t launch_mul_mat_q4(const Q4View &w, const int8_t *xq, const uint32_t *xds, int64_t M, float *y,
                             int64_t ldy, const EpiParams &epi, hipStream_t stream);
// the same weight as Q8_0 planes (rows of dst.ld_qs bytes, transposed scales)
hipError_t launch_expand_q4(const Q4View &w, const WeightView &dst, hipStream_t stream);

}  // namespace s2x
