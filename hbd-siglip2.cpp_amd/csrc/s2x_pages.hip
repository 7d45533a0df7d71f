// s2x_pages.hip -- pages of a cache: block tables in a new order with the copies
// that it takes (fork), the held pages moved to the front (compact), and the
// copying itself.
//
// Which pages are held follows from the tables alone, so no count of holders is
// kept between calls: a word a page takes the smallest of the marks that the rows
// leave there, whatever their order -- 0 where a row (or the caller's pin) holds
// the page as one that is not written to any more, 1 + i where it is row i's open
// last page.  So a page left at 1 + i is open to row i and to no other holder but
// later rows with it open, which get copies.
#include "s2x_device.h"
#include "s2x_search.h"

namespace s2x {

constexpr int KP_NT = 1024, KP_TILE = 4 * KP_NT;  // pages of a workgroup's tile
constexpr uint32_t KP_FREE = 0xffffffffu;

// Workspace: marks, the tiles' counts, the rows that get copies and their number
// (fork) or the moved pages' ranks (compact).
struct KpWs {
    uint32_t *mark;
    int32_t  *tile, *list;
    int       tiles;
};
static __host__ __device__ inline int kp_tiles(int64_t n_pages) { return (int)((n_pages + KP_TILE - 1) / KP_TILE); }
static __host__ __device__ inline KpWs kp_ws(const KvPages &p) {
    KpWs w;
    w.tiles = kp_tiles(p.n_pages);
    w.mark = (uint32_t *)p.ws;
    w.tile = (int32_t *)(w.mark + p.n_pages);
    w.list = w.tile + w.tiles + 1;
    return w;
}
size_t kv_pages_workspace(int64_t n_pages) {
    const int64_t list = n_pages > KV_MAX_SEQ ? n_pages : KV_MAX_SEQ;
    return (size_t)(n_pages + kp_tiles(n_pages) + 1 + list) * 4;
}

// Sum over the workgroup's KP_NT threads in every thread, and the sum before
// this one.
__device__ __forceinline__ int kp_scan(int v, int &total, int32_t *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int in = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const int t = __shfl_up(in, o);
        if (lane >= o) in += t;
    }
    __syncthreads();  // (sums of an earlier call are read)
    if (lane == WAVE - 1) sums[wave] = in;
    __syncthreads();
    int before = in - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < KP_NT / WAVE; ++w) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return before;
}

__device__ __forceinline__ int64_t kp_have(const KvPages &p, int len) {  // entries of a row of `len` tokens
    return min(((int64_t)len + (1 << p.page_shift) - 1) >> p.page_shift, p.ld_table);
}

template <bool FORK>
__global__ __launch_bounds__(256) void k_pages_clear(KvPages p) {
    const KpWs w = kp_ws(p);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < p.n_pages) w.mark[i] = FORK && p.pinned && p.pinned[i] ? 0u : FORK ? KP_FREE : 0u;
}

// Row i's table and marks.  An open page: the row's last one, where it has room
// and lies in the table.
struct KpRow {
    int     src, len;
    int64_t have;  // entries
    bool    open;
};
__device__ __forceinline__ KpRow kp_row(const KvPages &p, int i) {
    KpRow r;
    r.src = p.parent[i];
    r.len = r.src >= 0 && r.src < p.n_seq ? max(p.kv_len[r.src], 0) : 0;
    r.have = kp_have(p, r.len);
    r.open = (r.len & ((1 << p.page_shift) - 1)) != 0 && r.have << p.page_shift >= r.len;
    return r;
}
__device__ __forceinline__ int kp_entry(const KvPages &p, int row, int64_t j) {
    const int id = p.table[(int64_t)row * p.ld_table + j];
    return id >= 0 && id < p.n_pages ? id : -1;
}

__global__ __launch_bounds__(256) void k_fork_mark(KvPages p) {
    const KpWs w = kp_ws(p);
    const int i = blockIdx.y;
    const KpRow r = kp_row(p, i);
    if (blockIdx.x == 0 && threadIdx.x == 0) p.len_out[i] = r.len;
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < p.ld_out; j += (int64_t)gridDim.x * 256) {
        int id = -1;
        if (j < r.have) {
            id = kp_entry(p, r.src, j);
            if (id >= 0) atomicMin(&w.mark[id], r.open && j == r.have - 1 ? 1u + i : 0u);
        }
        p.table_out[(int64_t)i * p.ld_out + j] = id;
    }
}

// Tiles' counts of free pages (fork) or held ones (compact); fork's last
// workgroup: which rows get a copy, in order.
template <bool FORK>
__global__ __launch_bounds__(KP_NT) void k_pages_count(KvPages p) {
    __shared__ int32_t sums[KP_NT / WAVE];
    const KpWs w = kp_ws(p);
    int total;
    if (!FORK || (int)blockIdx.x < w.tiles) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t i = (int64_t)blockIdx.x * KP_TILE + k * KP_NT + threadIdx.x;
            if (i < p.n_pages) n += w.mark[i] == (FORK ? KP_FREE : 1u);
        }
        kp_scan(n, total, sums);
        if (threadIdx.x == 0) w.tile[blockIdx.x] = total;
        return;
    }
    int base = 0;
    for (int i0 = 0; i0 < p.n_out; i0 += KP_NT) {
        const int i = i0 + threadIdx.x;
        int last = -1;
        KpRow r = {};
        if (i < p.n_out) {
            r = kp_row(p, i);
            if (r.open) last = kp_entry(p, r.src, r.have - 1);
        }
        const bool want = last >= 0 && w.mark[last] != 1u + i;
        const int at = base + kp_scan(want, total, sums);
        base += total;
        if (i >= p.n_out) continue;
        p.copy_src[i] = want ? last : -1;
        p.copy_dst[i] = -1;
        p.copy_tok[i] = want ? r.len & ((1 << p.page_shift) - 1) : 0;
        if (want) {
            p.table_out[(int64_t)i * p.ld_out + r.have - 1] = -1;  // (until it gets its page)
            w.list[at] = i;
        }
    }
    if (threadIdx.x == 0) w.tile[w.tiles] = base;
}

// Counts of the tiles before this one and of all.
__device__ __forceinline__ int kp_before(const KpWs &w, int tile, int &all, int32_t *sums) {
    int a = 0, b = 0, t;
    for (int i = threadIdx.x; i < w.tiles; i += KP_NT) {
        const int c = w.tile[i];
        a += i < tile ? c : 0;
        b += c;
    }
    kp_scan(a, t, sums);
    kp_scan(b, all, sums);
    return t;
}

// The free pages in order: the first to the rows that get copies, the others to
// the list.
__global__ __launch_bounds__(KP_NT) void k_fork_assign(KvPages p) {
    __shared__ int32_t sums[KP_NT / WAVE];
    const KpWs w = kp_ws(p);
    const int64_t i0 = (int64_t)blockIdx.x * KP_TILE + 4 * threadIdx.x;
    bool is[4];
    int n = 0, all, total;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        is[k] = i0 + k < p.n_pages && w.mark[i0 + k] == KP_FREE;
        n += is[k];
    }
    const int n_copy = w.tile[w.tiles];
    const int first = kp_before(w, blockIdx.x, all, sums);
    int f = first + kp_scan(n, total, sums);
    const int left = max(all - n_copy, 0);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.count[0] = left;
        p.count[1] = n_copy;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = i0 + k;
        if (i >= left && i < p.n_pages) p.free_out[i] = -1;
        if (!is[k]) continue;
        if (f < n_copy) {
            const int row = w.list[f];
            const KpRow r = kp_row(p, row);
            p.copy_dst[row] = (int)i;
            p.table_out[(int64_t)row * p.ld_out + r.have - 1] = (int)i;
        } else {
            p.free_out[f - n_copy] = (int)i;
        }
        ++f;
    }
}

__global__ __launch_bounds__(256) void k_compact_mark(KvPages p) {
    const KpWs w = kp_ws(p);
    const int64_t have = kp_have(p, max(p.kv_len[blockIdx.y], 0));
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < have; j += (int64_t)gridDim.x * 256) {
        const int id = kp_entry(p, blockIdx.y, j);
        if (id >= 0) w.mark[id] = 1u;  // (several rows: all the same value)
    }
}

// N pages are held.  Page i >= N that is held is the (held before i - held before
// N)-th to move, page i < N that is not the (i - held before i)-th to be filled.
__global__ __launch_bounds__(KP_NT) void k_compact_assign(KvPages p) {
    __shared__ int32_t sums[KP_NT / WAVE];
    const KpWs w = kp_ws(p);
    const int64_t i0 = (int64_t)blockIdx.x * KP_TILE + 4 * threadIdx.x;
    bool is[4];
    int n = 0, all, total;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        is[k] = i0 + k < p.n_pages && w.mark[i0 + k] == 1u;
        n += is[k];
    }
    const int first = kp_before(w, blockIdx.x, all, sums);
    int before = first + kp_scan(n, total, sums);
    // held pages below N: those of the tiles before N's, and its own
    const int tn = all / KP_TILE;
    int below = 0, tiles_below;
    for (int64_t i = (int64_t)tn * KP_TILE + threadIdx.x; i < all; i += KP_NT) below += w.mark[i] == 1u;
    int a = 0;
    for (int i = threadIdx.x; i < tn; i += KP_NT) a += w.tile[i];
    kp_scan(below + a, tiles_below, sums);
    const int n_move = all - tiles_below;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.count[0] = all;
        p.count[1] = n_move;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = i0 + k;
        if (i >= p.n_pages) break;
        if (i >= n_move && i < p.n_pages / 2) p.copy_src[i] = p.copy_dst[i] = -1;
        if (is[k] && i >= all) {
            const int rank = before - tiles_below;
            p.copy_src[rank] = (int)i;
            w.list[i] = rank;
        } else if (!is[k] && i < all) {
            p.copy_dst[(int)i - before] = (int)i;
        }
        before += is[k];
    }
}

__global__ __launch_bounds__(256) void k_compact_tables(KvPages p) {
    const KpWs w = kp_ws(p);
    const int64_t have = kp_have(p, max(p.kv_len[blockIdx.y], 0)), N = p.count[0];
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < p.ld_out; j += (int64_t)gridDim.x * 256) {
        int id = j < have ? kp_entry(p, blockIdx.y, j) : -1;
        if (id >= N) id = p.copy_dst[w.list[id]];
        p.table_out[(int64_t)blockIdx.y * p.ld_out + j] = id;
    }
}

static dim3 kp_rows(int64_t width, int64_t rows) {
    const int64_t x = (width + 255) / 256;
    return dim3((unsigned)(x < 1 ? 1 : x > 64 ? 64 : x), (unsigned)rows);
}
hipError_t launch_kv_fork(const KvPages &p, hipStream_t stream) {
    const int tiles = kp_tiles(p.n_pages);
    if (tiles) hipLaunchKernelGGL(k_pages_clear<true>, dim3((unsigned)((p.n_pages + 255) / 256)), dim3(256), 0, stream, p);
    if (p.n_out) hipLaunchKernelGGL(k_fork_mark, kp_rows(p.ld_out, p.n_out), dim3(256), 0, stream, p);
    hipLaunchKernelGGL(k_pages_count<true>, dim3(tiles + 1), dim3(KP_NT), 0, stream, p);
    hipLaunchKernelGGL(k_fork_assign, dim3(tiles ? tiles : 1), dim3(KP_NT), 0, stream, p);
    return hipGetLastError();
}
hipError_t launch_kv_compact(const KvPages &p, hipStream_t stream) {
    const int tiles = kp_tiles(p.n_pages);
    if (tiles) hipLaunchKernelGGL(k_pages_clear<false>, dim3((unsigned)((p.n_pages + 255) / 256)), dim3(256), 0, stream, p);
    if (p.n_seq) hipLaunchKernelGGL(k_compact_mark, kp_rows(p.ld_table, p.n_seq), dim3(256), 0, stream, p);
    if (tiles) hipLaunchKernelGGL(k_pages_count<false>, dim3(tiles), dim3(KP_NT), 0, stream, p);
    hipLaunchKernelGGL(k_compact_assign, dim3(tiles ? tiles : 1), dim3(KP_NT), 0, stream, p);
    if (p.n_seq) hipLaunchKernelGGL(k_compact_tables, kp_rows(p.ld_out, p.n_seq), dim3(256), 0, stream, p);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Copying.  A page's rows in 16-byte pieces, in the order of memory: `outer`
// rows of `mid` rows of `run` pieces that follow each other, as long as the
// layout and the number of tokens allow.  A workgroup takes CP_CHUNK pieces of a
// page of one plane (keys or values of one cache), all loads before the first
// store.  Bound by the bytes.
// ---------------------------------------------------------------------------
constexpr int CP_NT = 256, CP_PER = 4, CP_CHUNK = CP_NT * CP_PER;

__global__ __launch_bounds__(CP_NT) void k_kv_copy(KvCopy p, int parts, int by_token) {
    const int plane = blockIdx.y, c = plane >> 1;
    v4u *base = reinterpret_cast<v4u *>(plane & 1 ? p.c[c].v : p.c[c].k);
    const uint32_t n = (uint32_t)(p.n_dev ? min(p.n, max(*p.n_dev, (int64_t)0)) : p.n);  // n <= 2^24, parts <= 64
    const uint32_t d8 = p.kv.d_head / 8, page = 1u << p.kv.page_shift, heads = p.kv.n_head;
    const uint32_t lh = (uint32_t)p.kv.ld_head / 8, lt = (uint32_t)p.kv.ld_tok / 8;
    const int64_t lp = p.kv.ld_page / 8;
    for (uint32_t u = blockIdx.x; u < n * parts; u += gridDim.x) {
        const uint32_t e = u / (uint32_t)parts, part = u - e * parts;
        const int src = p.src[e], dst = p.dst[e];
        if (src < 0 || dst < 0 || src >= p.kv.n_pages || dst >= p.kv.n_pages || src == dst) continue;  // (uniform)
        const uint32_t toks = p.n_tok ? (uint32_t)min(max(p.n_tok[e], 0), (int)page) : page;
        uint32_t outer = by_token ? toks : heads, mid = by_token ? heads : toks, run = d8;
        const uint32_t so = by_token ? lt : lh, sm = by_token ? lh : lt;
        if (sm == run || mid == 1) {
            run *= mid;
            mid = 1;
            if (so == run || outer == 1) {
                run *= outer;
                outer = 1;
            }
        }
        const uint32_t all = outer * mid * run, per = mid * run;
        const v4u *from = base + src * lp;
        v4u *to = base + dst * lp;
        for (uint64_t i0 = (uint64_t)part * CP_CHUNK; i0 < all; i0 += (uint64_t)parts * CP_CHUNK) {
            v4u t[CP_PER];
            uint32_t at[CP_PER];
#pragma unroll
            for (int k = 0; k < CP_PER; ++k) {
                const uint32_t i = (uint32_t)min(i0 + k * CP_NT + threadIdx.x, (uint64_t)all - 1);
                at[k] = i;
                if (outer > 1 || mid > 1) {
                    const uint32_t a = i / per, rest = i - a * per, b = rest / run;
                    at[k] = a * so + b * sm + (rest - b * run);
                }
                t[k] = from[at[k]];
            }
#pragma unroll
            for (int k = 0; k < CP_PER; ++k)
                if (i0 + k * CP_NT + threadIdx.x < all) to[at[k]] = t[k];
        }
    }
}

hipError_t launch_kv_copy(const KvCopy &p, hipStream_t stream) {
    const int64_t pieces = (int64_t)p.kv.n_head * p.kv.d_head / 8 << p.kv.page_shift;
    int64_t parts = (pieces + CP_CHUNK - 1) / CP_CHUNK;
    parts = parts > 64 ? 64 : parts;
    const int64_t units = p.n * parts, most = 1 << 14;
    const int by_token = p.kv.ld_tok > p.kv.ld_head;
    hipLaunchKernelGGL(k_kv_copy, dim3((unsigned)(units < most ? units : most), 2 * p.n_cache), dim3(CP_NT), 0, stream, p,
                       (int)parts, by_token);
    return hipGetLastError();
}

}  // namespace s2x
