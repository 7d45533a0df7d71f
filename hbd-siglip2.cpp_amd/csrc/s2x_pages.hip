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
// (fork) or the moved pages' ranks (compact), the rows' open pages (fork).
struct KpWs {
    uint32_t *mark;
    int32_t  *tile, *list, *last;
    int       tiles;
};
static __host__ __device__ inline int kp_tiles(int64_t n_pages) { return (int)((n_pages + KP_TILE - 1) / KP_TILE); }
static __host__ __device__ inline KpWs kp_ws(const KvPages &p) {
    KpWs w;
    w.tiles = kp_tiles(p.n_pages);
    w.mark = (uint32_t *)p.ws;
    w.tile = (int32_t *)(w.mark + p.n_pages);
    w.last = w.tile + w.tiles + 1;
    w.list = w.last + KV_MAX_SEQ;
    return w;
}
size_t kv_pages_workspace(int64_t n_pages) {
    const int64_t list = n_pages > KV_MAX_SEQ ? n_pages : KV_MAX_SEQ;
    return (size_t)(n_pages + kp_tiles(n_pages) + 1 + KV_MAX_SEQ + list) * 4;
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
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.len_out[i] = r.len;
        w.last[i] = r.open ? kp_entry(p, r.src, r.have - 1) : -1;
    }
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < p.ld_out; j += (int64_t)gridDim.x * 256) {
        int id = -1;
        if (j < r.have) {
            id = kp_entry(p, r.src, j);
            if (id >= 0) atomicMin(&w.mark[id], r.open && j == r.have - 1 ? 1u + i : 0u);
        }
        p.table_out[(int64_t)i * p.ld_out + j] = id;
    }
}

// Row i and the page that it copies (-1: none), until it gets its own.
__device__ __forceinline__ void kp_want(const KvPages &p, int i, int last) {
    const int len = p.len_out[i];
    p.copy_src[i] = last;
    p.copy_dst[i] = -1;
    p.copy_tok[i] = last >= 0 ? len & ((1 << p.page_shift) - 1) : 0;
    if (last >= 0) p.table_out[(int64_t)i * p.ld_out + kp_have(p, len) - 1] = -1;
}
__device__ __forceinline__ void kp_give(const KvPages &p, int row, int page) {
    p.copy_dst[row] = page;
    p.table_out[(int64_t)row * p.ld_out + kp_have(p, p.len_out[row]) - 1] = page;
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
        const int last = i < p.n_out ? w.last[i] : -1;
        const bool want = last >= 0 && w.mark[last] != 1u + i;
        const int at = base + kp_scan(want, total, sums);
        base += total;
        if (i < p.n_out) kp_want(p, i, want ? last : -1);
        if (want) w.list[at] = i;
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
            kp_give(p, w.list[f], (int)i);
        } else {
            p.free_out[f - n_copy] = (int)i;
        }
        ++f;
    }
}

// The same of few pages, where a workgroup counts all marks, and all rows that get
// copies, itself rather than after another launch: with the copies, 480 rows over 8,000
// pages 22.6 us, with the launch 23.8; a compaction that moves 4,000 pages 105 and 107.
constexpr int KP_FEW = 8 * KP_TILE;
__device__ __forceinline__ void kp_marks(const KpWs &w, int64_t n_pages, uint32_t what, uint32_t (&is)[KP_FEW / KP_TILE]) {
    v4u m[KP_FEW / KP_TILE];
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t) {  // bit k of is[t]: page t KP_TILE + 4 tid + k
        const int64_t i0 = (int64_t)t * KP_TILE + 4 * threadIdx.x;
        m[t] = v4u{~what, ~what, ~what, ~what};
        if (i0 + 4 <= n_pages) {
            m[t] = *reinterpret_cast<const v4u *>(w.mark + i0);
        } else {
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (i0 + k < n_pages) m[t][k] = w.mark[i0 + k];
        }
    }
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t) {
        is[t] = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) is[t] |= (uint32_t)(m[t][k] == what) << k;
    }
}
__global__ __launch_bounds__(KP_NT) void k_fork_assign_few(KvPages p) {
    __shared__ int32_t sums[KP_NT / WAVE];
    __shared__ int32_t list[KV_MAX_SEQ];
    const KpWs w = kp_ws(p);
    uint32_t is[KP_FEW / KP_TILE];
    kp_marks(w, p.n_pages, KP_FREE, is);
    int n_copy = 0, all, before, total;
    for (int i0 = 0; i0 < p.n_out; i0 += KP_NT) {
        const int i = i0 + threadIdx.x, last = i < p.n_out ? w.last[i] : -1;
        const bool want = last >= 0 && w.mark[last] != 1u + i;
        const int at = n_copy + kp_scan(want, total, sums);
        n_copy += total;
        if (want) list[at] = i;
        // (a row that gets a page has its place and table entry from the workgroup of that page)
        if (blockIdx.x == 0 && i < p.n_out) {
            p.copy_src[i] = want ? last : -1;
            p.copy_tok[i] = want ? p.len_out[i] & ((1 << p.page_shift) - 1) : 0;
            if (!want) p.copy_dst[i] = -1;
        }
    }
    int a = 0, b = 0, mine = 0;
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t) {
        const int n = __builtin_popcount(is[t]);
        if (t < (int)blockIdx.x) a += n;
        if (t == (int)blockIdx.x) mine = n;
        b += n;
    }
    kp_scan(a, before, sums);
    kp_scan(b, all, sums);
    int f = before + kp_scan(mine, total, sums);  // (and the list is there)
    const int left = max(all - n_copy, 0);
    if (blockIdx.x == 0) {
        if (threadIdx.x == 0) {
            p.count[0] = left;
            p.count[1] = n_copy;
        }
        for (int k = all + threadIdx.x; k < n_copy; k += KP_NT) kp_give(p, list[k], -1);
    }
    uint32_t bits = 0;
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t)
        if (t == (int)blockIdx.x) bits = is[t];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int64_t i = (int64_t)blockIdx.x * KP_TILE + 4 * threadIdx.x + k;
        if (i >= left && i < p.n_pages) p.free_out[i] = -1;
        if (!(bits >> k & 1)) continue;
        if (f < n_copy) kp_give(p, list[f], (int)i);
        else p.free_out[f - n_copy] = (int)i;
        ++f;
    }
}

// All of a fork in one workgroup, marks in LDS: few entries and pages, whose time
// would be that of the launches (4 rows of 26 entries: 3.9 us, in three launches 14;
// 96 rows of 112 11 against 13, 240 21 against 14).
constexpr int KP_ONE_PAGES = 16 * KP_NT, KP_ONE_ENTRIES = 12 * KP_NT;
__global__ __launch_bounds__(KP_NT) void k_fork_one(KvPages p) {
    __shared__ uint32_t mark[KP_ONE_PAGES];
    __shared__ int32_t sums[KP_NT / WAVE], src[KP_NT], have[KP_NT], list[KP_NT], last[KP_NT];
    __shared__ bool open[KP_NT];
    const int tid = threadIdx.x, n_pages = (int)p.n_pages, ld = (int)p.ld_out;
    KpRow r = {};
    if (tid < p.n_out) {
        r = kp_row(p, tid);
        src[tid] = r.src;
        have[tid] = (int)r.have;
        open[tid] = r.open;
        last[tid] = -1;
        p.len_out[tid] = r.len;
    }
    for (int i = tid; i < n_pages; i += KP_NT) mark[i] = p.pinned && p.pinned[i] ? 0u : KP_FREE;
    __syncthreads();
#pragma unroll 4
    for (int e = tid; e < p.n_out * ld; e += KP_NT) {
        const int i = e / ld, j = e - i * ld;
        int id = -1;
        if (j < have[i]) {
            id = kp_entry(p, src[i], j);
            if (id >= 0) {
                const bool o = open[i] && j == have[i] - 1;
                atomicMin(&mark[id], o ? 1u + i : 0u);
                if (o) last[i] = id;
            }
        }
        p.table_out[e] = id;
    }
    __syncthreads();
    int n_copy, all;
    const int page = tid < p.n_out ? last[tid] : -1;
    const bool want = page >= 0 && mark[page] != 1u + tid;
    const int at = kp_scan(want, n_copy, sums);
    if (want) list[at] = tid;
    const int per = (n_pages + KP_NT - 1) / KP_NT;  // pages of a thread, at most 16
    int n = 0;
    for (int k = 0; k < per; ++k) n += tid * per + k < n_pages && mark[tid * per + k] == KP_FREE;
    int f = kp_scan(n, all, sums);
    const int left = max(all - n_copy, 0);
    if (tid == 0) {
        p.count[0] = left;
        p.count[1] = n_copy;
    }
    if (tid < p.n_out) {
        p.copy_src[tid] = want ? page : -1;
        p.copy_tok[tid] = want ? r.len & ((1 << p.page_shift) - 1) : 0;
        if (!want || at >= all) p.copy_dst[tid] = -1;
        if (want && at >= all) p.table_out[tid * ld + r.have - 1] = -1;
    }
    for (int i = left + tid; i < n_pages; i += KP_NT) p.free_out[i] = -1;
    for (int k = 0; k < per; ++k) {
        const int i = tid * per + k;
        if (i >= n_pages || mark[i] != KP_FREE) continue;
        if (f < n_copy) {
            const int row = list[f];
            p.copy_dst[row] = i;
            p.table_out[row * ld + have[row] - 1] = i;
        } else {
            p.free_out[f - n_copy] = i;
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

// `all` pages are held, `below` of them among the first `all`, `before` of them
// before page i.  Page i >= all that is held is the (before - below)-th to move, page
// i < all that is not the (i - before)-th to be filled.
__device__ __forceinline__ void kp_place(const KvPages &p, const KpWs &w, int64_t i, bool held, int &before, int all, int below) {
    if (i >= p.n_pages) return;
    if (i >= all - below && i < p.n_pages / 2) p.copy_src[i] = p.copy_dst[i] = -1;
    if (held && i >= all) {
        const int rank = before - below;
        p.copy_src[rank] = (int)i;
        w.list[i] = rank;
    } else if (!held && i < all) {
        p.copy_dst[(int)i - before] = (int)i;
    }
    before += held;
}
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
    for (int k = 0; k < 4; ++k) kp_place(p, w, i0 + k, is[k], before, all, tiles_below);
}

// (as k_fork_assign_few)
__global__ __launch_bounds__(KP_NT) void k_compact_assign_few(KvPages p) {
    __shared__ int32_t sums[KP_NT / WAVE];
    const KpWs w = kp_ws(p);
    uint32_t is[KP_FEW / KP_TILE];
    kp_marks(w, p.n_pages, 1u, is);
    int a = 0, b = 0, mine = 0, c = 0, first, all, below, total;
    uint32_t bits = 0;
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t) {
        const int n = __builtin_popcount(is[t]);
        if (t < (int)blockIdx.x) a += n;
        if (t == (int)blockIdx.x) {
            mine = n;
            bits = is[t];
        }
        b += n;
    }
    kp_scan(a, first, sums);
    kp_scan(b, all, sums);
    int before = first + kp_scan(mine, total, sums);
#pragma unroll
    for (int t = 0; t < KP_FEW / KP_TILE; ++t) {
        const int n = min(max(all - t * KP_TILE - 4 * (int)threadIdx.x, 0), 4);  // of this thread's below N
        c += __builtin_popcount(is[t] & ((1u << n) - 1));
    }
    kp_scan(c, below, sums);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.count[0] = all;
        p.count[1] = all - below;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        kp_place(p, w, (int64_t)blockIdx.x * KP_TILE + 4 * threadIdx.x + k, bits >> k & 1, before, all, below);
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
    if (p.n_out <= KP_NT && p.n_out * p.ld_out <= KP_ONE_ENTRIES && p.n_pages <= KP_ONE_PAGES) {
        hipLaunchKernelGGL(k_fork_one, dim3(1), dim3(KP_NT), 0, stream, p);
        return hipGetLastError();
    }
    const int tiles = kp_tiles(p.n_pages);
    if (tiles) hipLaunchKernelGGL(k_pages_clear<true>, dim3((unsigned)((p.n_pages + 255) / 256)), dim3(256), 0, stream, p);
    if (p.n_out) hipLaunchKernelGGL(k_fork_mark, kp_rows(p.ld_out, p.n_out), dim3(256), 0, stream, p);
    if (p.n_pages <= KP_FEW) {
        hipLaunchKernelGGL(k_fork_assign_few, dim3(tiles ? tiles : 1), dim3(KP_NT), 0, stream, p);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_pages_count<true>, dim3(tiles + 1), dim3(KP_NT), 0, stream, p);
    hipLaunchKernelGGL(k_fork_assign, dim3(tiles), dim3(KP_NT), 0, stream, p);
    return hipGetLastError();
}
hipError_t launch_kv_compact(const KvPages &p, hipStream_t stream) {
    const int tiles = kp_tiles(p.n_pages);
    if (tiles) hipLaunchKernelGGL(k_pages_clear<false>, dim3((unsigned)((p.n_pages + 255) / 256)), dim3(256), 0, stream, p);
    if (p.n_seq) hipLaunchKernelGGL(k_compact_mark, kp_rows(p.ld_table, p.n_seq), dim3(256), 0, stream, p);
    if (p.n_pages <= KP_FEW) {
        hipLaunchKernelGGL(k_compact_assign_few, dim3(tiles ? tiles : 1), dim3(KP_NT), 0, stream, p);
    } else {
        hipLaunchKernelGGL(k_pages_count<false>, dim3(tiles), dim3(KP_NT), 0, stream, p);
        hipLaunchKernelGGL(k_compact_assign, dim3(tiles), dim3(KP_NT), 0, stream, p);
    }
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
