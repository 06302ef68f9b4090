// Pages of a cache: token rows into pages and back, rows copied in the pools of many layers at once, and the bookkeeping
// of forked, freed and compacted sequences (gfx950).  Everything here moves bytes or counts: the copies are bound by HBM,
// the bookkeeping by the latency of a launch.
//
// The bookkeeping is deterministic: ranks come from scans in index order, reference counts from commutative integer
// updates.  Parts that need an order over all pages run in one workgroup (a scan over 4096 pages is one step of it); what
// follows from their result (table rows, page copies) runs over the whole chip in a second launch.
#include "pages.h"

namespace kda355 {
namespace {

constexpr int ROW = KDA355_LATENT_ROW, LAT = KDA355_LATENT_DIM;
constexpr int ROW_Q = ROW / 8, LAT_Q = LAT / 8;  // 16-byte pieces of a cache row, of its latent part
constexpr int TOK_THREADS = 192, TOKENS = 8, PIECES = TOKENS * ROW_Q / TOK_THREADS;  // 3 pieces a thread
static_assert(PIECES * TOK_THREADS == TOKENS * ROW_Q, "");
constexpr int COPY_THREADS = 256, COPY_PER = 4;   // 16 KiB a workgroup
constexpr int MAX_PAIRS = 1 << 23;                // rows of a launch: 256 threads each, below 2^32 in all
constexpr int MOST_HOLDERS = 1 << 30;             // no count reaches it

// ------------------------------------------------------------------------------------------------ token rows
// A workgroup moves TOKENS rows: as many lanes find where they stand, then every thread has PIECES reads under way at once.  64 k
// tokens read back and 6 k written: 33.7 us with 8 rows (4.9 TB/s); data in the caches, 30.2 with 8, 31.7 with 32, and a small
// call 6.2 us with 8, 9.4 with 32.
__global__ void __launch_bounds__(TOK_THREADS) append_kernel(KdaLatentTokensArgs a) {
    __shared__ char* to[TOKENS];
    const int64_t first = (int64_t)blockIdx.x * TOKENS;
    if (threadIdx.x < TOKENS) {
        const int64_t t = first + threadIdx.x, slot = t < a.T ? a.slots[t] : -1;
        char* row = nullptr;
        if (slot >= 0 && slot < a.pages * a.page_size) {
            const int64_t page = slot / a.page_size;
            row = static_cast<char*>(a.cache) + 2 * (page * a.page_stride + (slot - page * a.page_size) * ROW);
        }
        to[threadIdx.x] = row;
    }
    __syncthreads();
    u32x4 x[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        if (!to[t]) continue;
        const uint16_t* src = c < LAT_Q ? static_cast<const uint16_t*>(a.latent) + (first + t) * a.latent_row + c * 8
                                        : static_cast<const uint16_t*>(a.k_pe) + (first + t) * a.pe_row + (c - LAT_Q) * 8;
        x[i] = *reinterpret_cast<const u32x4*>(src);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        if (to[t]) *reinterpret_cast<u32x4*>(to[t] + c * 16) = x[i];
    }
}

__global__ void __launch_bounds__(TOK_THREADS) gather_kernel(KdaLatentTokensArgs a) {
    __shared__ const char* from[TOKENS];
    __shared__ char* to[TOKENS];
    const int64_t first = (int64_t)blockIdx.x * TOKENS;
    if (threadIdx.x < TOKENS) {
        const int64_t t = first + threadIdx.x;
        const char* row = nullptr;
        char* out = nullptr;
        if (t < a.T) {
            int lo = 0, hi = a.N;  // the sequence of row t: the last n with cu[n] <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.cu[mid] <= t) lo = mid; else hi = mid;
            }
            const int64_t j = t - a.cu[lo];
            if (j >= 0 && t < a.cu[lo + 1]) {
                out = static_cast<char*>(a.out) + 2 * t * a.out_row;
                const int64_t p = j / a.page_size;
                if (p < a.table_width) {
                    const int64_t page = a.block_table[lo * a.table_stride + p];
                    if (page >= 0 && page < a.pages)
                        row = static_cast<const char*>(a.cache) + 2 * (page * a.page_stride + (j - p * a.page_size) * ROW);
                }
            }
        }
        from[threadIdx.x] = row;
        to[threadIdx.x] = out;
    }
    __syncthreads();
    u32x4 x[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        x[i] = from[t] ? *reinterpret_cast<const u32x4*>(from[t] + c * 16) : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        if (to[t]) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(to[t] + c * 16));  // (39.5 -> 33.7 us)
    }
}

// ------------------------------------------------------------------------------------------------ row copies
// One 16 KiB segment of row src -> row dst of one pool.  The stores pass the caches: 600 MB moved in 134 us instead of 137, 64
// part-filled pages copied in 4 pools and their bookkeeping in 16.3 instead of 17.3; 8 pieces a thread instead of 4: 210 us.
__device__ __forceinline__ void copy_segment(const KdaPool& p, int64_t src, int64_t dst, int seg) {
    if (src < 0 || src >= p.slots || dst < 0 || dst >= p.slots || src == dst) return;
    const char* s = static_cast<const char*>(p.base) + src * p.slot_stride;
    char* d = static_cast<char*>(p.base) + dst * p.slot_stride;
    const int64_t b0 = (int64_t)seg * COPY_THREADS * COPY_PER * 16 + threadIdx.x * 16;
    u32x4 x[COPY_PER];
#pragma unroll
    for (int i = 0; i < COPY_PER; ++i) {
        const int64_t b = b0 + i * COPY_THREADS * 16;
        if (b < p.row_bytes) x[i] = *reinterpret_cast<const u32x4*>(s + b);
    }
#pragma unroll
    for (int i = 0; i < COPY_PER; ++i) {
        const int64_t b = b0 + i * COPY_THREADS * 16;
        if (b < p.row_bytes) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4*>(d + b));
    }
}

__global__ void __launch_bounds__(COPY_THREADS) copy_rows_kernel(KdaPagesArgs a) {
    copy_segment(a.pool[blockIdx.z], a.src[blockIdx.x], a.dst[blockIdx.x], blockIdx.y);
}

// ------------------------------------------------------------------------------------------------ fork
__device__ __forceinline__ int row_len(const KdaPagesArgs& a, int row) {
    const int64_t most = (int64_t)a.table_width * a.page_size;
    const int64_t n = a.seq_lens[row];
    return (int)(n < 0 ? 0 : n > most ? most : n);
}

// pair i -> workspace[i] = page to copy from (-1: none), workspace[n + i] = page taken (-1: none needed, -2: no page
// left, -3: pair skipped).  A part-filled last page that is a hole needs none: a page taken for it would hold what its last
// owner left, and the child would see it.  The stack and its height follow.
__global__ void __launch_bounds__(SCAN_THREADS) fork_take_kernel(KdaPagesArgs a) {
    __shared__ int sw[SCAN_THREADS / 64];
    int top = a.num_free[0];
    top = top < 0 ? 0 : top > a.pages ? a.pages : top;
    int taken = 0;
    for (int i0 = 0; i0 < a.n; i0 += SCAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int ok = 0, tail = 0, last = -1;  // is the parent's last page part-filled and there; that page
        if (i < a.n) {
            const int par = a.src[i], child = a.dst[i];
            ok = par >= 0 && par < a.rows && child >= 0 && child < a.rows && par != child;
            const int len = ok ? row_len(a, par) : 0;
            if (len % a.page_size != 0) last = a.block_table[par * a.table_stride + len / a.page_size];
            tail = last >= 0 && last < a.pages;
        }
        int total;
        const int rank = taken + block_scan(tail, sw, total);
        if (i < a.n) {
            int from = -1, to = ok ? -1 : -3;
            if (tail) {
                to = -2;
                if (rank < top) {
                    const int page = a.free_pages[top - 1 - rank];
                    a.free_pages[top - 1 - rank] = -1;
                    if (page >= 0 && page < a.pages) {
                        to = page;
                        from = last;
                    }
                }
            }
            a.workspace[i] = from;
            a.workspace[a.n + i] = to;
        }
        taken += total;
    }
    if (threadIdx.x == 0) a.num_free[0] = top - (taken < top ? taken : top);
}

// blockIdx.z < num_pools: a segment of the copied page; the last z: the child's row of the table
__global__ void __launch_bounds__(COPY_THREADS) fork_rows_kernel(KdaPagesArgs a) {
    const int i = blockIdx.x;
    const int to = a.workspace[a.n + i];
    if ((int)blockIdx.z < a.num_pools) {
        if (to >= 0) copy_segment(a.pool[blockIdx.z], a.workspace[i], to, blockIdx.y);
        return;
    }
    if (blockIdx.y != 0 || to == -3) return;
    const int par = a.src[i], child = a.dst[i];
    const int len = to == -2 ? 0 : row_len(a, par);
    const int full = len / a.page_size;
    const int32_t* from = a.block_table + par * a.table_stride;
    int32_t* row = a.block_table + child * a.table_stride;
    for (int j = threadIdx.x; j < a.table_width; j += COPY_THREADS) {
        int page = -1;
        if (j < full) {
            page = from[j];
            if (page >= 0 && page < a.pages) atomicAdd(a.ref_counts + page, 1);
        } else if (j == full && to >= 0) {
            page = to;
            a.ref_counts[page] = 1;
        }
        row[j] = page;
    }
    if (threadIdx.x == 0) a.seq_lens[child] = len;
}

// ------------------------------------------------------------------------------------------------ free
// A reference is taken back by a plain difference, and the last holder marks the page.  Counts may change in any order: a holder
// too many (a caller's mistake) finds zero or less, or the mark, or what wraps around below it, and puts its difference back.
// (Compare and swap on a page that 1000 sequences share: 3.1 ms instead of 93 us.)
__global__ void __launch_bounds__(COPY_THREADS) free_rows_kernel(KdaPagesArgs a) {
    const int r = a.src[blockIdx.x];
    if (r < 0 || r >= a.rows) return;
    const int used = (row_len(a, r) + a.page_size - 1) / a.page_size;
    int32_t* row = a.block_table + r * a.table_stride;
    for (int j = threadIdx.x; j < a.table_width; j += COPY_THREADS) {
        const int page = row[j];
        if (j < used && page >= 0 && page < a.pages) {
            const int before = atomicSub(a.ref_counts + page, 1);
            if (before <= 1 || before >= MOST_HOLDERS) atomicAdd(a.ref_counts + page, before == 1 ? FREED : 1);
        }
        row[j] = -1;
    }
    __syncthreads();  // every thread has read the length
    if (threadIdx.x == 0) a.seq_lens[r] = 0;
}

// The same in one workgroup and one launch, where there is little to give up: what each page loses is counted in LDS, so that no
// two threads meet in memory.  128 table entries 3.7 us (two launches 5.0), 2048 4.8 (5.7), 4160 5.9 (5.6; with differences in
// memory 9.2), 8192 9.8 (7.6).  A launch takes 2.7 us of the caller's time, so it is taken up to where the GPU is about as fast.
constexpr int FREE_SMALL = 5 * SCAN_THREADS, FREE_STEPS = 4;  // table entries, those of a thread at a time
constexpr int FREE_PAGES = 16 * 1024;
__global__ void __launch_bounds__(SCAN_THREADS) free_small_kernel(KdaPagesArgs a) {
    __shared__ int lost[FREE_PAGES];
    __shared__ int sw[SCAN_THREADS / 64];
    for (int i = threadIdx.x; i < a.pages; i += SCAN_THREADS) lost[i] = 0;
    __syncthreads();
    const int all = a.n * a.table_width;
    for (int e0 = threadIdx.x; e0 < all; e0 += FREE_STEPS * SCAN_THREADS) {
        int32_t* at[FREE_STEPS];
        int page[FREE_STEPS];
#pragma unroll
        for (int k = 0; k < FREE_STEPS; ++k) {  // rows, lengths and pages of all of them under way at once
            const int e = min(e0 + k * SCAN_THREADS, all - 1), i = e / a.table_width, j = e - i * a.table_width;
            const int r = a.src[i], row = min(max(r, 0), a.rows - 1);
            at[k] = a.block_table + row * a.table_stride + j;
            page[k] = *at[k];
            const bool mine = e0 + k * SCAN_THREADS < all && r == row;
            if (!mine) at[k] = nullptr;
            if (!mine || (int64_t)j * a.page_size >= row_len(a, row)) page[k] = -1;
        }
#pragma unroll
        for (int k = 0; k < FREE_STEPS; ++k) {
            if (page[k] >= 0 && page[k] < a.pages) atomicAdd(&lost[page[k]], 1);
            if (at[k]) *at[k] = -1;
        }
    }
    __syncthreads();  // every thread has read the lengths
    for (int i = threadIdx.x; i < a.n; i += SCAN_THREADS) {
        const int r = a.src[i];
        if (r >= 0 && r < a.rows) a.seq_lens[r] = 0;
    }
    int top = a.num_free[0];
    top = top < 0 ? 0 : top > a.pages ? a.pages : top;
    for (int hi = a.pages; hi > 0; hi -= FREE_STEPS * SCAN_THREADS) {  // the highest pages first
        int mine[FREE_STEPS], count = 0;
#pragma unroll
        for (int k = 0; k < FREE_STEPS; ++k) {
            const int p = hi - 1 - FREE_STEPS * (int)threadIdx.x - k;
            mine[k] = 0;
            if (p < 0 || lost[p] == 0) continue;
            const int held = a.ref_counts[p];
            if (held <= 0) continue;  // (a caller's mistake)
            mine[k] = lost[p] >= held;
            a.ref_counts[p] = mine[k] ? 0 : held - lost[p];
            count += mine[k];
        }
        int total;
        int slot = top + block_scan(count, sw, total);
#pragma unroll
        for (int k = 0; k < FREE_STEPS; ++k)
            if (mine[k]) {
                if (slot < a.pages) a.free_pages[slot] = hi - 1 - FREE_STEPS * (int)threadIdx.x - k;
                ++slot;
            }
        top += total;
    }
    if (threadIdx.x == 0) a.num_free[0] = top < a.pages ? top : a.pages;
}

// ------------------------------------------------------------------------------------------------ compact
// workspace: remap [pages] | sources [pages / 2] | destinations [pages / 2], padded with -1
__global__ void __launch_bounds__(SCAN_THREADS) compact_plan_kernel(KdaPagesArgs a) {
    __shared__ int sw[SCAN_THREADS / 64];
    const int pages = a.pages, half = pages / 2;
    int32_t* remap = a.workspace;
    int32_t* msrc = remap + pages;
    int32_t* mdst = msrc + half;
    int mine = 0, live;
    for (int p = threadIdx.x; p < pages; p += SCAN_THREADS) mine += a.ref_counts[p] > 0;
    block_scan(mine, sw, live);
    int holes = 0, movers = 0;
    for (int p0 = 0; p0 < pages; p0 += SCAN_THREADS) {
        const int p = p0 + threadIdx.x;
        const bool held = p < pages && a.ref_counts[p] > 0;
        const int hole = p < live && !held, mover = held && p >= live;  // (live <= pages)
        int total;
        const int rank = block_scan(hole | (mover << 16), sw, total);  // at most 1024 of either in a step
        if (hole) mdst[holes + (rank & 0xffff)] = p;
        if (mover) msrc[movers + (rank >> 16)] = p;
        if (p < pages) remap[p] = p;
        holes += total & 0xffff;
        movers += total >> 16;
    }
    __syncthreads();  // the lists are written (holes == movers, at most pages / 2)
    for (int i = threadIdx.x; i < half; i += SCAN_THREADS) {
        if (i < movers) {
            const int s = load_fresh(msrc + i), d = load_fresh(mdst + i);
            remap[s] = d;
            a.ref_counts[d] = a.ref_counts[s];
            a.ref_counts[s] = 0;
        } else {
            msrc[i] = -1;
            mdst[i] = -1;
        }
    }
    for (int j = threadIdx.x; j < pages; j += SCAN_THREADS) a.free_pages[j] = j < pages - live ? pages - 1 - j : -1;
    if (threadIdx.x == 0) a.num_free[0] = pages - live;
}

__global__ void __launch_bounds__(COPY_THREADS) compact_move_kernel(KdaPagesArgs a) {
    const int half = a.pages / 2;
    if ((int)blockIdx.z < a.num_pools) {
        if ((int)blockIdx.x >= half) return;
        copy_segment(a.pool[blockIdx.z], a.workspace[a.pages + blockIdx.x], a.workspace[a.pages + half + blockIdx.x],
                     blockIdx.y);
        return;
    }
    if (blockIdx.y != 0) return;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x)
        for (int j = threadIdx.x; j < a.table_width; j += COPY_THREADS) {
            int32_t* e = a.block_table + r * a.table_stride + j;
            const int page = *e;
            if (page >= 0 && page < a.pages) *e = a.workspace[page];
        }
}

int check_tokens(const KdaLatentTokensArgs* a, const char* what) {
    KDA_CHECK_ARG(a != nullptr, "%s: null args", what);
    KDA_CHECK_ARG(a->T >= 0 && a->pages >= 1 && a->page_size >= 1, "%s: T=%lld pages=%lld page_size=%d", what,
                  (long long)a->T, (long long)a->pages, a->page_size);
    KDA_CHECK_ARG(a->T < (1ll << 25), "%s: %lld token rows in one call (less than 2^25)", what, (long long)a->T);
    KDA_CHECK_ARG(a->cache, "%s: a required pointer is null", what);
    KDA_CHECK_ARG(aligned(a->cache, 16) && a->page_stride % 8 == 0 && a->page_stride >= (int64_t)a->page_size * ROW,
                  "%s: cache pages must be dense and 16-byte aligned", what);
    return 0;
}

// segments of the longest row; every pool checked
int check_pools(const KdaPagesArgs* a, const char* what, int* segs) {
    KDA_CHECK_ARG(a->num_pools >= 0 && a->num_pools <= KDA355_MAX_POOLS, "%s: num_pools=%d", what, a->num_pools);
    int64_t most = 0;
    for (int i = 0; i < a->num_pools; ++i) {
        const KdaPool& p = a->pool[i];
        KDA_CHECK_ARG(p.base && p.slots >= 0, "%s: pool %d is empty", what, i);
        KDA_CHECK_ARG(aligned(p.base, 16) && p.row_bytes > 0 && p.row_bytes % 16 == 0 && p.slot_stride % 16 == 0 &&
                          p.slot_stride >= p.row_bytes,
                      "%s: the rows of pool %d must be 16-byte aligned and a multiple of 16 bytes", what, i);
        most = p.row_bytes > most ? p.row_bytes : most;
    }
    const int64_t per = COPY_THREADS * COPY_PER * 16, n = (most + per - 1) / per;
    KDA_CHECK_ARG(n <= 65535, "%s: rows of %lld bytes are too long", what, (long long)most);
    *segs = n < 1 ? 1 : (int)n;
    return 0;
}

int check_table(const KdaPagesArgs* a, const char* what, bool lens) {
    KDA_CHECK_ARG(a->rows >= 1 && a->table_width >= 1 && a->pages >= 1 && a->pages < 2 * MAX_PAIRS && a->page_size >= 1,
                  "%s: rows=%d table_width=%d pages=%d page_size=%d", what, a->rows, a->table_width, a->pages, a->page_size);
    KDA_CHECK_ARG((int64_t)a->table_width * a->page_size < (1ll << 31), "%s: a table row spans 2^31 tokens or more", what);
    KDA_CHECK_ARG(a->table_stride >= a->table_width, "%s: table_stride < table_width", what);
    KDA_CHECK_ARG(a->block_table && a->ref_counts && a->free_pages && a->num_free && (!lens || a->seq_lens),
                  "%s: a required pointer is null", what);
    return 0;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int kda355_latent_append_launch(const KdaLatentTokensArgs* a, kda355_stream_t stream) {
    if (const int rc = check_tokens(a, "latent_append")) return rc;
    if (a->T == 0) return 0;
    KDA_CHECK_ARG(a->latent && a->k_pe && a->slots, "latent_append: a required pointer is null");
    KDA_CHECK_ARG(aligned(a->latent, 16) && aligned(a->k_pe, 16) && a->latent_row % 8 == 0 && a->pe_row % 8 == 0,
                  "latent_append: latent and k_pe rows must be 16-byte aligned");
    const int64_t wgs = (a->T + TOKENS - 1) / TOKENS;
    launch_kernel(append_kernel, dim3((uint32_t)wgs), dim3(TOK_THREADS), reinterpret_cast<hipStream_t>(stream), *a);
    return launched("latent_append");
}

extern "C" int kda355_latent_gather_launch(const KdaLatentTokensArgs* a, kda355_stream_t stream) {
    if (const int rc = check_tokens(a, "latent_gather")) return rc;
    if (a->T == 0 || a->N == 0) return 0;
    KDA_CHECK_ARG(a->N > 0 && a->table_width >= 1 && a->table_stride >= a->table_width, "latent_gather: N=%d table_width=%d",
                  a->N, a->table_width);
    KDA_CHECK_ARG(a->block_table && a->cu && a->out, "latent_gather: a required pointer is null");
    KDA_CHECK_ARG(aligned(a->out, 16) && a->out_row % 8 == 0, "latent_gather: out rows must be 16-byte aligned");
    const int64_t wgs = (a->T + TOKENS - 1) / TOKENS;
    launch_kernel(gather_kernel, dim3((uint32_t)wgs), dim3(TOK_THREADS), reinterpret_cast<hipStream_t>(stream), *a);
    return launched("latent_gather");
}

extern "C" int kda355_copy_rows_launch(const KdaPagesArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "copy_rows: null args");
    int segs;
    if (const int rc = check_pools(a, "copy_rows", &segs)) return rc;
    KDA_CHECK_ARG(a->n >= 0 && a->n < MAX_PAIRS, "copy_rows: n=%d", a->n);
    if (a->n == 0 || a->num_pools == 0) return 0;
    KDA_CHECK_ARG(a->src && a->dst, "copy_rows: a required pointer is null");
    launch_kernel(copy_rows_kernel, dim3(a->n, segs, a->num_pools), dim3(COPY_THREADS),
                  reinterpret_cast<hipStream_t>(stream), *a);
    return launched("copy_rows");
}

extern "C" int kda355_fork_pages_launch(const KdaPagesArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "fork_pages: null args");
    int segs;
    if (const int rc = check_pools(a, "fork_pages", &segs)) return rc;
    if (const int rc = check_table(a, "fork_pages", true)) return rc;
    KDA_CHECK_ARG(a->n >= 0 && a->n < MAX_PAIRS, "fork_pages: n=%d", a->n);
    if (a->n == 0) return 0;
    KDA_CHECK_ARG(a->src && a->dst && a->workspace, "fork_pages: a required pointer is null");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    launch_kernel(fork_take_kernel, dim3(1), dim3(SCAN_THREADS), s, *a);
    launch_kernel(fork_rows_kernel, dim3(a->n, segs, a->num_pools + 1), dim3(COPY_THREADS), s, *a);
    return launched("fork_pages");
}

extern "C" int kda355_free_pages_launch(const KdaPagesArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "free_pages: null args");
    if (const int rc = check_table(a, "free_pages", true)) return rc;
    KDA_CHECK_ARG(a->n >= 0 && a->n < MAX_PAIRS, "free_pages: n=%d", a->n);
    if (a->n == 0) return 0;
    KDA_CHECK_ARG(a->src, "free_pages: a required pointer is null");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if ((int64_t)a->n * a->table_width <= FREE_SMALL && a->pages <= FREE_PAGES) {
        launch_kernel(free_small_kernel, dim3(1), dim3(SCAN_THREADS), s, *a);
        return launched("free_pages");
    }
    launch_kernel(free_rows_kernel, dim3(a->n), dim3(COPY_THREADS), s, *a);
    launch_kernel(free_push_kernel, dim3(1), dim3(SCAN_THREADS), s, *a);
    return launched("free_pages");
}

extern "C" int kda355_compact_pages_launch(const KdaPagesArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "compact_pages: null args");
    int segs;
    if (const int rc = check_pools(a, "compact_pages", &segs)) return rc;
    if (const int rc = check_table(a, "compact_pages", false)) return rc;
    KDA_CHECK_ARG(a->workspace, "compact_pages: a required pointer is null");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    launch_kernel(compact_plan_kernel, dim3(1), dim3(SCAN_THREADS), s, *a);
    const int half = a->pages / 2;
    launch_kernel(compact_move_kernel, dim3(half < 1 ? 1 : half, segs, a->num_pools + 1), dim3(COPY_THREADS), s, *a);
    return launched("compact_pages");
}
