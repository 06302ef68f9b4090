// Sequences cut to a budget of tokens by their accumulated weights (gfx950): which tokens of each layer stay, the rows that move, the
// books.  Of a sequence of len > keep tokens the first `fixed` stay (pages that others hold too), the last `recent` stay, and of those between
// the heaviest.  Only what has to move moves: with left = keep - recent, the i-th place below left whose token goes gets the i-th staying
// token from above, and the recent ones follow in order.
//
// 1. A workgroup a (sequence, layer): the weight of the last one that stays, by its bits from the top, eight at a time over a histogram in LDS; then
//    the places and tokens of the pairs by ranks in index order, and the weights moved.
// 2. The pairs' rows: no place of a pair is read by another, so all at once.
// 3. The recent rows, in place: their new places may be other recent rows' old ones, so a workgroup takes a strip of columns and walks
//    down, reading a step's rows before it writes any of them (a row moves down, so what is read later has not been written).
// 4. Table rows, lengths and counts, and what nobody holds any more onto the stack.
// All are bound by memory or, for few tokens, by their launches.
#include "pages.h"

namespace kda355 {
namespace {

constexpr int MOST_ROWS = 1 << 20;
constexpr int PAIRS = 64;                        // of a workgroup at a time
constexpr int MOVE_THREADS = 256;
constexpr int STRIP = 8, SHIFT_ROWS = 4;         // 16-byte pieces of a strip, rows of a thread at a time

struct Plan {
    int left;         // keep - recent
    int most;         // pairs of a sequence and layer
    int move_grid;
};
// workspace: the lengths of the sequences that are cut, -1 for others [n]; pairs of (sequence, layer) [n][layers]; their
// places and tokens [n][layers][2][most]
__device__ __forceinline__ int32_t* lens_of(const KdaEvictArgs& a) { return static_cast<int32_t*>(a.workspace); }
__device__ __forceinline__ int32_t* pairs_of(const KdaEvictArgs& a, int i, int l) { return lens_of(a) + a.n + i * a.num_layers + l; }
__device__ __forceinline__ int32_t* lists_of(const KdaEvictArgs& a, const Plan& p, int i, int l) {
    return lens_of(a) + a.n + (int64_t)a.n * a.num_layers + ((int64_t)i * a.num_layers + l) * 2 * p.most;
}
__device__ __forceinline__ char* token_at(const KdaEvictArgs& a, const KdaEvictLayer& y, int row, int j) {
    const int col = j / a.page_size, page = a.block_table[row * a.table_stride + col];
    return static_cast<char*>(y.cache) + page * y.page_stride + (int64_t)(j - col * a.page_size) * y.token_bytes;
}

// larger weights have larger keys; a NaN has the largest, -0 that of 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return ~0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__global__ void __launch_bounds__(SCAN_THREADS) select_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int hist[256];
    __shared__ int sw[SCAN_THREADS / 64];
    __shared__ int flags[4];  // fixed, is there a hole, given before; digit, rank in it
    const int i = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    const int row = a.src[i];
    const KdaEvictLayer y = a.layer[l];
    if (tid < 4) flags[tid] = 0;
    __syncthreads();
    int len = -1;
    if (row >= 0 && row < a.rows) {
        const int64_t most = (int64_t)a.table_width * a.page_size;
        len = (int)min((int64_t)a.seq_lens[row], most);
        if (len > a.keep) {
            const int used = (len + a.page_size - 1) / a.page_size;
            int fixed = 0, bad = 0;
            for (int j = tid; j < used; j += SCAN_THREADS) {
                const int page = a.block_table[row * a.table_stride + j];
                if (page < 0 || page >= a.pages) bad = 1;
                else if (a.ref_counts[page] > 1) fixed = (int)min((int64_t)(j + 1) * a.page_size, (int64_t)INT32_MAX);
            }
            for (int j = tid; j < i; j += SCAN_THREADS) bad |= a.src[j] == row;
            if (fixed) atomicMax(&flags[0], fixed);
            if (bad) flags[1] = 1;
        }
    }
    __syncthreads();
    const int fixed = flags[0];
    const bool cut = len > a.keep && !flags[1] && fixed <= p.left;
    if (l == 0 && tid == 0) lens_of(a)[i] = cut ? len : -1;
    if (!cut) {
        if (tid == 0) *pairs_of(a, i, l) = 0;
        return;
    }
    float* const weights = y.weights + row * y.weights_row;
    const int end = len - a.recent;  // candidates [fixed, end), `stay` of them stay
    int stay = p.left - fixed;
    __syncthreads();
    // ---- the key of the last one that stays, and how many with this key stay
    uint32_t prefix = 0, mask = 0;
    if (stay > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = fixed + tid; j < end; j += SCAN_THREADS) {
                const uint32_t k = key_of(weights[j]);
                if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & 255], 1);
            }
            __syncthreads();
            const int mine = tid < 256 ? hist[255 - tid] : 0;
            int total;
            const int before = block_scan(mine, sw, total);
            if (before < stay && stay <= before + mine) {
                flags[2] = 255 - tid;
                flags[3] = stay - before;
            }
            __syncthreads();
            prefix |= (uint32_t)flags[2] << shift;
            mask |= 255u << shift;
            stay = flags[3];
            __syncthreads();
        }
    } else {
        prefix = ~0u, stay = 0;  // none stays (with a NaN's key: none of them)
    }
    // ---- places below left whose token goes, tokens from left on that stay, in index order
    int32_t* const places = lists_of(a, p, i, l);
    int32_t* const tokens = places + p.most;
    int ties = 0, holes = 0, movers = 0;
    for (int j0 = fixed; j0 < end; j0 += SCAN_THREADS) {
        const int j = j0 + tid;
        const uint32_t k = j < end ? key_of(weights[j]) : 0u;
        const bool tie = j < end && k == prefix;
        int total;
        const int rank = ties + block_scan(tie, sw, total);
        ties += total;
        const bool stays = j < end && (k > prefix || (tie && rank < stay));
        const int hole = j < p.left && j < end && !stays, mover = j >= p.left && stays;
        const int at = block_scan(hole | mover << 16, sw, total);
        if (hole) places[holes + (at & 0xffff)] = j;
        if (mover) tokens[movers + (at >> 16)] = j;
        holes += total & 0xffff;
        movers += total >> 16;
    }
    if (tid == 0) *pairs_of(a, i, l) = holes;
    __syncthreads();  // the lists are written (as many places as tokens)
    // ---- the weights
    for (int k = tid; k < holes; k += SCAN_THREADS) weights[load_fresh(places + k)] = weights[load_fresh(tokens + k)];
    __syncthreads();
    for (int k0 = 0; k0 < a.recent; k0 += SCAN_THREADS) {
        const int k = k0 + tid;
        const float x = k < a.recent ? weights[end + k] : 0.f;
        __syncthreads();
        if (k < a.recent) weights[p.left + k] = x;
        __syncthreads();
    }
    for (int j = a.keep + tid; j < len; j += SCAN_THREADS) weights[j] = 0.f;
}

__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(KdaEvictArgs a, Plan p) {
    __shared__ char* at[2][PAIRS];
    const int i = blockIdx.y, l = blockIdx.z;
    const int pairs = *pairs_of(a, i, l);
    if ((int)blockIdx.x * PAIRS >= pairs) return;
    const int32_t* lists = lists_of(a, p, i, l);
    const KdaEvictLayer y = a.layer[l];
    const int row = a.src[i], pieces = (int)(y.token_bytes / 16);
    for (int first = blockIdx.x * PAIRS; first < pairs; first += gridDim.x * PAIRS) {
        const int count = min(pairs - first, PAIRS);
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * count; k += MOVE_THREADS) {
            const int which = k >= count, pair = which ? k - count : k;
            at[which][pair] = token_at(a, y, row, lists[(int64_t)which * p.most + first + pair]);
        }
        __syncthreads();
        const int all = count * pieces;
        for (int k0 = threadIdx.x; k0 < all; k0 += 4 * MOVE_THREADS) {
            u32x4 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = k0 + k * MOVE_THREADS, pair = e / pieces;
                if (e < all) x[k] = *reinterpret_cast<const u32x4*>(at[1][pair] + (e - pair * pieces) * 16);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int e = k0 + k * MOVE_THREADS, pair = e / pieces;
                if (e < all) *reinterpret_cast<u32x4*>(at[0][pair] + (e - pair * pieces) * 16) = x[k];
            }
        }
    }
}

__global__ void __launch_bounds__(SCAN_THREADS) shift_kernel(KdaEvictArgs a, Plan p) {
    const int i = blockIdx.y, l = blockIdx.z;
    const int len = lens_of(a)[i];
    if (len < 0) return;
    const KdaEvictLayer y = a.layer[l];
    const int row = a.src[i], pieces = (int)(y.token_bytes / 16), piece = blockIdx.x * STRIP + threadIdx.x % STRIP;
    constexpr int STEP = SCAN_THREADS / STRIP;  // rows of a step's part
    const int first = threadIdx.x / STRIP;
    const bool some = piece < pieces;
    for (int k0 = 0; k0 < a.recent; k0 += SHIFT_ROWS * STEP) {
        u32x4 x[SHIFT_ROWS];
#pragma unroll
        for (int s = 0; s < SHIFT_ROWS; ++s) {
            const int k = k0 + s * STEP + first;
            if (some && k < a.recent) x[s] = *reinterpret_cast<const u32x4*>(token_at(a, y, row, len - a.recent + k) + piece * 16);
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < SHIFT_ROWS; ++s) {
            const int k = k0 + s * STEP + first;
            if (some && k < a.recent) *reinterpret_cast<u32x4*>(token_at(a, y, row, p.left + k) + piece * 16) = x[s];
        }
        __syncthreads();  // (a later step reads no place that an earlier one wrote)
    }
}

// The row's first pages stay, the rest of its tokens' pages go, entries past the tokens follow the first ones.
__global__ void __launch_bounds__(MOVE_THREADS) books_kernel(KdaEvictArgs a) {
    const int i = blockIdx.x;
    const int len = lens_of(a)[i];
    if (len < 0) return;
    const int row = a.src[i];
    const int used = (len + a.page_size - 1) / a.page_size, kept = (a.keep + a.page_size - 1) / a.page_size;
    int32_t* table = a.block_table + row * a.table_stride;
    for (int j = kept + threadIdx.x; j < used; j += MOVE_THREADS) atomicCAS(a.ref_counts + table[j], 1, FREED);  // (none is held twice)
    __syncthreads();
    const int by = used - kept;
    if (by > 0)
        for (int j0 = kept; j0 < a.table_width; j0 += MOVE_THREADS) {
            const int j = j0 + threadIdx.x;
            const int32_t next = j + by < a.table_width ? table[j + by] : -1;
            __syncthreads();
            if (j < a.table_width) table[j] = next;
            __syncthreads();
        }
    if (threadIdx.x == 0) a.seq_lens[row] = a.keep;
}

int check_evict(const KdaEvictArgs* a) {
    KDA_CHECK_ARG(a != nullptr, "evict_tokens: null args");
    KDA_CHECK_ARG(a->num_layers >= 0 && a->num_layers <= KDA355_MAX_POOLS && a->n >= 0 && a->n < MOST_ROWS, "evict_tokens: num_layers=%d n=%d",
                  a->num_layers, a->n);
    KDA_CHECK_ARG(a->rows >= 1 && a->table_width >= 1 && a->pages >= 1 && a->page_size >= 1,
                  "evict_tokens: rows=%d table_width=%d pages=%d page_size=%d", a->rows, a->table_width, a->pages, a->page_size);
    KDA_CHECK_ARG((int64_t)a->table_width * a->page_size < (1ll << 30), "evict_tokens: a table row spans 2^30 tokens or more");
    KDA_CHECK_ARG(a->keep >= 1 && a->recent >= 0 && a->recent <= a->keep, "evict_tokens: keep=%d recent=%d", a->keep, a->recent);
    return 0;
}

Plan plan_of(const KdaEvictArgs* a) {
    Plan p;
    const int64_t span = (int64_t)a->table_width * a->page_size;
    p.left = a->keep - a->recent;
    const int64_t goes = span - a->keep;  // no more tokens go from below `left` than go in all
    p.most = (int)(goes <= 0 ? 0 : goes < p.left ? goes : p.left);
    return p;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int64_t kda355_evict_tokens_workspace_bytes(const KdaEvictArgs* a) {
    if (const int rc = check_evict(a)) return rc;
    const int64_t lists = (int64_t)a->n * a->num_layers;
    return 4 * (a->n + lists * (1 + 2 * (int64_t)plan_of(a).most));
}

extern "C" int kda355_evict_tokens_launch(const KdaEvictArgs* a, kda355_stream_t stream) {
    if (const int rc = check_evict(a)) return rc;
    KDA_CHECK_ARG((a->flags & ~KDA355_EVICT_MORE) == 0, "evict_tokens: unknown flags 0x%x", a->flags);
    KDA_CHECK_ARG(a->table_stride >= a->table_width, "evict_tokens: table_stride < table_width");
    KDA_CHECK_ARG(a->num_layers >= 1, "evict_tokens: no layers");
    const int64_t span = (int64_t)a->table_width * a->page_size;
    int64_t pieces = 1;
    for (int l = 0; l < a->num_layers; ++l) {
        const KdaEvictLayer& y = a->layer[l];
        KDA_CHECK_ARG(y.cache && y.weights, "evict_tokens: layer %d: a required pointer is null", l);
        KDA_CHECK_ARG(aligned(y.cache, 16) && y.token_bytes > 0 && y.token_bytes % 16 == 0 && y.token_bytes < (1 << 20) && y.page_stride % 16 == 0 &&
                          y.page_stride >= a->page_size * y.token_bytes,
                      "evict_tokens: the tokens of layer %d must be a multiple of 16 bytes, aligned and dense within a page", l);
        KDA_CHECK_ARG(y.weights_row >= span, "evict_tokens: rows of weights %d are shorter than the table's tokens", l);
        pieces = y.token_bytes / 16 > pieces ? y.token_bytes / 16 : pieces;
    }
    if (a->n == 0 || span <= a->keep) return 0;  // (no row can be longer)
    KDA_CHECK_ARG(a->src && a->block_table && a->seq_lens && a->ref_counts && a->free_pages && a->num_free, "evict_tokens: a required pointer is null");
    const int64_t need = kda355_evict_tokens_workspace_bytes(a);
    KDA_CHECK_ARG(a->workspace && aligned(a->workspace, 16) && a->workspace_bytes >= need, "evict_tokens: needs %lld bytes of 16-byte aligned workspace",
                  (long long)need);
    KDA_CHECK_ARG((int64_t)a->n <= 65535, "evict_tokens: %d rows in one call (at most 65535)", a->n);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    Plan p = plan_of(a);
    const int64_t chunks = ((int64_t)p.most + PAIRS - 1) / PAIRS, fill = 4096 / (a->n * a->num_layers) + 1;
    p.move_grid = (int)(chunks < fill ? chunks : fill);
    launch_kernel(select_kernel, dim3(a->n, a->num_layers), dim3(SCAN_THREADS), s, *a, p);
    if (p.move_grid) launch_kernel(move_kernel, dim3(p.move_grid, a->n, a->num_layers), dim3(MOVE_THREADS), s, *a, p);
    if (a->recent) launch_kernel(shift_kernel, dim3((uint32_t)((pieces + STRIP - 1) / STRIP), a->n, a->num_layers), dim3(SCAN_THREADS), s, *a, p);
    if (!(a->flags & KDA355_EVICT_MORE)) {
        launch_kernel(books_kernel, dim3(a->n), dim3(MOVE_THREADS), s, *a);
        KdaPagesArgs b = {};
        b.ref_counts = a->ref_counts, b.free_pages = a->free_pages, b.num_free = a->num_free, b.pages = a->pages;
        launch_kernel(free_push_kernel, dim3(1), dim3(SCAN_THREADS), s, b);
    }
    return launched("evict_tokens");
}
