// Sequences cut to a budget of tokens by their accumulated weights (gfx950): which tokens of each layer stay, the rows that move, the
// books.  Of a sequence of len > keep tokens the first `fixed` stay (pages that others hold too), the last `recent` stay, and of those between
// the heaviest.  Only what has to move moves: with left = keep - recent, the i-th place below left whose token goes gets the i-th staying
// token from above, and the recent ones follow in order.
//
// 1. A workgroup a (sequence, layer): the weight of the last one that stays, by its bits from the top, 11 at a time over a histogram in LDS;
//    then the places and tokens of the pairs by ranks in index order, and the weights moved; few pairs' rows at once.
// 2. The pairs' rows: no place of a pair is read by another, so all at once.
// 3. The recent rows.  Where they move by their own number or more, all at once.  Else in place: their new places are other recent rows' old
//    ones, so a workgroup takes a strip of columns and walks down, reading a step's rows before it writes any of them (a row moves
//    down, so what is read later has not been written).  Beside it, for few table entries, the books.
// 4. For many entries: table rows, lengths and counts, then what nobody holds any more onto the stack.
// All are bound by memory or, for few tokens, by their launches.
#include "pages.h"

namespace kda355 {
namespace {

constexpr int MOST_ROWS = 1 << 20;
constexpr int PAIRS = 64;                        // of a workgroup at a time
constexpr int MOVE_THREADS = 256;
constexpr int STRIP = 8, SHIFT_ROWS = 4;         // 16-byte pieces of a strip, rows of a thread at a time
constexpr int FEW = 128;                         // pairs that the first kernel moves itself
constexpr int WAVES = SCAN_THREADS / 64, BINS = 2048, SOME = 16 * 1024, ROW_PAGES = 2048;
constexpr int BOOK_ENTRIES = 4096, BOOK_PAGES = 16 * 1024;  // up to so many table entries and pages the books take one workgroup

struct Plan {
    int left;         // keep - recent
    int most;         // pairs of a sequence and layer
    int tail;         // pages that hold the recent tokens, at most
    int strips;       // workgroups of a sequence and layer in the third kernel
    int books;        // the books beside it
};
// workspace: the lengths of the sequences that are cut, -1 for others [n]; pairs of (sequence, layer) [n][layers]; the pages from the
// first recent token's on [n][tail] (the books change the table); places and tokens of the pairs [n][layers][2][most]
__device__ __forceinline__ int32_t* lens_of(const KdaEvictArgs& a) { return static_cast<int32_t*>(a.workspace); }
__device__ __forceinline__ int32_t* pairs_of(const KdaEvictArgs& a, int i, int l) { return lens_of(a) + a.n + i * a.num_layers + l; }
__device__ __forceinline__ int32_t* tail_of(const KdaEvictArgs& a, const Plan& p, int i) {
    return lens_of(a) + a.n + (int64_t)a.n * a.num_layers + (int64_t)i * p.tail;
}
__device__ __forceinline__ int32_t* lists_of(const KdaEvictArgs& a, const Plan& p, int i, int l) {
    return tail_of(a, p, a.n) + ((int64_t)i * a.num_layers + l) * 2 * p.most;
}
__device__ __forceinline__ char* token_in(const KdaEvictArgs& a, const KdaEvictLayer& y, int page, int j) {
    return static_cast<char*>(y.cache) + page * y.page_stride + (int64_t)(j % a.page_size) * y.token_bytes;
}
__device__ __forceinline__ char* token_at(const KdaEvictArgs& a, const KdaEvictLayer& y, int row, int j) {
    return token_in(a, y, a.block_table[row * a.table_stride + j / a.page_size], j);
}
// count rows, from at[1][..] to at[0][..], by THREADS threads
template <int THREADS>
__device__ __forceinline__ void copy_tokens(char* const (*at)[PAIRS], int count, int pieces) {
    const int all = count * pieces;
    for (int k0 = threadIdx.x; k0 < all; k0 += 4 * THREADS) {
        u32x4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = k0 + k * THREADS, pair = e / pieces;
            if (e < all) x[k] = *reinterpret_cast<const u32x4*>(at[1][pair] + (e - pair * pieces) * 16);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int e = k0 + k * THREADS, pair = e / pieces;
            if (e < all) *reinterpret_cast<u32x4*>(at[0][pair] + (e - pair * pieces) * 16) = x[k];
        }
    }
}

// larger weights have larger keys; a NaN has the largest, -0 that of 0
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return ~0u;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ int below(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0)); }

// The keys of the tokens before the recent ones: wave w has a run of them, in rounds of 64 in index order, so that ranks take one exchange
// between the waves.  R > 0: in registers, up to 1024 R of them; R = 0: read anew (from L2) wherever they are needed.
template <int R>
struct Keys {
    const float* weights;
    int first, end, rounds;  // of this wave
    uint32_t k[R ? R : 1];
    __device__ __forceinline__ Keys(const float* w, int stop) : weights(w) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        rounds = ((stop + 63) / 64 + WAVES - 1) / WAVES;
        first = wave * rounds * 64 + lane;
        end = stop;
        if constexpr (R > 0) {
            float x[R];
#pragma unroll
            for (int r = 0; r < R; ++r) x[r] = weights[max(min(first + r * 64, end - 1), 0)];  // (no branches; `weights` has a first one)
#pragma unroll
            for (int r = 0; r < R; ++r) k[r] = key_of(x[r]);
        }
    }
    // f(position, key, is it a candidate: at or after `fixed`) for all rounds, in order
    template <typename F>
    __device__ __forceinline__ void each(int fixed, F f) const {
        auto there = [&](int j) { return j < end && j >= fixed; };
        if constexpr (R > 0) {
#pragma unroll
            for (int r = 0; r < R; ++r)
                if (r < rounds) f(first + r * 64, k[r], there(first + r * 64));
        } else {
            constexpr int U = 16;  // in flight (131072 keys: 10 to 15 us a pass)
            for (int r0 = 0; r0 < rounds; r0 += U) {
                float x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = weights[min(first + (r0 + u) * 64, end - 1)];  // (no branches)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (r0 + u < rounds) f(first + (r0 + u) * 64, key_of(x[u]), there(first + (r0 + u) * 64));
            }
        }
    }
};
// the sum of the waves before this one (x: the same in a wave's lanes); total: of all
__device__ __forceinline__ int before_wave(int x, int* sw, int& total) {
    __syncthreads();  // sw free again
    if ((threadIdx.x & 63) == 0) sw[threadIdx.x >> 6] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
        const int v = sw[i];
        if (i < (int)(threadIdx.x >> 6)) before += v;
        total += v;
    }
    return before;
}

template <int R>
__global__ void __launch_bounds__(SCAN_THREADS) select_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int hist[BINS];
    __shared__ int sw[WAVES];
    __shared__ int flags[6];  // fixed; is there a hole or was the row given before; digit, rank in it, keys with it; keys gathered
    __shared__ char* at[2][PAIRS];
    __shared__ int few[2][FEW];  // the first pairs
    __shared__ uint32_t some[R ? 1 : SOME];
    __shared__ int pages[ROW_PAGES];  // the first of the row's
    const int i = blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    const int row = a.src[i];
    const KdaEvictLayer y = a.layer[l];
    if (tid < 6) flags[tid] = 0;
    hist[tid] = hist[tid + SCAN_THREADS] = 0;
    int len = -1;
    if (row >= 0 && row < a.rows) len = (int)min((int64_t)a.seq_lens[row], (int64_t)a.table_width * a.page_size);
    if (len <= a.keep) len = -1;
    const int end = len - a.recent;  // candidates [fixed, end), `stay` of them stay
    float* const weights = y.weights + (len < 0 ? 0 : row) * y.weights_row;
    const Keys<R> keys(weights, len < 0 ? 0 : end);
    float late[4];  // the first recent ones, for the end
#pragma unroll
    for (int u = 0; u < 4; ++u) late[u] = weights[len < 0 ? 0 : min(end + u * SCAN_THREADS + tid, len - 1)];
    __syncthreads();
    if (len >= 0) {
        const int used = (len + a.page_size - 1) / a.page_size, tail = end / a.page_size;
        int fixed = 0, bad = 0;
        for (int j = tid; j < used; j += SCAN_THREADS) {
            const int page = a.block_table[row * a.table_stride + j];
            if (page < 0 || page >= a.pages) bad = 1;
            else if (a.ref_counts[page] > 1) fixed = (j + 1) * a.page_size;
            if (l == 0 && j >= tail) tail_of(a, p, i)[j - tail] = page;
            if (j < ROW_PAGES) pages[j] = page;
        }
        for (int j = tid; j < i; j += SCAN_THREADS) bad |= a.src[j] == row;
        if (fixed) atomicMax(&flags[0], fixed);
        if (bad) flags[1] = 1;
    }
    __syncthreads();
    const int fixed = flags[0];
    const bool cut = len >= 0 && !flags[1] && fixed <= p.left;
    if (l == 0 && tid == 0) lens_of(a)[i] = cut ? len : -1;
    if (!cut) {
        if (tid == 0) *pairs_of(a, i, l) = 0;
        return;
    }
    int stay = p.left - fixed, total;
    // ---- the key of the last one that stays, how many with this key stay, and whether all with it do
    uint32_t prefix = ~0u;  // none stays: not even a NaN, of which `stay` = 0 do
    bool all = false;
    if (stay > 0) {
        prefix = 0;
        auto pick = [&](uint32_t shift) {  // the digit of the stay-th largest key from the histogram, which is cleared
            __syncthreads();
            // the largest digits first: thread t has 2047 - 2 t and 2046 - 2 t
            const int hi = hist[BINS - 1 - 2 * tid], lo = hist[BINS - 2 - 2 * tid];
            const int before = block_scan(hi + lo, sw, total);
            if (before < stay && stay <= before + hi + lo) {
                const bool upper = stay <= before + hi;
                flags[2] = upper ? BINS - 1 - 2 * tid : BINS - 2 - 2 * tid;
                flags[3] = stay - before - (upper ? 0 : hi);
                flags[4] = upper ? hi : lo;
            }
            hist[BINS - 1 - 2 * tid] = hist[BINS - 2 - 2 * tid] = 0;
            __syncthreads();
            prefix |= (uint32_t)flags[2] << shift;
            stay = flags[3];
            all = stay == flags[4];
        };
        auto count = [&](uint32_t k, bool there, uint32_t mask, uint32_t shift, uint32_t bins) {
            if (there && (k & mask) == prefix) atomicAdd(&hist[k >> shift & bins], 1);
        };
        keys.each(fixed, [&](int, uint32_t k, bool there) { count(k, there, 0, 21, 2047); });
        pick(21);
        if (R == 0 && flags[4] <= SOME) {  // the other digits over the keys that have the first one, gathered in LDS
            keys.each(fixed, [&](int, uint32_t k, bool there) {
                if (there && (k & ~0u << 21) == prefix) some[atomicAdd(&flags[5], 1)] = k;
            });
            __syncthreads();
            const int n = flags[5];
            for (int j = tid; j < n; j += SCAN_THREADS) count(some[j], true, ~0u << 21, 10, 2047);
            pick(10);
            for (int j = tid; j < n; j += SCAN_THREADS) count(some[j], true, ~0u << 10, 0, 1023);
        } else {
            keys.each(fixed, [&](int, uint32_t k, bool there) { count(k, there, ~0u << 21, 10, 2047); });
            pick(10);
            keys.each(fixed, [&](int, uint32_t k, bool there) { count(k, there, ~0u << 10, 0, 1023); });
        }
        pick(0);
    }
    // ---- places below left whose token goes, tokens from left on that stay, in index order
    int32_t* const places = lists_of(a, p, i, l);
    int32_t* const tokens = places + p.most;
    int ties = 0;
    if (!all) {  // the first `stay` of those with the key stay
        keys.each(fixed, [&](int, uint32_t k, bool there) { ties += __popcll(__builtin_amdgcn_ballot_w64(there && k == prefix)); });
        ties = before_wave(ties, sw, total);
    }
    int holes = 0, movers = 0;
    auto marks = [&](auto f) {  // f(position, is it a hole, is it a mover, their ballots)
        int t = ties;
        keys.each(fixed, [&](int j, uint32_t k, bool there) {
            bool stays = there && k >= prefix;
            if (!all) {
                const bool tie = there && k == prefix;
                const uint64_t tied = __builtin_amdgcn_ballot_w64(tie);
                if (tie) stays = t + below(tied) < stay;
                t += __popcll(tied);
            }
            const bool hole = there && !stays && j < p.left, mover = stays && j >= p.left;
            f(j, hole, mover, __builtin_amdgcn_ballot_w64(hole), __builtin_amdgcn_ballot_w64(mover));
        });
    };
    marks([&](int, bool, bool, uint64_t h, uint64_t m) { holes += __popcll(h), movers += __popcll(m); });
    int pairs;
    holes = before_wave(holes, sw, pairs);
    movers = before_wave(movers, sw, total);  // (as many)
    const bool few_pairs = pairs <= FEW;
    marks([&](int j, bool hole, bool mover, uint64_t h, uint64_t m) {
        if (hole) (few_pairs ? few[0] : places)[holes + below(h)] = j;
        if (mover) (few_pairs ? few[1] : tokens)[movers + below(m)] = j;
        holes += __popcll(h), movers += __popcll(m);
    });
    if (tid == 0) *pairs_of(a, i, l) = pairs;
    __syncthreads();  // the lists are written
    // ---- few rows; the weights
    if (few_pairs) {
        if (tid < pairs) weights[few[0][tid]] = weights[few[1][tid]];
        for (int first = 0; first < pairs; first += PAIRS) {
            const int n = min(pairs - first, PAIRS);
            if (tid < 2 * PAIRS && tid % PAIRS < n) {
                const int j = few[tid / PAIRS][first + tid % PAIRS], col = j / a.page_size;
                at[tid / PAIRS][tid % PAIRS] = token_in(a, y, col < ROW_PAGES ? pages[col] : a.block_table[row * a.table_stride + col], j);
            }
            __syncthreads();
            copy_tokens<SCAN_THREADS>(at, n, (int)(y.token_bytes / 16));
            __syncthreads();
        }
    } else {
        for (int k0 = tid; k0 < pairs; k0 += 8 * SCAN_THREADS) {
            int from[8], to[8];
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int k = min(k0 + u * SCAN_THREADS, pairs - 1);
                from[u] = load_fresh(tokens + k), to[u] = load_fresh(places + k);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = weights[from[u]];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (k0 + u * SCAN_THREADS < pairs) weights[to[u]] = x[u];
        }
    }
    __syncthreads();
    for (int k0 = 0; k0 < a.recent; k0 += 4 * SCAN_THREADS) {
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + u * SCAN_THREADS + tid;
            x[u] = k0 == 0 ? late[u] : k < a.recent ? weights[end + k] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = k0 + u * SCAN_THREADS + tid;
            if (k < a.recent) weights[p.left + k] = x[u];
        }
        __syncthreads();
    }
    for (int j = a.keep + tid; j < len; j += SCAN_THREADS) weights[j] = 0.f;
}

__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(KdaEvictArgs a, Plan p) {
    __shared__ char* at[2][PAIRS];
    const int i = blockIdx.y, l = blockIdx.z;
    const int pairs = *pairs_of(a, i, l);
    if (pairs <= FEW) return;
    const int32_t* lists = lists_of(a, p, i, l);
    const KdaEvictLayer y = a.layer[l];
    const int row = a.src[i], pieces = (int)(y.token_bytes / 16);
    for (int first = blockIdx.x * PAIRS; first < pairs; first += gridDim.x * PAIRS) {
        const int count = min(pairs - first, PAIRS);
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * PAIRS; k += MOVE_THREADS)
            if (k % PAIRS < count) at[k / PAIRS][k % PAIRS] = token_at(a, y, row, lists[(int64_t)(k / PAIRS) * p.most + first + k % PAIRS]);
        __syncthreads();
        copy_tokens<MOVE_THREADS>(at, count, pieces);
    }
}

// A row's first pages stay, the rest of its tokens' pages go, entries past the tokens follow the first ones.
__device__ __forceinline__ void book(const KdaEvictArgs& a, int i) {
    const int len = lens_of(a)[i];
    if (len < 0) return;
    const int row = a.src[i];
    const int used = (len + a.page_size - 1) / a.page_size, kept = (a.keep + a.page_size - 1) / a.page_size;
    int32_t* table = a.block_table + row * a.table_stride;
    for (int j = kept + threadIdx.x; j < used; j += blockDim.x) atomicCAS(a.ref_counts + table[j], 1, FREED);  // (none is held twice)
    __syncthreads();
    const int by = used - kept;
    if (by > 0)
        for (int j0 = kept; j0 < a.table_width; j0 += blockDim.x) {
            const int j = j0 + threadIdx.x;
            const int32_t next = j + by < a.table_width ? table[j + by] : -1;
            __syncthreads();
            if (j < a.table_width) table[j] = next;
            __syncthreads();
        }
    if (threadIdx.x == 0) a.seq_lens[row] = a.keep;
}

__global__ void __launch_bounds__(MOVE_THREADS) books_kernel(KdaEvictArgs a) { book(a, blockIdx.x); }

__global__ void __launch_bounds__(SCAN_THREADS) shift_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int sw[WAVES];
    __shared__ char* at[2][PAIRS];
    const int i = blockIdx.y, l = blockIdx.z, tid = threadIdx.x;
    if ((int)blockIdx.x == p.strips) {  // the books, by one workgroup
        if (i || l) return;
        for (int k = 0; k < a.n; ++k) book(a, k);
        __syncthreads();
        push_freed<true>(a.ref_counts, a.free_pages, a.num_free, a.pages, sw);
        return;
    }
    const int len = lens_of(a)[i];
    if (len < 0) return;
    const KdaEvictLayer y = a.layer[l];
    const int row = a.src[i], pieces = (int)(y.token_bytes / 16), end = len - a.recent;
    const int32_t* tail = tail_of(a, p, i);
    const int first_page = end / a.page_size;
    // The places are below keep: their pages stay where they are in the table, unlike those of the tokens.
    auto token = [&](int k) { return token_in(a, y, tail[(end + k) / a.page_size - first_page], end + k); };
    auto place = [&](int k) { return token_at(a, y, row, p.left + k); };
    if (len - a.keep >= a.recent) {
        for (int first = blockIdx.x * PAIRS; first < a.recent; first += p.strips * PAIRS) {
            const int count = min(a.recent - first, PAIRS);
            __syncthreads();
            if (tid < 2 * PAIRS && tid % PAIRS < count) at[tid / PAIRS][tid % PAIRS] = tid < PAIRS ? place(first + tid) : token(first + tid - PAIRS);
            __syncthreads();
            copy_tokens<SCAN_THREADS>(at, count, pieces);
        }
        return;
    }
    const int piece = blockIdx.x * STRIP + tid % STRIP;
    if ((int)blockIdx.x * STRIP >= pieces) return;
    constexpr int STEP = SCAN_THREADS / STRIP;  // rows of a step's part
    const bool some = piece < pieces;
    for (int k0 = tid / STRIP; k0 - tid / STRIP < a.recent; k0 += SHIFT_ROWS * STEP) {
        u32x4 x[SHIFT_ROWS];
#pragma unroll
        for (int s = 0; s < SHIFT_ROWS; ++s)
            if (some && k0 + s * STEP < a.recent) x[s] = *reinterpret_cast<const u32x4*>(token(k0 + s * STEP) + piece * 16);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < SHIFT_ROWS; ++s)
            if (some && k0 + s * STEP < a.recent) *reinterpret_cast<u32x4*>(place(k0 + s * STEP) + piece * 16) = x[s];
        __syncthreads();  // (a later step reads no place that an earlier one wrote)
    }
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
    p.tail = (int)((a->recent + a->page_size - 1) / a->page_size + 1);
    return p;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int64_t kda355_evict_tokens_workspace_bytes(const KdaEvictArgs* a) {
    if (const int rc = check_evict(a)) return rc;
    const int64_t lists = (int64_t)a->n * a->num_layers;
    const Plan p = plan_of(a);
    return 4 * (a->n * (1 + (int64_t)p.tail) + lists * (1 + 2 * (int64_t)p.most));
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
    const int lists = a->n * a->num_layers;
    const int64_t fill = 4096 / lists + 1;  // workgroups of a sequence and layer
    const auto some = [](int64_t x, int64_t y) { return (int)(x < y ? x : y); };
    const auto cdiv = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    // the candidates: at most all tokens but the recent ones
    const int64_t most = span - a->recent;
    launch_kernel(most <= 4 * SCAN_THREADS ? select_kernel<4> : most <= 16 * SCAN_THREADS ? select_kernel<16> : select_kernel<0>,
                  dim3(a->n, a->num_layers), dim3(SCAN_THREADS), s, *a, p);
    if (p.most > FEW)
        launch_kernel(move_kernel, dim3(some(cdiv(p.most, PAIRS), fill), a->n, a->num_layers), dim3(MOVE_THREADS), s, *a, p);
    const bool last = !(a->flags & KDA355_EVICT_MORE);
    const int strips = (int)cdiv(pieces, STRIP), parts = some(cdiv(a->recent, PAIRS), fill / 4 + 1);
    p.strips = a->recent == 0 ? 0 : strips > parts ? strips : parts;
    p.books = last && (int64_t)a->n * a->table_width <= BOOK_ENTRIES && a->pages <= BOOK_PAGES;
    if (p.strips + p.books)
        launch_kernel(shift_kernel, dim3(p.strips + p.books, p.strips ? a->n : 1, p.strips ? a->num_layers : 1), dim3(SCAN_THREADS), s, *a, p);
    if (last && !p.books) {
        launch_kernel(books_kernel, dim3(a->n), dim3(MOVE_THREADS), s, *a);
        KdaPagesArgs b = {};
        b.ref_counts = a->ref_counts, b.free_pages = a->free_pages, b.num_free = a->num_free, b.pages = a->pages;
        launch_kernel(free_push_kernel, dim3(1), dim3(SCAN_THREADS), s, b);
    }
    return launched("evict_tokens");
}
