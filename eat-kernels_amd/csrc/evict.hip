// Sequences cut to a budget of tokens by their accumulated weights (gfx950): which tokens of each layer stay, the rows that move, the
// books.  Of a sequence of len > keep tokens the first `fixed` stay (pages that others hold too), the last `recent` stay, and of those between
// the heaviest.  Only what has to move moves: with left = keep - recent, the i-th place below left whose token goes gets the i-th staying
// token from above, and the recent ones follow in order.
//
// 1. A workgroup a (sequence, layer): the weight of the last one that stays, by its bits from the top, 11 at a time over a histogram in LDS;
//    then the places and tokens of the pairs by ranks in index order, and the weights moved; few pairs' rows at once.  Long sequences by a
//    workgroup for 8192 tokens, with a launch for each digit, one for the parts' counts and one for the lists; the weights go with the rows.
// 2. The pairs' rows: no place of a pair is read by another, so all at once.
// 3. The recent rows.  Where they move by their own number or more, all at once.  Else in place: their new places are other recent rows' old
//    ones, so a workgroup takes a strip of columns and walks down, reading a step's rows before it writes any of them (a row moves
//    down, so what is read later has not been written).  Beside them the books: table rows, lengths and counts, and for few of them what
//    nobody holds any more onto the stack.
// 4. For many: that.
// The rows are bound by memory (2 and 3 for 800 MB: 180 us, 4.5 TB/s), the rest by the latency of its steps: 1 takes 13 us for one sequence
// of 4160 tokens, 18 for 64 in 4 layers, 39 for 131072 and 100001 in 7.
#include "pages.h"

namespace kda355 {
namespace {

constexpr int MOST_ROWS = 1 << 20;
constexpr int PAIRS = 64;                        // of a workgroup at a time
constexpr int MOVE_THREADS = 256;
constexpr int STRIP = 8, SHIFT_ROWS = 4;         // 16-byte pieces of a strip, rows of a thread at a time
constexpr int FEW = 128;                         // pairs that the first kernel moves itself
constexpr int WAVES = SCAN_THREADS / 64, BINS = 2048, ROW_PAGES = 2048;
constexpr int PART_KEYS = 8, PART = PART_KEYS * SCAN_THREADS;  // of a thread, of a workgroup
// Pairs of so many (sequence, layer)s at once, and so many bytes of them (if not of a single sequence): a table's tokens, not the sequences',
// set a list's length, and all lists of 256 rows that hold 131072 tokens in 24 layers would be 1.5 GiB.
constexpr int AT_ONCE = 1024;
constexpr int64_t LIST_BYTES = 128 << 20;
constexpr int BOOK_ROWS = 64, BOOK_ENTRIES = 4096, BOOK_PAGES = 16 * 1024;  // up to so many rows, table entries and pages the books take one workgroup

enum { ROWS = 1, ALL };
struct Plan {
    int left;         // keep - recent
    int most;         // pairs of a sequence and layer
    int tail;         // pages that hold the recent tokens, at most
    int strips;       // workgroups of a sequence and layer in the third kernel
    int books;        // the books beside it: none, by a workgroup for each sequence, all by one
    int parts;        // workgroups that select for a sequence and layer, 0: one
    int first, rows;  // sequences of this run
};
// workspace: the lengths of the sequences that are cut, -1 for others [n]; pairs of (sequence, layer) [n][layers]; the pages from the
// first recent token's on [n][tail] (the books change the table); of a run of sequences the places and tokens of the pairs
// [rows][layers][2][most]; with parts: the tokens that stay for being held elsewhere [n], and of a run histograms [rows][layers][3][BINS]
// and counts of the parts [rows][layers][parts][4]
__device__ __forceinline__ int32_t* lens_of(const KdaEvictArgs& a) { return static_cast<int32_t*>(a.workspace); }
__device__ __forceinline__ int32_t* pairs_of(const KdaEvictArgs& a, int i, int l) { return lens_of(a) + a.n + i * a.num_layers + l; }
__device__ __forceinline__ int32_t* tail_of(const KdaEvictArgs& a, const Plan& p, int i) {
    return lens_of(a) + a.n + (int64_t)a.n * a.num_layers + (int64_t)i * p.tail;
}
__device__ __forceinline__ int32_t* lists_of(const KdaEvictArgs& a, const Plan& p, int i, int l) {  // i: of the run, from here on
    return tail_of(a, p, a.n) + ((int64_t)i * a.num_layers + l) * 2 * p.most;
}
__device__ __forceinline__ int32_t* fixed_of(const KdaEvictArgs& a, const Plan& p) { return lists_of(a, p, p.rows, 0); }
__device__ __forceinline__ int32_t* hist_of(const KdaEvictArgs& a, const Plan& p, int i, int l) {
    return fixed_of(a, p) + a.n + ((int64_t)i * a.num_layers + l) * 3 * BINS;
}
__device__ __forceinline__ int32_t* counts_of(const KdaEvictArgs& a, const Plan& p, int i, int l) {
    return hist_of(a, p, p.rows, 0) + ((int64_t)i * a.num_layers + l) * 4 * p.parts;
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

// The keys of tokens from .. stop - 1, up to 1024 R of them, in registers: wave w has a run of them, in rounds of 64 in index order, so that
// ranks take one exchange between the waves.
template <int R>
struct Keys {
    int first, end, rounds;  // of this wave
    uint32_t k[R];
    __device__ __forceinline__ Keys(const float* weights, int from, int stop) {
        rounds = ((stop - from + 63) / 64 + WAVES - 1) / WAVES;
        first = from + (threadIdx.x >> 6) * rounds * 64 + (threadIdx.x & 63);
        end = stop;
        float x[R];
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = weights[max(min(first + r * 64, end - 1), 0)];  // (no branches; `weights` has a first one)
#pragma unroll
        for (int r = 0; r < R; ++r) k[r] = key_of(x[r]);
    }
    // f(position, key, is it a candidate: at or after `fixed`) for all rounds, in order
    template <typename F>
    __device__ __forceinline__ void each(int fixed, F f) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = first + r * 64;
            if (r < rounds) f(j, k[r], j < end && j >= fixed);
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

// tokens of the row in slot i, -1 where nothing is to be cut
__device__ __forceinline__ int length_of(const KdaEvictArgs& a, int row) {
    int len = -1;
    if (row >= 0 && row < a.rows) len = (int)min((int64_t)a.seq_lens[row], (int64_t)a.table_width * a.page_size);
    return len <= a.keep ? -1 : len;
}
// The tokens that stay for being held elsewhere into flags[0], whether there is a hole or the row was given before into flags[1] (zeros
// before, a barrier after); the pages of the recent tokens, if `tail`; the first pages into `pages`, if there is such a list.
__device__ __forceinline__ void look(const KdaEvictArgs& a, const Plan& p, int i, int row, int len, int* flags, bool tail, int* pages) {
    const int used = (len + a.page_size - 1) / a.page_size, from = (len - a.recent) / a.page_size;
    int fixed = 0, bad = 0;
    for (int j = threadIdx.x; j < used; j += SCAN_THREADS) {
        const int page = a.block_table[row * a.table_stride + j];
        if (page < 0 || page >= a.pages) bad = 1;
        else if (a.ref_counts[page] > 1) fixed = (j + 1) * a.page_size;
        if (tail && j >= from) tail_of(a, p, i)[j - from] = page;
        if (pages && j < ROW_PAGES) pages[j] = page;
    }
    for (int j = threadIdx.x; j < i; j += SCAN_THREADS) bad |= a.src[j] == row;
    if (fixed) atomicMax(&flags[0], fixed);
    if (bad) flags[1] = 1;
}

// The stay-th largest key, digit by digit from the top: 11 bits, 11 and 10.
struct Last {
    uint32_t prefix;  // its digits so far; ~0 if none stays (not even a NaN, of which `stay` = 0 do)
    int stay;         // how many with these digits stay
    bool all;         // whether all do
    __device__ __forceinline__ explicit Last(int n) : prefix(n > 0 ? 0u : ~0u), stay(n), all(false) {}
    static __device__ __forceinline__ int shift(int digit) { return digit == 0 ? 21 : digit == 1 ? 10 : 0; }
    // histogram of a digit over the keys with the digits before it
    __device__ __forceinline__ void count(int* hist, int digit, uint32_t k, bool there) const {
        const uint32_t mask = digit == 0 ? 0u : ~0u << shift(digit - 1);
        if (there && (k & mask) == prefix) atomicAdd(&hist[k >> shift(digit) & (digit < 2 ? 2047 : 1023)], 1);
    }
    // the digit from the histogram, which is cleared; found: 3 words in LDS
    __device__ __forceinline__ void pick(int* hist, int digit, int* found, int* sw) {
        const int t = threadIdx.x;
        int total;
        __syncthreads();
        // the largest digits first: thread t has 2047 - 2 t and 2046 - 2 t
        const int hi = hist[BINS - 1 - 2 * t], lo = hist[BINS - 2 - 2 * t];
        const int before = block_scan(hi + lo, sw, total);
        if (before < stay && stay <= before + hi + lo) {
            const bool upper = stay <= before + hi;
            found[0] = upper ? BINS - 1 - 2 * t : BINS - 2 - 2 * t;
            found[1] = stay - before - (upper ? 0 : hi);
            found[2] = upper ? hi : lo;
        }
        hist[BINS - 1 - 2 * t] = hist[BINS - 2 - 2 * t] = 0;
        __syncthreads();
        prefix |= (uint32_t)found[0] << shift(digit);
        stay = found[1];
        all = stay == found[2];
    }
    // f(position, is it a hole: a place below left whose token goes, is it a mover: a token from left on that stays, their ballots); ties:
    // tokens with the key before this wave's
    template <int R, typename F>
    __device__ __forceinline__ void marks(const Keys<R>& keys, int fixed, int left, int ties, F f) const {
        keys.each(fixed, [&](int j, uint32_t k, bool there) {
            bool stays = there && k >= prefix;
            if (!all) {  // the first `stay` of those with the key stay
                const bool tie = there && k == prefix;
                const uint64_t tied = __builtin_amdgcn_ballot_w64(tie);
                if (tie) stays = ties + below(tied) < stay;
                ties += __popcll(tied);
            }
            const bool hole = there && !stays && j < left, mover = stays && j >= left;
            f(j, hole, mover, __builtin_amdgcn_ballot_w64(hole), __builtin_amdgcn_ballot_w64(mover));
        });
    }
};
// The recent weights where they go, zeros behind them, by one workgroup; late: the first 4 x 1024.
__device__ __forceinline__ void shift_weights(const KdaEvictArgs& a, const Plan& p, float* weights, int len, const float (&late)[4]) {
    const int end = len - a.recent, tid = threadIdx.x;
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

template <int R>
__global__ void __launch_bounds__(SCAN_THREADS) select_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int hist[BINS];
    __shared__ int sw[WAVES];
    __shared__ int flags[5];  // of `look`; of `pick`
    __shared__ char* at[2][PAIRS];
    __shared__ int few[2][FEW];  // the first pairs
    __shared__ int pages[ROW_PAGES];  // the first of the row's
    const int i = p.first + blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    const int row = a.src[i];
    const KdaEvictLayer y = a.layer[l];
    if (tid < 5) flags[tid] = 0;
    hist[tid] = hist[tid + SCAN_THREADS] = 0;
    const int len = length_of(a, row), end = len - a.recent;  // candidates [fixed, end)
    float* const weights = y.weights + (len < 0 ? 0 : row) * y.weights_row;
    const Keys<R> keys(weights, 0, len < 0 ? 0 : end);
    float late[4];  // the first recent ones, for the end
#pragma unroll
    for (int u = 0; u < 4; ++u) late[u] = weights[len < 0 ? 0 : min(end + u * SCAN_THREADS + tid, len - 1)];
    __syncthreads();
    if (len >= 0) look(a, p, i, row, len, flags, l == 0, pages);
    __syncthreads();
    const int fixed = flags[0];
    const bool cut = len >= 0 && !flags[1] && fixed <= p.left;
    if (l == 0 && tid == 0) lens_of(a)[i] = cut ? len : -1;
    if (!cut) {
        if (tid == 0) *pairs_of(a, i, l) = 0;
        return;
    }
    int total;
    Last last(p.left - fixed);
    if (last.stay > 0)
#pragma unroll
        for (int d = 0; d < 3; ++d) {
            keys.each(fixed, [&](int, uint32_t k, bool there) { last.count(hist, d, k, there); });
            last.pick(hist, d, flags + 2, sw);
        }
    // ---- holes and movers, in index order
    int32_t* const places = lists_of(a, p, blockIdx.x, l);
    int32_t* const tokens = places + p.most;
    int ties = 0;
    if (!last.all) {
        keys.each(fixed, [&](int, uint32_t k, bool there) { ties += __popcll(__builtin_amdgcn_ballot_w64(there && k == last.prefix)); });
        ties = before_wave(ties, sw, total);
    }
    int holes = 0, movers = 0;
    last.marks(keys, fixed, p.left, ties, [&](int, bool, bool, uint64_t h, uint64_t m) { holes += __popcll(h), movers += __popcll(m); });
    int pairs;
    holes = before_wave(holes, sw, pairs);
    movers = before_wave(movers, sw, total);  // (as many)
    const bool few_pairs = pairs <= FEW;
    last.marks(keys, fixed, p.left, ties, [&](int j, bool hole, bool mover, uint64_t h, uint64_t m) {
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
    shift_weights(a, p, weights, len, late);
}

// The same of more tokens, by a workgroup for 8192 of each (sequence, layer): what a row's pages say, the histograms of three digits, the
// counts of each part, the lists.
__global__ void __launch_bounds__(SCAN_THREADS) look_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int flags[2];
    const int i = p.first + blockIdx.x, l = blockIdx.y, tid = threadIdx.x;
    int32_t* const hist = hist_of(a, p, blockIdx.x, l);
#pragma unroll
    for (int k = 0; k < 3 * BINS; k += SCAN_THREADS) hist[k + tid] = 0;
    if (tid == 0) *pairs_of(a, i, l) = 0;
    if (l) return;
    if (tid < 2) flags[tid] = 0;
    const int row = a.src[i], len = length_of(a, row);
    __syncthreads();
    if (len >= 0) look(a, p, i, row, len, flags, true, nullptr);
    __syncthreads();
    if (tid) return;
    lens_of(a)[i] = len >= 0 && !flags[1] && flags[0] <= p.left ? len : -1;
    fixed_of(a, p)[i] = flags[0];
}

// PASS 0 to 2: the histogram of a digit.  3: the part's counts.  4: its lists.
template <int PASS>
__global__ void __launch_bounds__(SCAN_THREADS) part_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int hist[BINS];
    __shared__ int sw[WAVES];
    __shared__ int found[3], earlier[3];  // of `pick`; the parts before this one: tokens with the key, holes, movers
    const int i = p.first + blockIdx.y, l = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int len = lens_of(a)[i], from = blockIdx.x * PART, end = len - a.recent;
    if (len < 0 || from >= end) return;
    const KdaEvictLayer y = a.layer[l];
    const Keys<PART_KEYS> keys(y.weights + a.src[i] * y.weights_row, from, min(end, from + PART));
    const int fixed = fixed_of(a, p)[i];
    int32_t* const hists = hist_of(a, p, blockIdx.y, l);
    int x[3][2];
#pragma unroll
    for (int d = 0; d < 3 && d < PASS; ++d) x[d][0] = hists[d * BINS + tid], x[d][1] = hists[d * BINS + SCAN_THREADS + tid];
    Last last(p.left - fixed);
    if (last.stay > 0) {
#pragma unroll
        for (int d = 0; d < 3 && d < PASS; ++d) {
            hist[tid] = x[d][0], hist[tid + SCAN_THREADS] = x[d][1];
            last.pick(hist, d, found, sw);
        }
        if constexpr (PASS < 3) {
            if (PASS == 0) hist[tid] = hist[tid + SCAN_THREADS] = 0;
            __syncthreads();
            keys.each(fixed, [&](int, uint32_t k, bool there) { last.count(hist, PASS, k, there); });
            __syncthreads();
#pragma unroll
            for (int k = 0; k < BINS; k += SCAN_THREADS)
                if (hist[k + tid]) atomicAdd(hists + PASS * BINS + k + tid, hist[k + tid]);
        }
    }
    if constexpr (PASS < 3) return;
    // with the key below left and from it on; lighter ones below left, heavier ones from it on
    int32_t* const counts = counts_of(a, p, blockIdx.y, l);
    if constexpr (PASS == 3) {
        int n[4] = {}, total[4];
        keys.each(fixed, [&](int j, uint32_t k, bool there) {
            const bool low = j < p.left;
            n[0] += __popcll(__builtin_amdgcn_ballot_w64(there && k == last.prefix && low));
            n[1] += __popcll(__builtin_amdgcn_ballot_w64(there && k == last.prefix && !low));
            n[2] += __popcll(__builtin_amdgcn_ballot_w64(there && k < last.prefix && low));
            n[3] += __popcll(__builtin_amdgcn_ballot_w64(there && k > last.prefix && !low));
        });
#pragma unroll
        for (int k = 0; k < 4; ++k) before_wave(n[k], sw, total[k]);
        if (tid < 4) counts[4 * blockIdx.x + tid] = tid == 0 ? total[0] : tid == 1 ? total[1] : tid == 2 ? total[2] : total[3];
        return;
    }
    // ---- the parts before this one
    if (tid < 64) {
        int ties = 0, holes = 0, movers = 0;
        for (int c0 = 0; c0 < (int)blockIdx.x; c0 += 64) {
            int n[4] = {};
            if (c0 + lane < (int)blockIdx.x)
#pragma unroll
                for (int k = 0; k < 4; ++k) n[k] = counts[4 * (c0 + lane) + k];
            int sum = n[0] + n[1];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int v = __shfl_up(sum, d);
                if (lane >= d) sum += v;
            }
            const int left = last.stay - (ties + sum - n[0] - n[1]);  // of those with the key may stay from this part on
            const int low = max(0, min(left, n[0])), high = max(0, min(left - n[0], n[1]));
            holes += n[2] + n[0] - low, movers += n[3] + high;
            ties += __shfl(sum, 63);
        }
#pragma unroll
        for (int d = 1; d < 64; d *= 2) holes += __shfl_xor(holes, d), movers += __shfl_xor(movers, d);
        if (tid == 0) earlier[0] = ties, earlier[1] = holes, earlier[2] = movers;
    }
    int total, pairs, ties = 0, holes = 0, movers = 0;
    keys.each(fixed, [&](int, uint32_t k, bool there) { ties += __popcll(__builtin_amdgcn_ballot_w64(there && k == last.prefix)); });
    ties = before_wave(ties, sw, total) + earlier[0];
    last.marks(keys, fixed, p.left, ties, [&](int, bool, bool, uint64_t h, uint64_t m) { holes += __popcll(h), movers += __popcll(m); });
    holes = before_wave(holes, sw, pairs) + earlier[1];
    movers = before_wave(movers, sw, total) + earlier[2];
    int32_t* const places = lists_of(a, p, blockIdx.y, l);
    int32_t* const tokens = places + p.most;
    if (tid == 0 && from + PART >= end) *pairs_of(a, i, l) = earlier[1] + pairs;
    last.marks(keys, fixed, p.left, ties, [&](int j, bool hole, bool mover, uint64_t h, uint64_t m) {
        if (hole) places[holes + below(h)] = j;
        if (mover) tokens[movers + below(m)] = j;
        holes += __popcll(h), movers += __popcll(m);
    });
}

__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(KdaEvictArgs a, Plan p) {
    __shared__ char* at[2][PAIRS];
    const int i = p.first + blockIdx.y, l = blockIdx.z;
    const int pairs = *pairs_of(a, i, l);
    if (!p.parts && pairs <= FEW) return;
    const int32_t* lists = lists_of(a, p, blockIdx.y, l);
    const KdaEvictLayer y = a.layer[l];
    const int row = a.src[i], pieces = (int)(y.token_bytes / 16);
    float* const weights = y.weights + row * y.weights_row;
    for (int first = blockIdx.x * PAIRS; first < pairs; first += gridDim.x * PAIRS) {
        const int count = min(pairs - first, PAIRS);
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * PAIRS; k += MOVE_THREADS)
            if (k % PAIRS < count) at[k / PAIRS][k % PAIRS] = token_at(a, y, row, lists[(int64_t)(k / PAIRS) * p.most + first + k % PAIRS]);
        if (p.parts && (int)threadIdx.x < count) weights[lists[first + threadIdx.x]] = weights[lists[(int64_t)p.most + first + threadIdx.x]];
        __syncthreads();
        copy_tokens<MOVE_THREADS>(at, count, pieces);
    }
}

// A row's first pages stay, the rest of its tokens' pages go, entries past the tokens follow the first ones.  Of `count` rows from slot
// `first` on by one workgroup, up to 16 at a time.  (24 rows of 2200 tokens in 7
// layers, the launch with the recent rows: one after the other 18 us, so 9.)
__device__ __forceinline__ void books(const KdaEvictArgs& a, int first, int count) {
    int side = 1;  // rows at a time
    while (side < 16 && side < count) side *= 2;
    const int per = SCAN_THREADS / side, lane = threadIdx.x % per, kept = (a.keep + a.page_size - 1) / a.page_size;
    for (int k = 0; k < count; k += side) {
        const int i = first + min(k + (int)threadIdx.x / per, count - 1);
        const int len = k + (int)threadIdx.x / per < count ? lens_of(a)[i] : -1, row = len < 0 ? 0 : a.src[i];
        const int used = (len + a.page_size - 1) / a.page_size, by = len < 0 ? 0 : used - kept;
        int32_t* table = a.block_table + row * a.table_stride;
        for (int j = kept + lane; j < kept + by; j += per) atomicCAS(a.ref_counts + table[j], 1, FREED);  // (none is held twice)
        __syncthreads();
        for (int j0 = kept; j0 < a.table_width; j0 += per) {
            const int j = j0 + lane;
            const bool moves = by > 0 && j < a.table_width;
            const int32_t next = moves && j + by < a.table_width ? table[j + by] : -1;
            __syncthreads();
            if (moves) table[j] = next;
            __syncthreads();
        }
        if (lane == 0 && len >= 0) a.seq_lens[row] = a.keep;
    }
}

__global__ void __launch_bounds__(SCAN_THREADS) shift_kernel(KdaEvictArgs a, Plan p) {
    __shared__ int sw[WAVES];
    __shared__ char* at[2][PAIRS];
    const int i = blockIdx.y, l = blockIdx.z, tid = threadIdx.x;
    if ((int)blockIdx.x == p.strips) {  // the books
        if (l || (i && p.books == ALL)) return;
        if (p.books == ROWS) return books(a, i, 1);
        books(a, 0, a.n);
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
    if (p.parts) {  // the weights
        float* const weights = y.weights + row * y.weights_row;
        const int first = blockIdx.x * SCAN_THREADS + tid, step = p.strips * SCAN_THREADS;
        if (end >= a.keep) {  // no place is another one's token
            for (int k = first; k < a.recent; k += step) {
                weights[p.left + k] = weights[end + k];
                weights[end + k] = 0.f;
            }
            for (int j = a.keep + first; j < end; j += step) weights[j] = 0.f;
        } else if (blockIdx.x == 0) {
            float late[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) late[u] = weights[min(end + u * SCAN_THREADS + tid, len - 1)];
            shift_weights(a, p, weights, len, late);
        }
    }
    if (end >= a.keep) {
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
    KDA_CHECK_ARG(a->n <= 65535 || (int64_t)a->table_width * a->page_size <= a->keep, "evict_tokens: %d rows in one call (at most 65535)", a->n);
    return 0;
}

Plan plan_of(const KdaEvictArgs* a) {
    Plan p;
    const int64_t span = (int64_t)a->table_width * a->page_size;
    p.left = a->keep - a->recent;
    const int64_t goes = span - a->keep;  // no more tokens go from below `left` than go in all
    p.most = (int)(goes <= 0 ? 0 : goes < p.left ? goes : p.left);
    p.tail = (int)((a->recent + a->page_size - 1) / a->page_size + 1);
    // More candidates than a workgroup has registers for: by parts.  (One workgroup that read them anew for each digit: 124 us for sequences of
    // 131072 and 100001 tokens in 7 layers; the six launches of the parts 39.  For 256 times 4000 one launch takes 18 us and six would not.)
    const int64_t candidates = span - a->recent;
    p.parts = candidates <= 16 * SCAN_THREADS ? 0 : (int)((candidates + PART - 1) / PART);
    const int layers = a->num_layers > 0 ? a->num_layers : 1;
    const int64_t fit = LIST_BYTES / (8 * (int64_t)layers * (p.most > 0 ? p.most : 1)), at_once = AT_ONCE / layers;
    const int64_t rows = p.parts && at_once < fit ? at_once : fit;
    p.first = 0, p.rows = (int)(rows < 1 ? 1 : rows < a->n ? rows : a->n);
    return p;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int64_t kda355_evict_tokens_workspace_bytes(const KdaEvictArgs* a) {
    if (const int rc = check_evict(a)) return rc;
    const Plan p = plan_of(a);
    const int64_t run = (int64_t)p.rows * a->num_layers;
    const int64_t parts = p.parts ? a->n + run * (3 * BINS + 4 * (int64_t)p.parts) : 0;
    return 4 * (a->n * (1 + (int64_t)p.tail) + (int64_t)a->n * a->num_layers + run * 2 * p.most + parts);
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
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    Plan p = plan_of(a);
    const int64_t fill = 4096 / (a->n * a->num_layers) + 1;  // workgroups of a sequence and layer
    const auto some = [](int64_t x, int64_t y) { return (int)(x < y ? x : y); };
    const auto cdiv = [](int64_t x, int64_t y) { return (x + y - 1) / y; };
    for (; p.first < a->n; p.first += p.rows) {
        const int rows = some(p.rows, a->n - p.first);
        const dim3 threads(SCAN_THREADS);
        if (p.parts) {
            const dim3 grid(p.parts, rows, a->num_layers);
            launch_kernel(look_kernel, dim3(grid.y, grid.z), threads, s, *a, p);
            launch_kernel(part_kernel<0>, grid, threads, s, *a, p);
            launch_kernel(part_kernel<1>, grid, threads, s, *a, p);
            launch_kernel(part_kernel<2>, grid, threads, s, *a, p);
            launch_kernel(part_kernel<3>, grid, threads, s, *a, p);
            launch_kernel(part_kernel<4>, grid, threads, s, *a, p);
        } else
            launch_kernel(span - a->recent <= 4 * SCAN_THREADS ? select_kernel<4> : select_kernel<16>, dim3(rows, a->num_layers), threads, s, *a, p);
        if (p.most > (p.parts ? 0 : FEW))
            launch_kernel(move_kernel, dim3(some(cdiv(p.most, PAIRS), 4096 / (rows * a->num_layers) + 1), rows, a->num_layers), dim3(MOVE_THREADS), s, *a, p);
    }
    const bool last = !(a->flags & KDA355_EVICT_MORE);
    const int strips = (int)cdiv(pieces, STRIP), parts = some(cdiv(a->recent, PAIRS), fill / 4 + 1);
    p.strips = a->recent == 0 ? 0 : strips > parts ? strips : parts;
    if (p.parts) p.strips = p.strips > (p.parts + 3) / 4 ? p.strips : (p.parts + 3) / 4;  // (the weights are left to them)
    p.books = !last ? 0 : a->n <= BOOK_ROWS && (int64_t)a->n * a->table_width <= BOOK_ENTRIES && a->pages <= BOOK_PAGES ? ALL : ROWS;
    if (p.strips || p.books)
        launch_kernel(shift_kernel, dim3(p.strips + (p.books != 0), a->n, p.strips ? a->num_layers : 1), dim3(SCAN_THREADS), s, *a, p);
    if (p.books == ROWS) {
        KdaPagesArgs b = {};
        b.ref_counts = a->ref_counts, b.free_pages = a->free_pages, b.num_free = a->num_free, b.pages = a->pages;
        launch_kernel(free_push_kernel, dim3(1), dim3(SCAN_THREADS), s, b);
    }
    return launched("evict_tokens");
}
