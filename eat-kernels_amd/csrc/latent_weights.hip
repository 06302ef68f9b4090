// What an attention step over the paged latent cache gave every cached token (gfx950): weights[n, j] += sum_i e^(z_ij - lse_i) over the
// rows i = (token, head) of sequence n that see token j.
//
// Scores anew from the log-sums that the step left: the softmax weights are known only once its last key has been seen, and kept scores
// would be 4 bytes a row and token where a cache row is 400 or 1152 for all rows.  Keys stand still: a wave keeps 32 of them in
// registers as operand rows (16x16x32 instructions; from 4 bits widened as they come), the query rows pass through LDS in tiles of 16,
// and a lane adds up its row of every tile for its 4 + 4 keys.  One sum across the 16 lanes of a key at the end; no two workgroups
// write the same token, so the order of a sum depends on the sizes alone.  Two workgroups a CU, each with an equal run of units of 128
// keys through the sequences; up to 64 query rows stay in LDS from one unit of a sequence to the next, more come three tiles ahead.
//
// Bound: with many rows the products (matrix cores busy 40 %, LDS 21 % over the launch) and what does not run beside them.  16 sequences of
// 6000 to 9900 tokens, 8 x 96 rows: 127 us steady, 0.88 PFLOP/s; timed without bringing the query rows 102, with rows that stay in L1 115,
// without the exponentials 117, without either 92; some 15 go by before the first keys are there.  Eight waves a workgroup, which halves
// the rows' way from L2, and a barrier for two tiles: 123, but 62 against 48 with few rows; with a barrier a tile 136.  The loads of rows
// spread between the products: 134.  With few rows memory: 64 ragged sequences of 64 heads in 4 bits 48 us, 4.0 TB/s.  One sequence of 4097
// tokens, 12 heads: 7.6 us, lengths, keys and queries one after the other.
#include "latent.h"

namespace kda355 {
namespace {

constexpr int WAVES = 4, THREADS = WAVES * 64;
constexpr int KEYS = 32, UNIT = WAVES * KEYS;  // keys of a wave, of a workgroup
constexpr int RT = 16;                         // query rows of a tile
constexpr int STEPS = ROW / 32;                // matrix instructions of 16 keys and a tile
constexpr int Q_LAT = RT * LAT_BYTES, Q_LSE = Q_LAT + RT * PE_BYTES, Q_TILE = Q_LSE + 256, RING = 4;  // tiles in LDS
constexpr int Q_LOADS = RT / WAVES + 1;        // of a wave a tile
constexpr int AHEAD = 5;                       // operands read before they are needed

struct Plan {
    PageOf page, head;  // head: row / H
    int grid;
    bool dense;         // the rows of a sequence are one head stride apart throughout
};

__device__ __forceinline__ uint32_t units_of(int tokens) { return ((uint32_t)tokens + UNIT - 1) / UNIT; }
struct Run { uint32_t first, end; int n; uint32_t before; };
// This workgroup's units [first, end) of all, the sequence that holds the first one, and the units before that sequence.
__device__ __forceinline__ Run run_of(const KdaLatentWeightsArgs& a) {
    const int lane = threadIdx.x & 63;
    auto load = [&](int n) { return n < a.B ? units_of(tokens_of(a.seq_lens[n], a.table_width, a.page_size)) : 0u; };
    const uint32_t mine = load(lane);  // (loaded once where there are no more sequences)
    uint32_t all = mine;
    for (int n = lane + 64; n < a.B; n += 64) all += load(n);
    all = __builtin_amdgcn_readlane(scan_wave((int)all), 63);
    const uint32_t b = xcd_task(blockIdx.x, gridDim.x);  // neighbours read the same queries: on one XCD
    Run r = {(uint32_t)((uint64_t)b * all / gridDim.x), (uint32_t)((uint64_t)(b + 1) * all / gridDim.x), a.B, 0};
    for (int n0 = 0; n0 < a.B; n0 += 64) {
        const uint32_t t = n0 ? load(n0 + lane) : mine, s = (uint32_t)scan_wave((int)t);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(r.before + s > r.first);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            r.n = n0 + l;
            r.before += __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(t, l);
            break;
        }
        r.before += __builtin_amdgcn_readlane(s, 63);
    }
    return r;
}

// Latent row b of a tile stands at 1024 b, its piece p at place (p % 16) ^ turn(b) of each 16.  16-byte reads go 16 lanes at a time, lanes 0
// .. 3, 12 .. 15, 20 .. 23 and 24 .. 27 of 32 and the others: with these turns they touch all 16 places.
template <bool Q4>
__device__ __forceinline__ int turn(int b) { return (b & 3) << 2 | (Q4 ? b >> 2 & 3 : (b >> 3 & 1) << 1); }

template <typename T, bool Q4>
__global__ void __launch_bounds__(THREADS, 2) weights_kernel(KdaLatentWeightsArgs a, Plan p) {
    static_assert(2 * RING * Q_TILE <= 160 * 1024, "");
    __shared__ __align__(1024) unsigned char sm[RING * Q_TILE];
    const uint32_t lds = lds_offset(sm);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int c = lane & 15, quad = lane >> 4;
    const int rows = a.S * a.H, tiles = (rows + RT - 1) / RT;
    constexpr int CACHE_ROW = Q4 ? ROW4 : ROW_BYTES;
    const int64_t page_bytes = Q4 ? a.page_stride : a.page_stride * 2;
    // A key's operand of step i < 16 has of a lane quarter values 32 i + 8 quad .., from 4 bits, where 16 bytes are the 32 values of one scale,
    // 128 (i / 4) + 32 quad + 8 (i % 4) .. (the order of the contraction is free): piece 4 i + quad of a query row, or 16 (i / 4) + 4 quad +
    // i % 4.  Steps 16 and 17: pieces quad and 4 + quad of its positional part.
    const uint32_t at_latent = c * LAT_BYTES + (((Q4 ? quad << 2 : quad) ^ turn<Q4>(c)) << 4), at_pe = Q_LAT + c * PE_BYTES + ((quad ^ swz8(c)) << 4);
    const Run run = run_of(a);
    int n = run.n, held = -1;  // held: the sequence whose query rows are all in LDS
    uint32_t before = run.before;
    int tokens = 0;
    uint32_t units = 0;

    for (uint32_t u = run.first; u < run.end; ++u) {
        while (n < a.B) {  // (sequences without tokens have no units)
            tokens = __builtin_amdgcn_readfirstlane(tokens_of(a.seq_lens[n], a.table_width, a.page_size));
            units = units_of(tokens);
            if (u < before + units) break;
            before += units;
            ++n;
        }
        n = __builtin_amdgcn_readfirstlane(n);
        const int k0 = __builtin_amdgcn_readfirstlane((int)((u - before) * UNIT) + KEYS * w);

        // ---- query rows
        const char* const ql = static_cast<const char*>(a.q_latent) + n * (int64_t)a.S * a.ql_row * 2;
        const char* const qp = static_cast<const char*>(a.q_pe) + n * (int64_t)a.S * a.qp_row * 2;
        auto bring = [&](int tile) {
            const uint32_t to = lds + tile % RING * Q_TILE;
            const int first = tile * RT;
            uint64_t row[RT / WAVES];  // of the wave's latent rows
            int64_t pe;                // to the lane's row of positional parts
            if (p.dense) {
#pragma unroll
                for (int i = 0; i < RT / WAVES; ++i)
                    row[i] = (uint64_t)ql + (uint64_t)(uint32_t)min(first + w * (RT / WAVES) + i, rows - 1) * (uint64_t)(2 * a.ql_head);
                pe = min(first + 8 * (w & 1) + (lane >> 3), rows - 1) * (2 * a.qp_head);
            } else {
                auto at = [&](int r, int64_t stride, int64_t head) {
                    r = min(r, rows - 1);
                    const uint32_t s = p.head(r);
                    return 2 * (s * stride + (r - (int)s * a.H) * head);
                };
#pragma unroll
                for (int i = 0; i < RT / WAVES; ++i) row[i] = (uint64_t)ql + at(first + w * (RT / WAVES) + i, a.ql_row, a.ql_head);
                pe = at(first + 8 * (w & 1) + (lane >> 3), a.qp_row, a.qp_head);
            }
#pragma unroll
            for (int i = 0; i < RT / WAVES; ++i) {
                const int b = w * (RT / WAVES) + i;
                load_block_from(to + b * LAT_BYTES, row[i], ((lane & 48) | ((lane & 15) ^ turn<Q4>(b))) << 4);
            }
            if (w < 2)
                load_block<0>(to + Q_LAT + 8 * w * PE_BYTES, (uint64_t)qp + pe + (((lane & 7) ^ swz8(8 * w + (lane >> 3))) << 4));
            else  // the rows' log-sums, by both others: a compiler's load would be waited for with everything that is under way
                load_words(to + Q_LSE, (uint64_t)(a.lse + n * (int64_t)rows + min(first + c, rows - 1)));
        };
        // ---- keys
        u32x4 kf[2][STEPS];
        bool there[2];
        uint64_t from[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int key = k0 + 16 * y + c;
            const uint32_t pg = p.page((uint32_t)key);
            const int page = key < tokens ? a.block_table[n * a.table_stride + pg] : -1;
            there[y] = page >= 0 && page < a.pages;
            from[y] = (uint64_t)a.cache + page * page_bytes + (int64_t)((uint32_t)key - pg * (uint32_t)a.page_size) * CACHE_ROW;
            asm volatile("" : "+v"(from[y]));  // (a choice of two, not a branch)
            from[y] = there[y] ? from[y] : (uint64_t)zero_row;
        }
        u32x4 scales[2], codes[2][4];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const char* row = reinterpret_cast<const char*>(from[y]);
            if constexpr (Q4) {
                scales[y] = *reinterpret_cast<const u32x4*>(row + SCALES4);
#pragma unroll
                for (int j = 0; j < 4; ++j) codes[y][j] = *reinterpret_cast<const u32x4*>(row + 64 * j + 16 * quad);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) kf[y][i] = *reinterpret_cast<const u32x4*>(row + 64 * i + 16 * quad);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                kf[y][16 + i] = *reinterpret_cast<const u32x4*>(row + (Q4 ? PE4 : LAT_BYTES) + 64 * i + 16 * quad);
        }
        // what lane c < 8 adds to: key 16 (c / 4) + 4 quad + c % 4
        uint32_t mine = 0;  // of key 16 y + 4 quad + r: is it there
#pragma unroll
        for (int y = 0; y < 2; ++y) mine |= ((uint32_t)__builtin_amdgcn_ballot_w64(there[y]) >> 4 * quad & 15u) << 4 * y;
        float* const at = a.weights + n * a.weights_row + k0 + 16 * (c >> 2) + 4 * quad + (c & 3);
        const bool writes = c < 8 && (mine >> c & 1);
        const float old = writes ? *at : 0.f;
        // (query rows after the keys' loads: what waits for these does not wait for those)
        const bool stay = tiles <= RING;
        if (!stay || held != n) {
            for (int t = 0; t < min(tiles, stay ? RING : RING - 1); ++t) bring(t);
            held = stay ? n : -1;
        }
        if constexpr (Q4) {
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float scale = __uint_as_float((scales[y][j] >> 8 * quad & 255u) << 23);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[y][4 * j + e] = T::from4(codes[y][j][e], scale);
                }
        }
        // every row sees all 32 keys: no masks
        const bool plain = k0 + KEYS <= tokens - (a.S - 1) && __builtin_amdgcn_ballot_w64(mine != 255u) == 0;
        if (stay) {
            wait_loads<0>();
            __syncthreads();
        }

        float sum[2][4] = {};
        for (int tile = 0; tile < tiles; ++tile) {
            if (!stay) {
                if (tile + RING - 2 < tiles) wait_loads<(RING - 2) * Q_LOADS>(); else wait_loads<0>();
                lds_barrier();  // the tile is whole; all have read the one before it
            }
            if (!stay && tile + RING - 1 < tiles) bring(tile + RING - 1);
            const uint32_t from = lds + tile % RING * Q_TILE;
            const float lse = *reinterpret_cast<const float*>(sm + tile % RING * Q_TILE + Q_LSE + c * 4);
            f32x4 z[2][2] = {};
            auto query = [&](int i) {
                if (i >= 16) return lds_read16((from + at_pe) ^ (i - 16) << 6);
                return lds_read16(((from + at_latent) ^ (i & 3) << (Q4 ? 4 : 6)) + (i >> 2) * 256);
            };
            u32x4 q[AHEAD + 1];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) q[i] = query(i);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                if (i + AHEAD < STEPS) q[(i + AHEAD) % (AHEAD + 1)] = query(i + AHEAD);
#pragma unroll
                for (int y = 0; y < 2; ++y) z[y][i & 1] = T::mfma16(kf[y][i], q[i % (AHEAD + 1)], z[y][i & 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
            const int row = tile * RT + c;
            const bool alive = row < rows && lse != -INFINITY;
            auto add = [&](bool all) {
                const int left = all ? 0 : tokens - (a.S - 1 - (int)p.head(row)) - k0 - 4 * quad;  // keys that the row sees, from the lane's first on
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const f32x4 s = z[y][0] + z[y][1];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        // the difference first: it is small where the weight counts, and so is its rounding
                        const float e = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale, -lse) * 1.44269504088896f);
                        if (alive && (all || ((mine >> (4 * y + r) & 1) && 16 * y + r < left))) sum[y][r] += e;
                    }
                }
            };
            if (plain) add(true); else add(false);
        }
        // ---- the 16 rows of a key's lanes
        float out = 0.f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = sum16(sum[y][r]);
                if (c == 4 * y + r) out = s;
            }
        if (writes) *at = old + out;
        if (!stay || u + 1 == before + units) __syncthreads();  // the query rows are read
    }
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int kda355_latent_weights_launch(const KdaLatentWeightsArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "latent_weights: null args");
    KDA_CHECK_ARG(a->B >= 0 && a->S >= 1 && a->H >= 1 && a->page_size >= 1 && a->table_width >= 0 && a->num_cus >= 0 && a->num_cus <= 65536,
                  "latent_weights: B=%d S=%d H=%d page_size=%d table_width=%d num_cus=%d", a->B, a->S, a->H, a->page_size, a->table_width,
                  a->num_cus);
    KDA_CHECK_ARG((int64_t)a->S * a->H < (1ll << 29) && (int64_t)a->B * a->S * a->H < (1ll << 29) && a->B < (1 << 22),
                  "latent_weights: B * S * H is too large");
    const int64_t span = (int64_t)a->table_width * a->page_size;
    KDA_CHECK_ARG(span < (1ll << 31) - 256, "latent_weights: a table spans 2^31 tokens or more");
    KDA_CHECK_ARG(a->B * (span / 128 + 1) < (1ll << 31), "latent_weights: the tables span 2^38 tokens or more");
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "latent_weights: dtype %d", a->dtype);
    KDA_CHECK_ARG(a->cache_bits == 16 || a->cache_bits == 4, "latent_weights: cache_bits %d", a->cache_bits);
    KDA_CHECK_ARG(a->flags == 0, "latent_weights: unknown flags 0x%x", a->flags);
    if (a->B == 0) return 0;
    KDA_CHECK_ARG(a->q_latent && a->q_pe && a->cache && a->block_table && a->seq_lens && a->lse && a->weights && a->table_width >= 1,
                  "latent_weights: a required pointer is null");
    KDA_CHECK_ARG(a->pages >= 1 && a->table_stride >= a->table_width, "latent_weights: pages=%lld table_stride=%lld", (long long)a->pages,
                  (long long)a->table_stride);
    KDA_CHECK_ARG(a->weights_row >= span, "latent_weights: rows of weights are shorter than the table's tokens");
    KDA_CHECK_ARG(rows16(a->q_latent, a->ql_row, a->ql_head) && rows16(a->q_pe, a->qp_row, a->qp_head),
                  "latent_weights: q rows must be 16-byte aligned");
    const bool q4 = a->cache_bits == 4;
    KDA_CHECK_ARG(aligned(a->cache, 16) && a->page_stride % (q4 ? 16 : 8) == 0 && a->page_stride >= (int64_t)a->page_size * (q4 ? ROW4 : ROW),
                  "latent_weights: cache pages must be dense and 16-byte aligned");
    KDA_CHECK_ARG(a->scale > 0.f, "latent_weights: scale must be positive");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    Plan p;
    p.page = PageOf::by(a->page_size);
    p.head = PageOf::by(a->H);
    p.dense = a->S == 1 || (a->ql_row == a->H * a->ql_head && a->qp_row == a->H * a->qp_head);
    const int64_t most = a->B * ((span + UNIT - 1) / UNIT), fill = 2 * (a->num_cus ? a->num_cus : 256);
    p.grid = (int)(most < fill ? most : fill);
    auto launch = [&](auto type) {
        typedef decltype(type) T;
        launch_kernel(q4 ? weights_kernel<T, true> : weights_kernel<T, false>, dim3(p.grid), dim3(THREADS), s, *a, p);
    };
    if (a->dtype == KDA355_DTYPE_BF16) launch(Bf16{}); else launch(Fp16{});
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("latent_weights: launch failed: %s", hipGetErrorString(e));
        return KDA355_ELAUNCH;
    }
    return 0;
}
