// What an attention step over the paged latent cache gave every cached token (gfx950): weights[n, j] += sum_i e^(z_ij - lse_i) over the
// rows i = (token, head) of sequence n that see token j.
//
// Scores anew from the log-sums that the step left: the softmax weights are known only once its last key has been seen, and kept scores
// would be 4 bytes a row and token where a cache row is 400 or 1152 for all rows.  Keys stand still: a wave keeps 32 of them in
// registers as operand rows (16x16x32 instructions; from 4 bits widened as they come), the query rows pass through LDS in tiles of 16,
// and a lane adds up its row of every tile for its 4 + 4 keys.  One sum across the 16 lanes of a key at the end; no two workgroups
// write the same token, so the order of a sum depends on the sizes alone.
#include "latent.h"

namespace kda355 {
namespace {

constexpr int WAVES = 4, THREADS = WAVES * 64;
constexpr int KEYS = 32, UNIT = WAVES * KEYS;  // keys of a wave, of a workgroup
constexpr int RT = 16;                         // query rows of a tile
constexpr int STEPS = ROW / 32;                // matrix instructions of 16 keys and a tile
constexpr int Q_LAT = RT * LAT_BYTES, Q_TILE = Q_LAT + RT * PE_BYTES;

struct Plan {
    PageOf page;
    int grid;
};

__device__ __forceinline__ uint32_t units_of(int tokens) { return ((uint32_t)tokens + UNIT - 1) / UNIT; }
struct At { int n; uint32_t before; };
// the sequence that holds unit u of all (n = B: none), and the units before it
__device__ __forceinline__ At sequence_of(const KdaLatentWeightsArgs& a, uint32_t u) {
    const int lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (int n0 = 0; n0 < a.B; n0 += 64) {
        const int n = n0 + lane;
        const uint32_t t = n < a.B ? units_of(tokens_of(a.seq_lens[n], a.table_width, a.page_size)) : 0u;
        const uint32_t s = (uint32_t)scan_wave((int)t);
        const uint64_t hit = __builtin_amdgcn_ballot_w64(before + s > u);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            return {n0 + l, before + __builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(t, l)};
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return {a.B, before};
}

// A key's operand of step i: 8 values of a lane quarter.  In 16 bits values 32 i + 8 quad ..; from 4 bits, where 16 bytes are the 32 values of
// one scale, step 4 j + e has values 128 j + 32 quad + 8 e ... (the order of the contraction is free).  Returns the 16-byte piece of a query row.
template <bool Q4>
__device__ __forceinline__ int piece_of(int i, int quad) {
    if (i >= 16) return 4 * (i - 16) + quad;  // of the positional part
    return Q4 ? 16 * (i >> 2) + 4 * quad + (i & 3) : 4 * i + quad;
}

template <typename T, bool Q4>
__global__ void __launch_bounds__(THREADS, 2) weights_kernel(KdaLatentWeightsArgs a, Plan p) {
    __shared__ __align__(1024) unsigned char sm[2 * Q_TILE];
    const uint32_t lds = lds_offset(sm);
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int c = lane & 15, quad = lane >> 4;
    const int rows = a.S * a.H, tiles = (rows + RT - 1) / RT;
    constexpr int CACHE_ROW = Q4 ? ROW4 : ROW_BYTES;
    const int64_t page_bytes = Q4 ? a.page_stride : a.page_stride * 2;

    for (uint32_t u = blockIdx.x;; u += gridDim.x) {
        const At at = sequence_of(a, u);
        if (at.n >= a.B) return;
        const int n = __builtin_amdgcn_readfirstlane(at.n);
        const int tokens = __builtin_amdgcn_readfirstlane(tokens_of(a.seq_lens[n], a.table_width, a.page_size));
        const int k0 = __builtin_amdgcn_readfirstlane((int)((u - at.before) * UNIT) + KEYS * w);

        // ---- query rows: latent row b of a tile at 1024 b, its piece p at place (p % 16) ^ swz16(b) of each 16, positional parts as rows of 8
        auto bring = [&](int tile) {
            const uint32_t to = lds + (tile & 1) * Q_TILE;
#pragma unroll
            for (int i = 0; i < RT / WAVES; ++i) {
                const int b = w * (RT / WAVES) + i, r = min(tile * RT + b, rows - 1), s = r / a.H, h = r - s * a.H;
                const uint16_t* row = static_cast<const uint16_t*>(a.q_latent) + (n * (int64_t)a.S + s) * a.ql_row + h * a.ql_head;
                load_block<0>(to + b * LAT_BYTES, (uint64_t)row + (((lane & 48) | ((lane & 15) ^ swz16(b))) << 4));
            }
            if (w < 2) {
                const int b = 8 * w + (lane >> 3), r = min(tile * RT + b, rows - 1), s = r / a.H, h = r - s * a.H;
                const uint16_t* row = static_cast<const uint16_t*>(a.q_pe) + (n * (int64_t)a.S + s) * a.qp_row + h * a.qp_head;
                load_block<0>(to + Q_LAT + 8 * w * PE_BYTES, (uint64_t)row + (((lane & 7) ^ swz8(b)) << 4));
            }
        };
        auto lse_of = [&](int tile) {  // of the lane's row; -inf: it gives nothing
            const int r = tile * RT + c;
            return r < rows ? a.lse[n * (int64_t)rows + r] : -INFINITY;
        };
        bring(0);
        float lse = lse_of(0);

        // ---- keys
        u32x4 kf[2][STEPS];
        bool there[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int key = k0 + 16 * y + c;
            const uint32_t pg = p.page((uint32_t)key);
            const int page = key < tokens ? a.block_table[n * a.table_stride + pg] : -1;
            there[y] = page >= 0 && page < a.pages;
            uint64_t from = (uint64_t)a.cache + page * page_bytes + (int64_t)((uint32_t)key - pg * (uint32_t)a.page_size) * CACHE_ROW;
            asm volatile("" : "+v"(from));  // (a choice of two, not a branch)
            const char* row = reinterpret_cast<const char*>(there[y] ? from : (uint64_t)zero_row);
            if constexpr (Q4) {
                const u32x4 scales = *reinterpret_cast<const u32x4*>(row + SCALES4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x4 codes = *reinterpret_cast<const u32x4*>(row + 64 * j + 16 * quad);
                    const float scale = __uint_as_float((scales[j] >> 8 * quad & 255u) << 23);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kf[y][4 * j + e] = T::from4(codes[e], scale);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) kf[y][i] = *reinterpret_cast<const u32x4*>(row + 64 * i + 16 * quad);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                kf[y][16 + i] = *reinterpret_cast<const u32x4*>(row + (Q4 ? PE4 : LAT_BYTES) + 64 * i + 16 * quad);
        }
        // of key 16 y + 4 quad + r: is it there
        uint32_t mine = 0;
#pragma unroll
        for (int y = 0; y < 2; ++y) mine |= ((uint32_t)__builtin_amdgcn_ballot_w64(there[y]) >> 4 * quad & 15u) << 4 * y;
        wait_loads<0>();
        __syncthreads();

        float sum[2][4] = {};
        for (int tile = 0; tile < tiles; ++tile) {
            const uint32_t from = lds + (tile & 1) * Q_TILE;
            float next = -INFINITY;
            if (tile + 1 < tiles) {
                bring(tile + 1);
                next = lse_of(tile + 1);
            }
            f32x4 z[2][2] = {};
            auto query = [&](int i) {
                const int piece = piece_of<Q4>(i, quad);
                if (i >= 16) return lds_read16(from + Q_LAT + c * PE_BYTES + ((piece ^ swz8(c)) << 4));
                return lds_read16(from + c * LAT_BYTES + (piece >> 4) * 256 + (((piece & 15) ^ swz16(c)) << 4));
            };
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const u32x4 q = query(i);
#pragma unroll
                for (int y = 0; y < 2; ++y) z[y][i & 1] = T::mfma16(kf[y][i], q, z[y][i & 1]);
            }
            const int row = tile * RT + c, left = tokens - (a.S - 1 - row / a.H) - k0 - 4 * quad;  // keys that the row sees, from the lane's first on
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const f32x4 s = z[y][0] + z[y][1];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // the difference first: it is small where the weight counts, and so is its rounding
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale, -lse) * 1.44269504088896f);
                    if ((mine >> (4 * y + r) & 1) && 16 * y + r < left && lse != -INFINITY) sum[y][r] += e;
                }
            }
            lse = next;
            wait_loads<0>();
            __syncthreads();
        }
        // ---- the 16 rows of a key's lanes; lane c < 8 writes key 16 (c / 4) + 4 quad + c % 4
        float out = 0.f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = sum16(sum[y][r]);
                if (c == 4 * y + r) out = s;
            }
        if (c < 8 && (mine >> c & 1)) {
            float* x = a.weights + n * a.weights_row + k0 + 16 * (c >> 2) + 4 * quad + (c & 3);
            *x += out;
        }
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
    KDA_CHECK_ARG(span < (1ll << 31) - UNIT, "latent_weights: a table spans 2^31 tokens or more");
    KDA_CHECK_ARG(a->B * (span / UNIT + 1) < (1ll << 31), "latent_weights: the tables span 2^38 tokens or more");
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
