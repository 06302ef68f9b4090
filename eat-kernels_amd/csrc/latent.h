// What the kernels over the paged latent cache share (gfx950): its rows, pages and lengths, and the host's checks of alignment.
#pragma once
#include "attend.h"

namespace kda355 {
namespace {

constexpr int LAT = KDA355_LATENT_DIM, ROW = KDA355_LATENT_ROW, PE = KDA355_LATENT_PE;
constexpr int ROW_BYTES = ROW * 2, LAT_BYTES = LAT * 2, PE_BYTES = PE * 2;
// a row in 4 bits: codes, scales of GROUP values each, the positional part
constexpr int ROW4 = KDA355_LATENT_ROW_4BIT, GROUP = KDA355_LATENT_GROUP, SCALES4 = LAT / 2, PE4 = SCALES4 + LAT / GROUP;
static_assert(PE4 + PE_BYTES == ROW4, "");

struct PageOf {
    uint32_t mul, shift;  // x / page_size = x * mul >> shift, x < 2^31
    static PageOf by(int page_size) {
        int bits = 0;  // 2^bits >= page_size: mul page_size = 2^(31 + bits) + e, e < 2^bits, so the quotient is exact
        while ((1ll << bits) < page_size) ++bits;
        return {(uint32_t)(((1ull << (31 + bits)) + page_size - 1) / page_size), (uint32_t)(31 + bits)};
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t tok) const { return (uint32_t)((uint64_t)tok * mul >> shift); }
};
__device__ const uint4 zero_row[ROW_BYTES / 16] = {};  // what a token that is not there reads

__device__ __forceinline__ int tokens_of(int len, int width, int page_size) { return min(max(len, 0), width * page_size); }

__device__ __forceinline__ uint64_t of_lane(uint64_t x, int l) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute(4 * l, (int)(uint32_t)(x >> 32)) << 32 |
           (uint32_t)__builtin_amdgcn_ds_bpermute(4 * l, (int)(uint32_t)x);
}

inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// rows of 16-byte pieces: aligned base, strides in multiples of 8 elements
inline bool rows16(const void* p, int64_t s0, int64_t s1 = 0) { return aligned(p, 16) && s0 % 8 == 0 && s1 % 8 == 0; }

}  // namespace
}  // namespace kda355
