// What the page bookkeeping kernels share (gfx950): scans of one workgroup, and pages that were given up put on the stack.
#pragma once
#include "common.h"

namespace kda355 {
namespace {

constexpr int SCAN_THREADS = 1024;
constexpr int FREED = INT32_MIN;                  // count of a page freed in this call, until the stack has it

// ------------------------------------------------------------------------------------------------ scans
// exclusive prefix sum over the workgroup's threads; total in every thread
__device__ __forceinline__ int block_scan(int x, int* sw, int& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int s = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(s, d);
        if (lane >= d) s += y;
    }
    __syncthreads();  // sw free again
    if (lane == 63) sw[w] = s;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < SCAN_THREADS / 64; ++i) {
        const int v = sw[i];
        if (i < w) before += v;
        total += v;
    }
    return before + s - x;
}

// words that another thread of the workgroup wrote in this launch: past the vector L1
__device__ __forceinline__ int load_fresh(const int32_t* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ------------------------------------------------------------------------------------------------ stack
// The pages marked FREED, the highest first, by one workgroup.  FRESH: it marked them itself.
template <bool FRESH>
__device__ __forceinline__ void push_freed(int32_t* ref_counts, int32_t* free_pages, int32_t* num_free, int pages, int* sw) {
    int top = num_free[0];
    top = top < 0 ? 0 : top > pages ? pages : top;
    for (int hi = pages; hi > 0; hi -= 4 * SCAN_THREADS) {  // four pages a thread
        int mine[4], count = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int p = hi - 1 - 4 * (int)threadIdx.x - k;
            mine[k] = p >= 0 && (FRESH ? load_fresh(ref_counts + p) : ref_counts[p]) == FREED;
            count += mine[k];
        }
        int total;
        int at = top + block_scan(count, sw, total);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (mine[k]) {
                const int p = hi - 1 - 4 * (int)threadIdx.x - k;
                ref_counts[p] = 0;
                if (at < pages) free_pages[at] = p;
                ++at;
            }
        top += total;
    }
    if (threadIdx.x == 0) num_free[0] = top < pages ? top : pages;
}

__global__ void __launch_bounds__(SCAN_THREADS) free_push_kernel(KdaPagesArgs a) {
    __shared__ int sw[SCAN_THREADS / 64];
    push_freed<false>(a.ref_counts, a.free_pages, a.num_free, a.pages, sw);
}

// ------------------------------------------------------------------------------------------------ host
inline bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return KDA355_ELAUNCH;
}

}  // namespace
}  // namespace kda355
