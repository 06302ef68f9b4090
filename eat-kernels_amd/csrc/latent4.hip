// Token rows of the latent cache in 4 bits: into pages and back (gfx950).  Both move bytes: bound by HBM (65769 rows read and widened
// 19 us, 5.3 TB/s, of which the caches take a part; 6614 written 5.6), small calls by a launch (3.5 and 4.6).
//
// A row's 16-bit form is 72 pieces of 16 bytes, a lane each: four lanes hold the 32 values of a scale, find the largest among
// them through DPP and write a dword of codes each.  The scale is a power of two, so that scaling is exact and the conversion is one
// rounding.  Its exponent is the largest value's, less 2, so that this value is in [4, 8) steps; from 7 on, which would be cut to 6 by more
// than half the step of 2, the next exponent takes it.
#include "latent.h"

namespace kda355 {
namespace {

constexpr int ROW_Q = ROW / 8, LAT_Q = LAT / 8;  // 16-byte pieces of a row in 16 bits, of its latent part
constexpr int TOK_THREADS = 192, TOKENS = 8, PIECES = TOKENS * ROW_Q / TOK_THREADS;  // 3 pieces a thread
static_assert(PIECES * TOK_THREADS == TOKENS * ROW_Q && ROW_Q % 4 == 0 && TOK_THREADS % 4 == 0, "");

template <typename T>
struct Exponents;  // of the scales, so that every value is a finite number of the type, and for bf16 no subnormal one
template <>
struct Exponents<Bf16> { static constexpr int LEAST = -125, MOST = 125; };
template <>
struct Exponents<Fp16> { static constexpr int LEAST = -23, MOST = 13; };

// Of four lanes with the 32 values of a group: eight codes each, the scale's byte.
template <typename T>
__device__ __forceinline__ uint32_t round4(u32x4 x, uint32_t& byte) {
    float v[8];
    float a = 0.f;
    bool odd = false;  // an infinite value or a NaN: fmaxf would lose the latter
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = T::up((uint16_t)(x[i / 2] >> (i % 2 * 16)));
        a = fmaxf(a, fabsf(v[i]));
        odd |= !(fabsf(v[i]) < INFINITY);
    }
    if (odd) a = INFINITY;
    a = fmaxf(a, dpp<0xB1>(a));  // quad_perm [1,0,3,2]
    a = fmaxf(a, dpp<0x4E>(a));  // quad_perm [2,3,0,1]
    const uint32_t bits = __float_as_uint(a);
    int e = (int)(bits >> 23) - 127 - 2 + ((bits & 0x7fffffu) > 0x600000u);  // 7 x 2^e = 1.75 x 2^(e + 2)
    e = min(max(e, Exponents<T>::LEAST), Exponents<T>::MOST);
    const bool none = !(a < INFINITY);
    byte = none ? 255u : (uint32_t)(e + 127);
    const float scale = __uint_as_float((uint32_t)(e + 127) << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
    return none ? 0u : c;
}

template <typename T>
__global__ void __launch_bounds__(TOK_THREADS) append4_kernel(KdaLatentTokensArgs a) {
    __shared__ char* to[TOKENS];
    const int64_t first = (int64_t)blockIdx.x * TOKENS;
    if (threadIdx.x < TOKENS) {
        const int64_t t = first + threadIdx.x, slot = t < a.T ? a.slots[t] : -1;
        char* row = nullptr;
        if (slot >= 0 && slot < a.pages * a.page_size) {
            const int64_t page = slot / a.page_size;
            row = static_cast<char*>(a.cache) + page * a.page_stride + (slot - page * a.page_size) * ROW4;
        }
        to[threadIdx.x] = row;
    }
    __syncthreads();
    u32x4 x[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        x[i] = u32x4{0, 0, 0, 0};
        if (!to[t]) continue;
        const uint16_t* src = c < LAT_Q ? static_cast<const uint16_t*>(a.latent) + (first + t) * a.latent_row + c * 8
                                        : static_cast<const uint16_t*>(a.k_pe) + (first + t) * a.pe_row + (c - LAT_Q) * 8;
        x[i] = *reinterpret_cast<const u32x4*>(src);
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        uint32_t byte;
        const uint32_t codes = round4<T>(x[i], byte);  // (all lanes: the four of a group exchange)
        if (!to[t]) continue;
        if (c < LAT_Q) {
            *reinterpret_cast<uint32_t*>(to[t] + c * 4) = codes;
            if (c % 4 == 0) *reinterpret_cast<uint8_t*>(to[t] + SCALES4 + c / 4) = (uint8_t)byte;
        } else {
            *reinterpret_cast<u32x4*>(to[t] + PE4 + (c - LAT_Q) * 16) = x[i];
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(TOK_THREADS) gather4_kernel(KdaLatentTokensArgs a) {
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
                        row = static_cast<const char*>(a.cache) + page * a.page_stride + (j - p * a.page_size) * ROW4;
                }
            }
        }
        from[threadIdx.x] = row;
        to[threadIdx.x] = out;
    }
    __syncthreads();
    u32x4 x[PIECES];
    uint32_t scale[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        const char* row = from[t];
        x[i] = u32x4{0, 0, 0, 0};
        scale[i] = 0;
        if (row && c < LAT_Q) {
            x[i][0] = *reinterpret_cast<const uint32_t*>(row + c * 4);
            scale[i] = *reinterpret_cast<const uint8_t*>(row + SCALES4 + c / 4);
        } else if (row) {
            x[i] = *reinterpret_cast<const u32x4*>(row + PE4 + (c - LAT_Q) * 16);
        }
    }
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int p = i * TOK_THREADS + threadIdx.x, t = p / ROW_Q, c = p - t * ROW_Q;
        const u32x4 y = c < LAT_Q ? T::from4(x[i][0], __uint_as_float(scale[i] << 23)) : x[i];
        if (to[t]) __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(to[t] + c * 16));
    }
}

int check_tokens(const KdaLatentTokensArgs* a, const char* what) {
    KDA_CHECK_ARG(a != nullptr, "%s: null args", what);
    KDA_CHECK_ARG(a->T >= 0 && a->pages >= 1 && a->page_size >= 1, "%s: T=%lld pages=%lld page_size=%d", what,
                  (long long)a->T, (long long)a->pages, a->page_size);
    KDA_CHECK_ARG(a->T < (1ll << 25), "%s: %lld token rows in one call (less than 2^25)", what, (long long)a->T);
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "%s: dtype %d", what, a->dtype);
    KDA_CHECK_ARG(a->cache, "%s: a required pointer is null", what);
    KDA_CHECK_ARG(aligned(a->cache, 16) && a->page_stride % 16 == 0 && a->page_stride >= (int64_t)a->page_size * ROW4,
                  "%s: cache pages must be dense and 16-byte aligned", what);
    return 0;
}

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return KDA355_ELAUNCH;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int kda355_latent4_append_launch(const KdaLatentTokensArgs* a, kda355_stream_t stream) {
    if (const int rc = check_tokens(a, "latent4_append")) return rc;
    if (a->T == 0) return 0;
    KDA_CHECK_ARG(a->latent && a->k_pe && a->slots, "latent4_append: a required pointer is null");
    KDA_CHECK_ARG(rows16(a->latent, a->latent_row) && rows16(a->k_pe, a->pe_row),
                  "latent4_append: latent and k_pe rows must be 16-byte aligned");
    const dim3 grid((uint32_t)((a->T + TOKENS - 1) / TOKENS));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    launch_kernel(a->dtype == KDA355_DTYPE_BF16 ? append4_kernel<Bf16> : append4_kernel<Fp16>, grid, dim3(TOK_THREADS), s, *a);
    return launched("latent4_append");
}

extern "C" int kda355_latent4_gather_launch(const KdaLatentTokensArgs* a, kda355_stream_t stream) {
    if (const int rc = check_tokens(a, "latent4_gather")) return rc;
    if (a->T == 0 || a->N == 0) return 0;
    KDA_CHECK_ARG(a->N > 0 && a->table_width >= 1 && a->table_stride >= a->table_width, "latent4_gather: N=%d table_width=%d",
                  a->N, a->table_width);
    KDA_CHECK_ARG(a->block_table && a->cu && a->out, "latent4_gather: a required pointer is null");
    KDA_CHECK_ARG(rows16(a->out, a->out_row), "latent4_gather: out rows must be 16-byte aligned");
    const dim3 grid((uint32_t)((a->T + TOKENS - 1) / TOKENS));
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    launch_kernel(a->dtype == KDA355_DTYPE_BF16 ? gather4_kernel<Bf16> : gather4_kernel<Fp16>, grid, dim3(TOK_THREADS), s, *a);
    return launched("latent4_gather");
}
