// Latent attention, absorbed form over a paged cache (gfx950).
//
// One workgroup of 4 wave64 per (query row, head).  Each wave walks every fourth key with the row's dot product spread over
// its lanes and an online softmax (running maximum m, sum l and accumulator in fp32); the waves' parts are joined in LDS:
// o = sum_w e^(m_w - m) acc_w / sum_w e^(m_w - m) l_w.
#include "common.h"

namespace kda355 {
namespace {

constexpr int LAT = KDA355_LATENT_DIM, ROW = KDA355_LATENT_ROW;
constexpr int WAVES = 4;

template <typename T>
__device__ __forceinline__ float up(const void* base, int64_t i) { return (float)reinterpret_cast<const T*>(base)[i]; }

__device__ __forceinline__ float sum64(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

template <int NV>
struct Acc {
    float m = -INFINITY, l = 0.f, a[NV] = {};
    __device__ __forceinline__ void add(float z, const float (&v)[NV]) {
        const float mn = fmaxf(m, z);
        const float f = m == -INFINITY ? 0.f : __expf(m - mn);
        const float p = z == -INFINITY ? 0.f : __expf(z - mn);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < NV; ++i) a[i] = a[i] * f + p * v[i];
        m = mn;
    }
};

// joins the waves' parts; out elements lane + 64 i
template <typename T, int NV>
__device__ __forceinline__ void finish(Acc<NV>& c, void* out, int64_t at, float* lse) {
    __shared__ float sm[WAVES], sl[WAVES], sa[WAVES][NV * 64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < NV; ++i) sa[w][lane + 64 * i] = c.a[i];
    if (lane == 0) {
        sm[w] = c.m;
        sl[w] = c.l;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < WAVES; ++j) m = fmaxf(m, sm[j]);
    for (int j = 0; j < WAVES; ++j) l += sm[j] == -INFINITY ? 0.f : sl[j] * __expf(sm[j] - m);
    for (int e = threadIdx.x; e < NV * 64; e += WAVES * 64) {
        float o = 0.f;
        for (int j = 0; j < WAVES; ++j)
            if (sm[j] != -INFINITY) o += sa[j][e] * __expf(sm[j] - m);
        reinterpret_cast<T*>(out)[at + e] = (T)(l > 0.f ? o / l : 0.f);
    }
    if (lse && threadIdx.x == 0) *lse = l > 0.f ? m + __logf(l) : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(256) decode_kernel(KdaLatentDecodeArgs a) {
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int n = (int)(t / a.S), s = (int)(t - (int64_t)n * a.S);
    float q[9];
    for (int i = 0; i < 8; ++i) q[i] = up<T>(a.q_latent, t * a.ql_row + h * a.ql_head + lane + 64 * i) * a.scale;
    q[8] = up<T>(a.q_pe, t * a.qp_row + h * a.qp_head + lane) * a.scale;
    Acc<8> c;
    auto walk = [&](const int32_t* table, int width, int64_t len, int64_t hidden) {
        len = min(max(len, (int64_t)0), (int64_t)width * a.page_size) - hidden;
        for (int64_t j = w; j < len; j += WAVES) {
            const int64_t page = table[j / a.page_size];
            if (page < 0 || page >= a.pages) continue;
            const int64_t b = page * a.page_stride + (j % a.page_size) * ROW + lane;
            float v[8], z = q[8] * up<T>(a.cache, b + LAT);
            for (int i = 0; i < 8; ++i) {
                v[i] = up<T>(a.cache, b + 64 * i);
                z += q[i] * v[i];
            }
            c.add(sum64(z), v);
        }
    };
    if (a.prefix_table) walk(a.prefix_table, a.prefix_width, a.prefix_len[0], 0);
    walk(a.block_table + n * a.table_stride, a.table_width, a.seq_lens[n], a.S - 1 - s);
    finish<T>(c, a.out, t * a.out_row + h * a.out_head, a.lse ? a.lse + t * a.H + h : nullptr);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// rows of 16-byte pieces: aligned base, strides in multiples of 8 elements
bool rows16(const void* p, int64_t s0, int64_t s1 = 0) { return aligned(p, 16) && s0 % 8 == 0 && s1 % 8 == 0; }

int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return 0;
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return KDA355_ELAUNCH;
}

int check_decode_sizes(const KdaLatentDecodeArgs* a) {
    KDA_CHECK_ARG(a != nullptr, "latent_decode: null args");
    KDA_CHECK_ARG(a->B >= 0 && a->S >= 1 && a->H >= 1 && a->page_size >= 1 && a->table_width >= 0 && a->prefix_width >= 0 &&
                      a->num_cus >= 0,
                  "latent_decode: B=%d S=%d H=%d page_size=%d table_width=%d prefix_width=%d num_cus=%d", a->B, a->S, a->H,
                  a->page_size, a->table_width, a->prefix_width, a->num_cus);
    KDA_CHECK_ARG((int64_t)a->B * a->S * a->H < (1ll << 31), "latent_decode: B * S * H is too large");
    KDA_CHECK_ARG((int64_t)a->table_width * a->page_size < (1ll << 31) && (int64_t)a->prefix_width * a->page_size < (1ll << 31),
                  "latent_decode: a table spans 2^31 tokens or more");
    return 0;
}

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int64_t kda355_latent_decode_workspace_bytes(const KdaLatentDecodeArgs* a) {
    if (const int rc = check_decode_sizes(a)) return rc;
    return 0;
}

extern "C" int kda355_latent_decode_launch(const KdaLatentDecodeArgs* a, kda355_stream_t stream) {
    if (const int rc = check_decode_sizes(a)) return rc;
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "latent_decode: dtype %d", a->dtype);
    KDA_CHECK_ARG(a->flags == 0, "latent_decode: unknown flags 0x%x", a->flags);
    if (a->B == 0) return 0;
    KDA_CHECK_ARG(a->q_latent && a->q_pe && a->cache && a->block_table && a->seq_lens && a->out && a->table_width >= 1,
                  "latent_decode: a required pointer is null");
    KDA_CHECK_ARG(!a->prefix_table || (a->prefix_len && a->prefix_width >= 1), "latent_decode: prefix_table needs prefix_len");
    KDA_CHECK_ARG(a->pages >= 1 && a->table_stride >= a->table_width, "latent_decode: pages=%lld table_stride=%lld",
                  (long long)a->pages, (long long)a->table_stride);
    KDA_CHECK_ARG(rows16(a->q_latent, a->ql_row, a->ql_head) && rows16(a->q_pe, a->qp_row, a->qp_head) &&
                      rows16(a->out, a->out_row, a->out_head),
                  "latent_decode: q and out rows must be 16-byte aligned");
    KDA_CHECK_ARG(rows16(a->cache, a->page_stride) && a->page_stride >= (int64_t)a->page_size * ROW,
                  "latent_decode: cache pages must be dense and 16-byte aligned");
    const int64_t need = kda355_latent_decode_workspace_bytes(a);
    KDA_CHECK_ARG(need == 0 || (a->workspace && aligned(a->workspace, 256) && a->workspace_bytes >= need),
                  "latent_decode: needs %lld bytes of 256-byte aligned workspace", (long long)need);
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)(a->B * a->S), a->H);
    if (a->dtype == KDA355_DTYPE_BF16)
        hipLaunchKernelGGL(decode_kernel<__bf16>, grid, dim3(256), 0, s, *a);
    else
        hipLaunchKernelGGL(decode_kernel<_Float16>, grid, dim3(256), 0, s, *a);
    return launched("latent_decode");
}
