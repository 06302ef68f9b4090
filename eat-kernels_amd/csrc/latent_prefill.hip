// Latent attention, expanded form (gfx950): per-head keys of 128 | 64 (the 64 shared by the heads) and values of 128 over
// packed sequences, causal or not.
//
// A workgroup of 4 wave64 takes 128 query rows of one (sequence, head), 32 a wave, and walks the keys in tiles of 64:
// keys, shared parts and values come straight into LDS (40 KiB a tile, two tiles, so two workgroups share a CU), one barrier
// a tile, the next tile's loads under way while this one is computed.  Per wave and tile: scores 24 MFMAs, running softmax
// in registers, values 16 MFMAs (attend.h has the layouts).
//
// Bound: the matrix cores (40 MFMAs of 32 cycles a wave and tile) and close behind them LDS reads (every A operand is one
// 16-byte read a lane, 8 cycles of the CU's LDS, against 4 MFMAs running at a time) and exponentials.
#include <type_traits>

#include "attend.h"

namespace kda355 {
namespace {

constexpr int BM = 128, BN = 64, WAVES = 4;
constexpr int HD = 128, PE = 64;
constexpr int TILE_V = BN * HD * 2, TILE_PE = 2 * TILE_V, TILE_BYTES = TILE_PE + BN * PE * 2;  // k | v | shared part
constexpr int64_t MAX_ROW = 1 << 23;  // row strides up to this many elements: a tile's byte offsets stay below 2^31

struct Where { int n, tile; };
// row tile `i` of all sequences -> (sequence, its tile); n < 0 past the last one.  Every lane of a wave takes a sequence.
__device__ __forceinline__ Where locate(const int32_t* cu, int N, int64_t T, int i) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int n0 = 0; n0 < N; n0 += 64) {
        const int n = n0 + lane;
        int tiles = 0;
        if (n < N) {
            const int64_t a = min(max((int64_t)cu[n], (int64_t)0), T), b = min((int64_t)cu[n + 1], T);
            tiles = b > a ? (int)((b - a + BM - 1) / BM) : 0;
        }
        int s = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(s, d);
            if (lane >= d) s += y;
        }
        const uint64_t hit = __builtin_amdgcn_ballot_w64(before + s > i);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            return {n0 + l, i - before - (__builtin_amdgcn_readlane(s, l) - __builtin_amdgcn_readlane(tiles, l))};
        }
        before += __builtin_amdgcn_readlane(s, 63);
    }
    return {-1, 0};
}

template <typename T>
__global__ void __launch_bounds__(WAVES * 64, 2) prefill_kernel(KdaLatentPrefillArgs a, int tiles) {
    __shared__ __align__(1024) unsigned char sm[2 * TILE_BYTES];
    const int task = xcd_task(blockIdx.x, gridDim.x);  // an XCD works on few heads at a time: their keys stay in its L2
    const int h = __builtin_amdgcn_readfirstlane(task / tiles);
    const Where at = locate(a.cu_q, a.N, a.Tq, tiles - 1 - (task - h * tiles));  // long walks first
    const int n = __builtin_amdgcn_readfirstlane(at.n);
    if (n < 0) return;
    const int m0 = __builtin_amdgcn_readfirstlane(at.tile) * BM;
    const int64_t q0 = min(max((int64_t)a.cu_q[n], (int64_t)0), a.Tq), k0 = min(max((int64_t)a.cu_k[n], (int64_t)0), a.Tk);
    const int Lq = (int)(min((int64_t)a.cu_q[n + 1], a.Tq) - q0);
    const int Lk = (int)max(min((int64_t)a.cu_k[n + 1], a.Tk) - k0, (int64_t)0);
    const bool causal = a.flags & KDA355_LATENT_CAUSAL;
    const int shift = causal ? Lk - Lq : Lk;  // row i sees keys j <= i + shift, j < Lk
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 31, half = lane >> 5;
    const int row = m0 + 32 * w + c;

    // ---- queries: operand registers, straight from memory (rows past the end repeat the last one)
    u32x4 q[12];
    {
        const uint16_t* qr = static_cast<const uint16_t*>(a.q) + (q0 + min(row, Lq - 1)) * a.q_row + h * a.q_head + 8 * half;
#pragma unroll
        for (int i = 0; i < 12; ++i) q[i] = *reinterpret_cast<const u32x4*>(qr + 16 * i);
    }

    // ---- tile loads: wave w brings tokens 16 w .. 16 w + 15
    const uint16_t* kh = static_cast<const uint16_t*>(a.k) + k0 * a.k_row + h * a.k_head;
    const uint16_t* vh = static_cast<const uint16_t*>(a.v) + k0 * a.v_row + h * a.v_head;
    const uint16_t* ph = static_cast<const uint16_t*>(a.k_pe) + k0 * a.pe_row;
    const uint32_t lds = lds_offset(sm);
    uint32_t koff[4], voff[4], poff[2];  // byte offsets of this lane's pieces (k / v load i: tokens 16 w + 4 i ..; swz16)
    const int lt = 16 * w + (lane >> 4), pt = 16 * w + (lane >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t piece = ((lane & 15) ^ ((lane >> 4) << 2) ^ i) * 16;
        koff[i] = (uint32_t)lt * (uint32_t)(2 * a.k_row) + piece;
        voff[i] = (uint32_t)lt * (uint32_t)(2 * a.v_row) + piece;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) poff[i] = (uint32_t)pt * (uint32_t)(2 * a.pe_row) + ((lane & 7) ^ swz8(pt + 8 * i)) * 16;
    const uint32_t kstep = 8 * (uint32_t)a.k_row, vstep = 8 * (uint32_t)a.v_row, pstep = 16 * (uint32_t)a.pe_row;
    auto load_tile = [&](int j, int buf) {
        const int t0 = j * BN, left = Lk - t0;
        const u32x4 kr = tile_rsrc(kh + (int64_t)t0 * a.k_row), vr = tile_rsrc(vh + (int64_t)t0 * a.v_row),
                    pr = tile_rsrc(ph + (int64_t)t0 * a.pe_row);
        const uint32_t base = lds + buf * TILE_BYTES + 16 * w * (HD * 2), pbase = lds + buf * TILE_BYTES + TILE_PE + 16 * w * (PE * 2);
        auto issue = [&](auto whole) {
            uint32_t ko[4], vo[4], ks[4], vs[4], po[2], ps[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = whole || lt + 4 * i < left;
                ko[i] = in ? koff[i] : LDS_ZERO, ks[i] = i * kstep;
                vo[i] = in ? voff[i] : LDS_ZERO, vs[i] = i * vstep;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) po[i] = whole || pt + 8 * i < left ? poff[i] : LDS_ZERO, ps[i] = i * pstep;
            load_to_lds4(base, kr, ko, ks);
            load_to_lds4(base + TILE_V, vr, vo, vs);
            load_to_lds2(pbase, pr, po, ps);
        };
        if (left >= BN) issue(std::true_type{}); else issue(std::false_type{});
    };

    // ---- LDS read addresses (byte offsets within a tile; key step, value tile and key block are xors and constants)
    const uint32_t ka = c * (HD * 2) + ((half ^ swz16(c)) << 4);
    const uint32_t pa = TILE_PE + c * (PE * 2) + ((half ^ swz8(c)) << 4);
    const int i16 = lane & 15;
    uint32_t va[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int t = 4 * half + 8 * u + (i16 >> 2);
        const int e = 2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1);
        va[u] = TILE_V + t * (HD * 2) + ((e ^ swz16(t)) << 4) + (i16 & 1) * 8;
    }

    const float sc = a.scale * 1.44269504088896f;
    f32x16 acc[4] = {};
    float mo = M_START, l = 0.f;
    bool special = false;
    const int seen = min(Lk, min(m0 + BM, Lq) + shift);        // keys that any row of the workgroup sees
    const int mine = min(Lk, min(m0 + 32 * w + 32, Lq) + shift);  // ... of this wave
    const int full = min(Lk, m0 + 32 * w + 1 + shift);         // keys that every row of this wave sees
    const int ntiles = seen > 0 ? (seen + BN - 1) / BN : 0;

    if (ntiles > 0) load_tile(0, 0);
    for (int j = 0; j < ntiles; ++j) {
        wait_loads<0>();
        lds_barrier();  // tile j is whole, and every wave has read tile j - 1
        if (j + 1 < ntiles) load_tile(j + 1, (j + 1) & 1);
        const int t0 = j * BN;
        if (t0 >= mine) continue;  // wave-uniform; the barrier is at the top
        const uint32_t tb = lds + (j & 1) * TILE_BYTES;
        // ---- scores: 24 steps (key step i of 12, key block b of 2), the operands of the next four read while four run
        f32x16 s[2] = {};
        auto key = [&](int x) {
            const int i = x >> 1, b = x & 1;
            return i < 8 ? lds_read16((tb + ka + b * 32 * HD * 2) ^ (i << 5)) : lds_read16((tb + pa + b * 32 * PE * 2) ^ ((i - 8) << 5));
        };
        u32x4 kf[2][4];
#pragma unroll
        for (int x = 0; x < 4; ++x) kf[0][x] = key(x);
#pragma unroll
        for (int g = 0; g < 6; ++g) {
            __builtin_amdgcn_sched_barrier(0);
            if (g < 5)
#pragma unroll
                for (int x = 0; x < 4; ++x) kf[(g + 1) & 1][x] = key(4 * g + 4 + x);
#pragma unroll
            for (int x = 0; x < 4; ++x) s[x & 1] = T::mfma(kf[g & 1][x], q[2 * g + (x >> 1)], s[x & 1]);
        }
        __builtin_amdgcn_sched_barrier(0);
        const bool masked = t0 + BN > full;  // some row of the wave does not see some key of the tile
        if (masked) {
            const int last = min(row + shift, Lk - 1) - t0 - 4 * half;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (32 * b + (r & 3) + 8 * (r >> 2) > last) s[b][r] = -INFINITY;
        }
        // ---- running softmax: the maximum is raised, and the accumulator rescaled, only when some row of the wave
        // exceeds it by SLACK (the result is the same for any reference; weights stay within the type's range)
        float mx = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[b][r]);
        mx = max_halves(mx) * sc;
        if (__builtin_amdgcn_ballot_w64(mx - mo > T::B + T::SLACK)) {
            const float mn = mx - mo > T::B + T::SLACK ? mx - T::B : mo;  // by the row's own scores alone
            const float f = __builtin_amdgcn_exp2f(mo - mn);
            mo = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] *= f;
        }
        u32x4 p[4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[b][r], sc, -mo)), y = __builtin_amdgcn_exp2f(fmaf(s[b][r + 1], sc, -mo));
                l += x + y;
                p[2 * b + (r >> 3)][(r >> 1) & 3] = T::pack(x, y);
            }
        // ---- values
        auto value = [&](int k, int d) {
            const u32x2 v0 = lds_read_tr(((tb + va[0]) ^ (d << 6)) + k * 16 * HD * 2);
            const u32x2 v1 = lds_read_tr(((tb + va[1]) ^ (d << 6)) + k * 16 * HD * 2);
            return u32x4{v0.x, v0.y, v1.x, v1.y};
        };
        u32x4 vf[2][4];
#pragma unroll
        for (int d = 0; d < 4; ++d) vf[0][d] = value(0, d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            if (k < 3)
#pragma unroll
                for (int d = 0; d < 4; ++d) vf[(k + 1) & 1][d] = value(k + 1, d);
            if (masked)
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    special |= nonfinite<T>(vf[k & 1][d]);
                    vf[k & 1][d] = finite_part<T>(vf[k & 1][d]);
                }
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[d] = T::mfma(vf[k & 1][d], p[k], acc[d]);
        }
    }

    if (__builtin_amdgcn_ballot_w64(special)) {  // infinite or NaN values among the keys that not every row sees
        const int last = min(row + shift, Lk - 1);
#pragma unroll 1
        for (int j = max(full, 0) & ~(BN - 1); j < mine; ++j) {
            const uint16_t* vr = vh + (int64_t)j * a.v_row + 4 * half;
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = T::up(vr[32 * d + 8 * g + e]);
                        if (j <= last && !(fabsf(x) < INFINITY)) acc[d][4 * g + e] += x;
                    }
        }
    }

    // ---- o = acc / l
    l = sum_halves(l);
    if (row >= Lq) return;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint16_t* o = static_cast<uint16_t*>(a.out) + (q0 + row) * a.out_row + h * a.out_head + 4 * half;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float x0 = acc[d][4 * g] * inv, x1 = acc[d][4 * g + 1] * inv, x2 = acc[d][4 * g + 2] * inv, x3 = acc[d][4 * g + 3] * inv;
            *reinterpret_cast<u32x2*>(o + 32 * d + 8 * g) =
                l == 0.f ? u32x2{0u, 0u} : u32x2{T::pack(x0, x1), T::pack(x2, x3)};
        }
    if (a.lse && half == 0)
        a.lse[(q0 + row) * a.H + h] = l == 0.f ? -INFINITY : (mo + __builtin_amdgcn_logf(l)) * 0.69314718055995f;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// rows of 16-byte pieces: aligned base, strides in multiples of 8 elements
bool rows16(const void* p, int64_t s0, int64_t s1 = 0) { return aligned(p, 16) && s0 % 8 == 0 && s1 % 8 == 0; }
bool near(int64_t row) { return row >= 0 && row <= MAX_ROW; }

}  // namespace
}  // namespace kda355

using namespace kda355;

extern "C" int kda355_latent_prefill_launch(const KdaLatentPrefillArgs* a, kda355_stream_t stream) {
    KDA_CHECK_ARG(a != nullptr, "latent_prefill: null args");
    KDA_CHECK_ARG(a->N >= 0 && a->H >= 1 && a->Tq >= 0 && a->Tk >= 0, "latent_prefill: N=%d H=%d Tq=%lld Tk=%lld", a->N, a->H,
                  (long long)a->Tq, (long long)a->Tk);
    KDA_CHECK_ARG(a->dtype == KDA355_DTYPE_BF16 || a->dtype == KDA355_DTYPE_FP16, "latent_prefill: dtype %d", a->dtype);
    KDA_CHECK_ARG((a->flags & ~KDA355_LATENT_CAUSAL) == 0, "latent_prefill: unknown flags 0x%x", a->flags);
    if (a->N == 0 || a->Tq == 0) return 0;
    KDA_CHECK_ARG(a->Tq < (1ll << 30) && a->Tk < (1ll << 30), "latent_prefill: 2^30 tokens or more");
    KDA_CHECK_ARG(a->q && a->out && a->cu_q && a->cu_k && (a->Tk == 0 || (a->k && a->v && a->k_pe)),
                  "latent_prefill: a required pointer is null");
    KDA_CHECK_ARG(rows16(a->q, a->q_row, a->q_head) && rows16(a->k, a->k_row, a->k_head) && rows16(a->v, a->v_row, a->v_head) &&
                      rows16(a->k_pe, a->pe_row) && rows16(a->out, a->out_row, a->out_head),
                  "latent_prefill: rows must be 16-byte aligned");
    KDA_CHECK_ARG(near(a->k_row) && near(a->v_row) && near(a->pe_row), "latent_prefill: token strides of k, v and k_pe must be at most 2^23");
    KDA_CHECK_ARG(a->scale > 0.f, "latent_prefill: scale must be positive");
    const int64_t tiles = a->Tq / BM + a->N;  // at least the sum of every sequence's row tiles
    KDA_CHECK_ARG(tiles * a->H < (1ll << 23), "latent_prefill: grid too large");
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid((uint32_t)(tiles * a->H));
    if (a->dtype == KDA355_DTYPE_BF16)
        hipLaunchKernelGGL(prefill_kernel<Bf16>, grid, dim3(WAVES * 64), 0, s, *a, (int)tiles);
    else
        hipLaunchKernelGGL(prefill_kernel<Fp16>, grid, dim3(WAVES * 64), 0, s, *a, (int)tiles);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        set_error("latent_prefill: launch failed: %s", hipGetErrorString(e));
        return KDA355_ELAUNCH;
    }
    return 0;
}
