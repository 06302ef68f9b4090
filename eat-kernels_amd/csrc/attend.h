// What the latent attention kernels share (gfx950, wave64): element types, the 32x32x16 MFMA, loads straight into LDS, the
// running softmax of a 32-row tile, and values that a query does not see.
//
// A wave holds 32 query rows and computes transposed tiles: scores S^T [keys x rows] = K Q^T and outputs O^T [values x rows]
// = V^T P^T, so that a query row is a lane (l % 32, both halves h = l / 32) throughout: the softmax of a row runs down the
// lane's own registers and across the two halves once, and P^T leaves the scores' registers as the second product's operand
// without passing through LDS.  Register r of a 32 x 32 result holds row (r & 3) + 8 (r >> 2) + 4 h; operand element e of a
// lane is the k index 8 h + e.  The second product's k order is free, so element e of its 16-key step s stands for key
// 16 s + 4 h + (e & 3) + 8 (e >> 2), which is the scores' own order; V is read in the same order.
#pragma once
#include "common.h"

namespace kda355 {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

// Element types.  The weights p = 2^(z - m + B) of a row are rounded to the type for the second product: a matrix instruction
// takes both operands in one type, and weights in a high and a low part would be 40 to 47 % more matrix work.  The sums of the
// weights take them as they are, in fp32.  Errors of half a step on either side average over the keys: outputs are off by 1.7e-3 to
// 2.2e-3 of their norm in bf16 and 2.3e-4 to 2.6e-4 in fp16, where the final rounding alone gives 1.6e-3 to 1.7e-3 and 2.0e-4.
// m is a past maximum that z may exceed by SLACK before it is raised (raising it rescales the whole accumulator), so p <= 2^(B +
// SLACK).  bf16 has fp32's range: B = 0.  fp16 ends at 2^16 and loses precision below 2^-14: B = 9 keeps full precision for keys
// down to 2^-23 of the maximum.  z - m is one fused step and m was rounded: scores beyond 2^24, whose fp32 steps are whole units of
// the exponent, can pass fp16's end.
struct Bf16 {
    static constexpr float B = 0.f, SLACK = 8.f;
    static constexpr uint32_t EXP = 0x7f807f80u, EXP_ONE = 0x00800080u;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) { return f2bf2(x, y); }
    static __device__ __forceinline__ float up(uint16_t x) { return bf2f(x); }
    // the codes in byte BYTE
    template <int BYTE>
    static __device__ __forceinline__ uint32_t pair4(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
    }
    // eight 4-bit codes times a power of two (a float of its exponent), each rounded to the type; NaN where the scale is (255)
    static __device__ __forceinline__ u32x4 from4(uint32_t codes, float scale) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
    }
};
struct Fp16 {
    static constexpr float B = 9.f, SLACK = 6.f;
    static constexpr uint32_t EXP = 0x7c007c00u, EXP_ONE = 0x04000400u;
    static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2_t));
    }
    static __device__ __forceinline__ float up(uint16_t x) { return (float)__builtin_bit_cast(_Float16, x); }
    template <int BYTE>
    static __device__ __forceinline__ uint32_t pair4(uint32_t codes, float scale) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE));
    }
    static __device__ __forceinline__ u32x4 from4(uint32_t codes, float scale) {
        return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3))};
    }
};

// ------------------------------------------------------------------------------------------------ LDS
typedef __attribute__((address_space(3))) unsigned char lds_byte;
__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(lds_byte*)p; }

// 64 lanes x 16 bytes from global memory into 1 KiB of LDS at byte `lds` (wave-uniform), lane l's piece at lds + 16 l, from byte
// voff (a lane's) of the descriptor; pieces past its size read as zeros.  In asm, because the compiler would wait for every
// such load before any read of LDS; whoever reads the data waits with wait_loads() and a barrier.  A vector memory instruction
// may read an SGPR that a vector instruction wrote (readlane: spilled descriptors too) five wait states later at the earliest,
// and the compiler does not look into asm: s_nop 4.  A CU takes about 16 cycles a load, and a wave that asks for more than a few
// at once stalls: the kernels spread them between matrix instructions.
__device__ __forceinline__ void load_to_lds(uint32_t lds, u32x4 rsrc, uint32_t voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(lds)),
                 "v"(voff), "s"(rsrc)
                 : "memory");
}
// 64 lanes x 16 bytes from src (a lane's) + OFFSET into a block of LDS (the instruction adds its offset to both addresses)
template <int OFFSET>
__device__ __forceinline__ void load_block(uint32_t lds, uint64_t src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off offset:%2" ::"s"(__builtin_amdgcn_readfirstlane(lds - OFFSET)),
                 "v"(src), "n"(OFFSET)
                 : "memory");
}
// the same from a wave's address and a lane's offset (s_nop 4: see load_to_lds)
__device__ __forceinline__ void load_block_from(uint32_t lds, uint64_t base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base) : "memory");
}
__device__ __forceinline__ void load_words_from(uint32_t lds, uint64_t base, uint32_t off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(off), "s"(base) : "memory");
}
// 64 lanes x 4 bytes, lane l's to lds + 4 l
__device__ __forceinline__ void load_words(uint32_t lds, uint64_t src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(src) : "memory");
}
__device__ __forceinline__ u32x4 tile_rsrc(const void* base, uint32_t size) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a), (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)),
                 (uint32_t)__builtin_amdgcn_readfirstlane(size), 0x00020000u};
}
template <int N>
__device__ __forceinline__ void wait_loads() {  // all but the N youngest loads of this wave have arrived
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ u32x4 lds_read16(uint32_t at) {
    return *(__attribute__((address_space(3))) const u32x4*)(lds_byte*)(uintptr_t)at;
}
// transposed read of bytes: of 16 lanes, lane i gives the address of 8; lane i receives column i of the 8 x 16 matrix whose row r are the
// bytes at lanes 2 r and 2 r + 1
typedef int i32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 lds_read_tr8(uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(lds_byte*)(uintptr_t)at));
}
// transposed read: of 16 lanes, lane i gives the address of 4 elements; lane i receives element i % 4.. column i of the
// 4 x 16 matrix whose row r are the elements at lanes 4 r .. 4 r + 3
__device__ __forceinline__ u32x2 lds_read_tr(uint32_t at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_byte*)(uintptr_t)at));
}

// Token rows of 16-byte pieces in LDS: piece c of token t stands at c ^ f(t), f(t) = 4 (t & 3) + ((t >> 2) & 3), within
// each 16 pieces.  Rows are a multiple of 256 bytes (all 64 banks), so the piece position alone picks the banks: 16 lanes
// that read one piece of 16 consecutive tokens, and 16 lanes of a transposed read (4 consecutive pieces of 4 consecutive
// tokens), both touch all 16 positions.
__device__ __forceinline__ int swz16(int t) { return ((t & 3) << 2) | ((t >> 2) & 3); }
// rows of 8 pieces (two tokens a bank sweep): c ^ ((t >> 1) & 7)
__device__ __forceinline__ int swz8(int t) { return (t >> 1) & 7; }

// ------------------------------------------------------------------------------------------------ lanes
__device__ __forceinline__ float max_halves(float x) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float sum_halves(float x) {
    const u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// inclusive prefix sum over the lanes (all of them active)
__device__ __forceinline__ int scan_wave(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // within 16 lanes: 1, 2, 4, 8 below
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // lanes 15 and 47 to the 16 after them
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // lane 31 to the upper half
    return x;
}

// the sum over the lanes, in every lane
__device__ __forceinline__ float sum_wave(float x) {
    auto add = [&](int y) { x += __uint_as_float((uint32_t)y); };
    auto bits = [&] { return (int)__float_as_uint(x); };
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x111, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x112, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x114, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x118, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x142, 0xa, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, bits(), 0x143, 0xc, 0xf, false));
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane(bits(), 63));
}

// ------------------------------------------------------------------------------------------------ running softmax
// State of a lane's row: mo = m - B in log2 units, l = this half's sum of the weights.  Starts far below any score but
// finite, so that hidden scores (-inf) give weights of 0 and never a NaN.
constexpr float M_START = -1e30f;

// ------------------------------------------------------------------------------------------------ values nobody sees
// A product with weight 0 is not 0 where the value is infinite or NaN.  In tiles where some rows see a key and others do
// not, values that are not finite are taken out of the matrix product; a kernel that met one gives it to the rows that see
// it once its key loop is done.
template <typename T>
__device__ __forceinline__ bool nonfinite(u32x4 a) {
    uint32_t f = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) f |= (a[i] & T::EXP) + T::EXP_ONE;  // the exponent's carry reaches the half's top bit
    return (f & 0x80008000u) != 0;
}
// the finite values, zeros in place of the others
template <typename T>
__device__ __forceinline__ u32x4 finite_part(u32x4 v) {
    constexpr uint32_t E = T::EXP & 0xffffu;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] &= ((v[i] & E) == E ? 0u : 0xffffu) | ((v[i] >> 16 & E) == E ? 0u : 0xffff0000u);
    return v;
}

}  // namespace kda355
