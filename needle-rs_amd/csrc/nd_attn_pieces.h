// Shared by the attention kernels that put weights and queries into the matrix
// products as two f16 pieces (tree.hip, prefix.hip): the pieces, codes as f16,
// and loads that stop at a buffer's end.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace ndap {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef float floatx2_t __attribute__((ext_vector_type(2)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef float floatx4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef int intx4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// x / d for x, d with x d < 2^32, d > 0: 2^32 / d rounded up is above it by less
// than one, times x / 2^32 by less than 1 / d.
struct Divisor {
    uint32_t up;  // 0 for d = 1
    __host__ static Divisor of(uint32_t d) { return Divisor{uint32_t(((uint64_t(1) << 32) + d - 1) / d)}; }
    __device__ uint32_t quotient(uint32_t x) const { return up ? __umulhi(x, up) : x; }
};

__device__ inline float i8_at(uint32_t dw, int b) { return float(int32_t(dw << (24 - 8 * b)) >> 24); }

// fmaxf of three (a NaN loses), without the copies the compiler makes of
// operands it cannot show to be quiet.
__device__ inline float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Two numbers as an f16 pair, each to the nearest.
__device__ inline uint32_t f16_two(float x0, float x1)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2_t{x0, x1}), f16x2_t));
}

// x0, x1 (below 2^15) as two f16 pairs.  The first piece is off by 2^-11 of x or
// less and the remainder is exact, so that the second, to the nearest too, leaves
// 2^-23 of x at most (of x below 1/4, whose second piece is subnormal, 2^-25) on
// either side: cut off, the pieces left up to 6 2^-24 and always too little.
// (Written out, the remainder is a conversion and a subtraction; v_fma_mix_f32
// does both.)
__device__ inline void split2(float x0, float x1, uint32_t &h, uint32_t &l)
{
    h = f16_two(x0, x1);
    float r0, r1;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(h), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(h), "v"(x1));
    l = f16_two(r0, r1);
}

// The sign bits flipped, code c is c + 128; byte c of two dwords as f16 pairs:
// u + 128 read as a subnormal, times 2^15, less 128 * 2^-9, is code * 2^-9.
template <int C>
__device__ inline uint32_t f16_codes(uint32_t lo, uint32_t hi)
{
    const uint32_t u = __builtin_amdgcn_perm(hi, lo, 0x0c000c00u | uint32_t(4 + C) << 16 | uint32_t(C));
    const f16x2_t m = {_Float16(32768.0f), _Float16(32768.0f)}, a = {_Float16(-0.25f), _Float16(-0.25f)};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, u), m, a));
}

// Bytes 2 I, 2 I + 1 of a dword (sign bits flipped) as an f16 pair of codes:
// 1024 + (c + 128) - 1152.
template <int I>
__device__ inline uint32_t f16_pair(uint32_t x)
{
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, x, I ? 0x04030402u : 0x04010400u);
    const f16x2_t a = {_Float16(-1152.0f), _Float16(-1152.0f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, u) + a);
}

// Loads from a head's rows or scales: past the end (a chunk that is not full,
// at the ring's end) they give zeros.
typedef __amdgpu_buffer_rsrc_t rows_t;

__device__ inline rows_t rows_at(const void *p, uint32_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, int(bytes), 0x00027000);
}

// x as it is: what is added to it afterwards goes into the loads' own offsets.
__device__ inline uint32_t here(uint32_t x)
{
    asm("" : "+v"(x));
    return x;
}

__device__ inline bool any_of(bool b) { return __builtin_amdgcn_ballot_w64(b) != 0; }

// The same, not 0 where it is so.
__device__ inline uint32_t any32(bool b)
{
    const uint64_t m = __builtin_amdgcn_ballot_w64(b);
    return uint32_t(m) | uint32_t(m >> 32);
}

template <typename T>
__device__ inline T vec4(uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    return __builtin_bit_cast(T, u32x4_t{a, b, c, d});
}

}  // namespace ndap
