// What the 4-bit kernels share: how numbers of 4 bits are stored, quantised and fed to the tensor cores.
//
// A number q of 0 .. 15 stands for  step * q + low  (both bfloat16, one pair per group of numbers; two numbers lie in a
// byte, the first in its low half).  A group with a number that is not finite has step = low = NaN.
//
// The products run on mma.sync m16n8k32 with 8-bit floating operands.  The bytes 0 .. 15 read as e4m3 are exactly
// q * 2^-9 (subnormals up to 7, then the first normal numbers with the same spacing), so unpacking is an AND and a
// shift: three instructions for eight numbers, where a bfloat16 operand takes eleven, and this part's integer
// pipe runs only two warp instructions a cycle (measured: lop3, prmt and shf 1.98 per cycle and SM).  The other operand, x, is
// scaled by a power of two so that its largest magnitude lies in [128, 256), and split into two parts of 8 bits:
//   hi = e4m3(x')  (4 significant bits, rounded to nearest),  lo = e5m2(x' - hi)  (3 significant bits, down to 2^-16).
// Where hi is a normal number (x' >= 2^-6), what it leaves of a bfloat16 (8 significant bits) is a whole number of -8 .. 8 in
// units of x's last place, and all of those have at most 3 significant bits: hi + lo is x' exactly, down to 2^-14 of the
// largest.  Below, hi is within 2^-10 and lo within an eighth of the rest: 2^-14 absolutely, 2^-21 of the largest.  Measured on a
// B200: the e4m3 form issues 0.89 per cycle and SM against 0.48 for bfloat16 m16n8k16, so even in two parts it does 1.9
// times as many products; and it sums its 32 exact products and the accumulator before one rounding to nearest float32
// (checked: 2^25 + 3 is 2^25 + 4, 2^28 + 32 products of 1 is 2^28 + 32).
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

#define I4_GROUP_W 128            // inputs that share a step in a weight
#define I4_GROUP_KV 64            // numbers of a head that share a step in the cache
#define I4_TILE 1088              // bytes of a weight's tile: 16 outputs x 128 inputs, then 16 x (step, low)
#define I4_TILE_CODES 1024

// c += a b for a 16 x 32 (codes as e4m3) and b 32 x 8, hi parts e4m3 or lo parts e5m2
__device__ __forceinline__ void i4_mma_hi(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void i4_mma_lo(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e5m2.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t i4_low(uint32_t w) { return w & 0x0F0F0F0Fu; }              // numbers 0, 2, 4, 6 of eight
__device__ __forceinline__ uint32_t i4_high(uint32_t w) { return (w >> 4) & 0x0F0F0F0Fu; }      // numbers 1, 3, 5, 7

__device__ __forceinline__ uint32_t i4_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two f16 -> their hi parts (two e4m3 in 16 bits) and lo parts (two e5m2)
__device__ __forceinline__ void i4_split2(uint32_t x, uint32_t& hi, uint32_t& lo) {
    uint16_t h, l;
    uint32_t back, rest;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(h) : "r"(x));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(back) : "h"(h));
    asm("sub.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(x), "r"(back));
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(l) : "r"(rest));
    hi = h;
    lo = l;
}
// four scaled numbers -> a word of hi parts and a word of lo parts
__device__ __forceinline__ void i4_split4(float a, float b, float c, float d, uint32_t& hi, uint32_t& lo) {
    uint32_t h0, l0, h1, l1;
    i4_split2(i4_f16x2(a, b), h0, l0);
    i4_split2(i4_f16x2(c, d), h1, l1);
    hi = __byte_perm(h0, h1, 0x5410);
    lo = __byte_perm(l0, l1, 0x5410);
}
// The power of two that x is multiplied by so that a largest magnitude `most` lands in [128, 256), and its inverse.  Below 2^-119 the
// factor stays at 2^126 (a larger one is no float32).
__device__ __forceinline__ float i4_factor(float most, float& inverse) {
    int e = (int)(__float_as_uint(most) >> 23) - 127;                    // floor(log2 most); -127 for zero and subnormals
    e = max(e, -119);
    inverse = __uint_as_float((uint32_t)(e - 7 + 127) << 23);
    return __uint_as_float((uint32_t)(7 - e + 127) << 23);
}

__device__ __forceinline__ float i4_bf16_low(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float i4_bf16_high(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }

// The largest bfloat16 not above x / the smallest not below it (x finite)
__device__ __forceinline__ float i4_down(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float(((u >> 31) ? u + 0xFFFFu : u) & 0xFFFF0000u);
}
__device__ __forceinline__ float i4_up(float x) {
    const uint32_t u = __float_as_uint(x);
    return __uint_as_float(((u >> 31) ? u : u + 0xFFFFu) & 0xFFFF0000u);
}
// Step and low value of a group with smallest number `mn` and largest `mx`: low = mn, step = (mx - mn) / 15, both rounded to bfloat16
// so that low + 15 step reaches mx.  Halves are taken first so that the difference of two numbers near the largest float32
// stays finite.
__device__ __forceinline__ void i4_step_low(float mn, float mx, bool finite, float& step, float& low) {
    low = i4_down(mn);
    const float exact = __fdiv_rn(__fsub_rn(mx * 0.5f, low * 0.5f), 7.5f);
    step = i4_up(exact);
    if (fmaf(15.f, step, low) > 3.402823466e38f) step = i4_down(exact);       // 15 steps up is beyond the largest float32
    if (!finite || !(step <= 3.4e38f) || !(fabsf(low) <= 3.4e38f)) step = low = __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t i4_code(float x, float step, float low) {
    if (!(step > 0.f)) return 0;                                         // all numbers alike, or not finite
    return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x * 0.5f, low * 0.5f), step * 0.5f)), 0.f), 15.f);
}
__device__ __forceinline__ uint32_t i4_meta(float step, float low) {     // both are bfloat16 numbers already
    return (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xFFFF0000u);
}
