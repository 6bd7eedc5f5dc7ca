// What the 4-bit kernels share: how numbers of 4 bits are stored, quantised and fed to the tensor cores.
//
// A number q of 0 .. 15 stands for  step * q + low  (both bfloat16, one pair per group of numbers; two numbers lie in a
// byte, the first in its low half).  A group with a number that is not finite has step = low = NaN.
//
// The products run on mma.sync m16n8k16 with f16 operands.  The bits 0 .. 15 of a nibble in a half word are, read as f16, exactly
// q * 2^-24 (subnormal numbers are evenly spaced), and four bits further up q * 2^-20: a word of eight numbers becomes four operand
// registers with a shift and four ANDs, no conversion.  (A bfloat16 operand takes a third more and a subtraction on a pipe that
// issues two warp instructions a cycle and SM; 8-bit operands are turned into f16 by instructions of their own, 0.14 products
// of k 32 a cycle measured against 0.47 of k 16 in f16 or bfloat16.)  The other operand x is scaled by a power of two
// so that its largest magnitude lies in [2^14, 2^15), those that meet numbers four bits up by 2^-4 of that, and converted to
// f16, which has 11 significant bits: exact for a bfloat16 (8 bits) down to 2^-28 of the largest, and within 2^-35 of the
// largest below.  Products are exact.  Their sums are a float32's only where the x of an instruction (16 inputs) lie within 2^7 of each other:
// the tensor cores line products up by their operands' exponents, a subnormal number's is 2^-14 whatever its leading zeros, and
// what is below 2^-24 of the largest so found is cut off.  In units of code times x that is 2^-14 of the largest of the 16 x, for each of the
// 16 and for the sum so far; measured up to 1.6 such units where x spans 2^12, none where it is normally distributed, with or without a few
// inputs 300 times as large.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

#define I4_GROUP_W 128            // inputs that share a step in a weight
#define I4_GROUP_KV 64            // numbers of a head that share a step in the cache
#define I4_TILE 1088              // bytes of a weight's tile: 16 outputs x 128 inputs, then 16 x (step, low)
#define I4_TILE_CODES 1024

// c += a b for a 16 x 16 (codes) and b 16 x 8
__device__ __forceinline__ void i4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void i4_mma_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
#define I4_NEAR 0x000F000Fu       // numbers 0 and 4 of a word (shifted by 8: 2 and 6), as q * 2^-24
#define I4_FAR 0x00F000F0u        // numbers 1 and 5 (3 and 7), as q * 2^-20
#define I4_UNIT 5.9604644775390625e-08f      // 2^-24

__device__ __forceinline__ uint32_t i4_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Eight scaled numbers as the registers that meet a word's: (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16
__device__ __forceinline__ uint4 i4_operand(const float (&a)[8]) {
    return make_uint4(i4_f16x2(a[0], a[4]), i4_f16x2(a[1] * 0.0625f, a[5] * 0.0625f), i4_f16x2(a[2], a[6]),
                      i4_f16x2(a[3] * 0.0625f, a[7] * 0.0625f));
}
// The power of two that brings a largest magnitude `most` into [2^14, 2^15), and the exponent e of its inverse 2^(e - 14).  Below 2^-112
// the factor stays at 2^126 (a larger one is no float32).
__device__ __forceinline__ float i4_factor(float most, int& e) {
    e = max((int)(__float_as_uint(most) >> 23) - 127, -112);             // floor(log2 most); -127 for zero and subnormals
    return __uint_as_float((uint32_t)(14 - e + 127) << 23);
}
__device__ __forceinline__ float i4_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // -126 <= e <= 127

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
// stays finite.  What the codes stand for has to be a bfloat16: numbers beyond the largest one count as that one, and a step that would
// lead beyond it is rounded down (mx then lies an eighth of a step above code 15, still nearest to it).
__device__ __forceinline__ void i4_step_low(float mn, float mx, bool finite, float& step, float& low) {
    constexpr float MOST = 3.38953139e38f;                               // the largest bfloat16
    mn = fmaxf(fminf(mn, MOST), -MOST), mx = fmaxf(fminf(mx, MOST), -MOST);
    low = i4_down(mn);
    const float exact = __fdiv_rn(__fsub_rn(mx * 0.5f, low * 0.5f), 7.5f);
    step = i4_up(exact);
    if (fmaf(15.f, step, low) > MOST) step = i4_down(exact);
    if (!finite) step = low = __uint_as_float(0x7FC00000u);
}
__device__ __forceinline__ uint32_t i4_code(float x, float step, float low) {
    if (!(step > 0.f)) return 0;                                         // all numbers alike, or not finite
    return (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x * 0.5f, low * 0.5f), step * 0.5f)), 0.f), 15.f);
}
__device__ __forceinline__ uint32_t i4_meta(float step, float low) {     // both are bfloat16 numbers already
    return (__float_as_uint(step) >> 16) | (__float_as_uint(low) & 0xFFFF0000u);
}
