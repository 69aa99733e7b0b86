// Keys and values in pages of 8 bits, shared by the kernels that write and read them.
//
// A page's rows of one KV head are e4m3 values with one scale s = 2^e: row element = value * s, e the least whole number from EXP_MIN
// on with max |x| <= 448 * 2^e over the rows that the page holds.  A power of two, because e4m3 is a floating-point format: the
// values then keep their bits whatever e is, a page whose largest number grows has its earlier rows moved to the new scale without another
// rounding (but for those that become subnormal), and readers multiply by it exactly.  The scale of a page in which a key or value is
// NaN or infinite is NaN: whoever may read a row of that page gets NaN, nobody else does.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace cache8 {
constexpr int EXP_MIN = -100;                // pages of numbers below 448 * 2^-100 count as that large

// the scale of a page whose largest |x| has these bits (0 <= x; NaN and infinities order above all numbers)
__device__ __forceinline__ float scale_of(unsigned top_bits) {
    if (top_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    // x = 1.m * 2^(b - 127) and 448 = 1.75 * 2^8
    const int e = (int)(top_bits >> 23) - 127 - 8 + ((top_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((unsigned)(max(e, EXP_MIN) + 127) << 23);
}
// 1 / s for such a scale (NaN for NaN); e <= 120, so the quotient is a normal number
__device__ __forceinline__ float inverse_of(float s) {
    return s == s ? __uint_as_float((254u << 23) - __float_as_uint(s)) : s;
}
// two numbers to e4m3, nearest even: `lo` in the low byte
__device__ __forceinline__ unsigned short to_e4m3x2(float lo, float hi) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// two e4m3 values as halves, exact
__device__ __forceinline__ unsigned to_half2(unsigned short v) {
    unsigned r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ unsigned half2_low(unsigned v) { return to_half2((unsigned short)(v & 0xffffu)); }
__device__ __forceinline__ unsigned half2_high(unsigned v) { return to_half2((unsigned short)(v >> 16)); }
}  // namespace cache8
