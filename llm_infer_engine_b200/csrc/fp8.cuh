// Numbers of a cache in 8 bits: e4m3 codes with a power of two for each block of 16 positions of a head.
//
// A number x of a block is held as the code c = e4m3(x 2^-e), to the nearest and ties to even, and read as c 2^e. The block's
// exponent e is the smallest in [kExpMin, kExpMax] with (largest finite magnitude of the block) 2^-e <= 448, the largest
// e4m3 number. Why a power of two: multiplying by 2^-e rounds nothing, so a number is rounded once; a block whose exponent
// has to rise for a later position keeps its codes' digits (a code shifted down rounds a second time only where it falls below
// 2^-6, the smallest normal one, under 2^-13 of the block's largest number); and attention takes a block's scale as an addend of exponents.
// The relative error of a number is at most 2^-4 (half a step of 3 digits) as long as it is within 2^-13 of its block's
// largest, whose code is above 224. A smaller one is off by at most 2^-10 2^e, half the smallest step, and by as much again where an
// exponent rose over it. What is not finite is held as the code NaN, so that it shows; it does not enter the block's exponent.
#pragma once
#include "common.cuh"
#include <cuda_fp16.h>

namespace llmie {

constexpr int kExpBlock = 16;        // positions that share an exponent
constexpr int kFp8Page = 64;         // positions of a cache page
constexpr int kPageExps = kFp8Page / kExpBlock;
constexpr int kMostPages = 0x7fffffff / kFp8Page;            // of a table, that positions can be counted in 32 bits
constexpr int kExpMin = -64;         // blocks of zeros, and of numbers below 448 * 2^-64
constexpr int kExpMax = 119;         // numbers above 448 * 2^119 are held as that

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2_of(int e) { return __int_as_float((e + 127) << 23); }

// The exponent for a block whose largest finite magnitude has these bits: magnitude = m 2^x, m in [1, 2), and 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(unsigned bits) {
  const int x = (int)(bits >> 23) - 127;
  const int e = x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return bits == 0u ? kExpMin : min(max(e, kExpMin), kExpMax);
}
// The bits of |v|, or 0 where v is not finite.
__device__ __forceinline__ unsigned finite_magnitude(float v) {
  const unsigned b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ int clamp_exponent(int e) { return min(max(e, kExpMin), kExpMax); }

// Values of very different size. The tensor-core kernels weight a value's codes with w = 2^(s + ev - R + 7), R the largest s + ev so far
// less a slack of 8 at most, and sum the softmax's denominator from the same numbers, w 2^(-ev). Beside a block of far larger values, w is
// below float32 while w 2^(-ev) is not: it is nothing for the numerator, and may be all of the denominator (16 values of 1e30 and 16 zeros
// that are seen alike are 5e29 on average, not 1e30).
//   What is lost so is below 2^-126 2^64 = 2^-62 a key, and below 2^(15 + 64 - 126) = 2^-47 where a sum was brought to a bound more than
// 2^126 above; 2^20 keys together lose less than 2^-27. A denominator from 2^-12 on lacks less than 2^-15 of itself. A smaller one is
// that of R's own value, 2^(7 - ev) at least, with ev > 19 (values above 2e8), or of others as large: it is taken once more by the scores
// alone, sum_j 2^(s_j - R + 7). Those terms are below 2^(7 + 8 + 64) and the sum is at least 2^(7 - 119); their exponentials are taken 2^20
// larger, so that those above 2^-34 of it come out normal.
constexpr float kLeastDenominator = 0x1p-12f;
__device__ __forceinline__ float exp2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_term(float x) { return exp2_ftz(x + 20.f) * 0x1p-20f; }
// l 2^d, and sum + l 2^d, for sums l that are relative to a bound d <= 0 below the common one (f is 2^d): where 2^d alone would be below
// float32, in two steps.
__device__ __forceinline__ float times_exp2(float l, float f, float d) {
  if (!(d < -100.f)) return l * f;
  const float half = exp2_ftz(0.5f * d);
  return l * half * half;
}
__device__ __forceinline__ float add_times_exp2(float l, float f, float d, float sum) {
  if (!(d < -100.f)) return fmaf(f, l, sum);
  const float half = exp2_ftz(0.5f * d);
  return fmaf(l * half, half, sum);
}

// Two numbers, scaled, as two codes (a in the low byte); what is not finite becomes NaN.
__device__ __forceinline__ unsigned short to_e4m3x2(float a, float b) {
  a = (__float_as_uint(a) & 0x7f800000u) == 0x7f800000u ? __int_as_float(0x7fffffff) : a;
  b = (__float_as_uint(b) & 0x7f800000u) == 0x7f800000u ? __int_as_float(0x7fffffff) : b;
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// Two codes as two half-precision numbers: exact (e4m3 reaches from 2^-9 to 448).
__device__ __forceinline__ unsigned e4m3x2_to_half2(unsigned short c) {
  unsigned r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(unsigned short c) {
  const unsigned h = e4m3x2_to_half2(c);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Four codes times `factor`, a power of two of 1 at most: moved to a block exponent that is higher.
__device__ __forceinline__ unsigned lower_codes(unsigned w, float factor) {
  const float2 a = e4m3x2_to_float2((unsigned short)(w & 0xffffu)), b = e4m3x2_to_float2((unsigned short)(w >> 16));
  return (unsigned)to_e4m3x2(a.x * factor, a.y * factor) | ((unsigned)to_e4m3x2(b.x * factor, b.y * factor) << 16);
}
// 2^(from - to) for from <= to; below 2^-40 every code becomes zero anyway.
__device__ __forceinline__ float lower_factor(int from, int to) { return pow2_of(max(from - to, -60)); }

}  // namespace llmie
