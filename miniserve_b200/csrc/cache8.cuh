// The paged cache in 8 bits: what a head's vector is held as, and conversions to and from it.
//
// A vector x of d numbers is d codes (e4m3: sign, 4 bits of exponent, 3 of mantissa; 448 the largest) and one byte b, x_i = code_i * 2^(b - 127).
// The exponent e = b - 127 is the smallest with max |x| <= 448 * 2^e, so the largest number keeps all four significant bits and what is up to
// 2^14 times smaller too; a power of two, so that scaling rounds nothing and code * 2^e is a bfloat16 as it stands. e is kept within [-60, 7]:
// beyond 448 * 2^7 numbers saturate (as a cache in 16-bit floats would), below 2^-70 they become zero. A vector with a number that is not finite
// has b = 255 and zero codes: all of it reads as NaN, and a key or value that is masked can do no harm (no code is NaN, ever).
// Pools: codes [pages, kv_heads, page_size, d], exponents [pages, kv_heads, page_size].
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace ms {

constexpr int C8_EXP_MIN = 127 - 60, C8_EXP_MAX = 127 + 7, C8_NAN = 255;

// The byte of a vector whose largest magnitude has these bits (of a float32; NaN and infinity lie above all finite ones).
__device__ __forceinline__ int c8_exponent(uint32_t amax_bits) {
  if (amax_bits >= 0x7F800000u) return C8_NAN;
  // 448 = 1.75 * 2^8: the next exponent up where the mantissa is beyond 0.75
  const int b = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
  return min(max(b, C8_EXP_MIN), C8_EXP_MAX);
}
// 2^-(b - 127): what numbers are multiplied by before they are rounded to codes; 0 for a vector that is not finite
__device__ __forceinline__ float c8_inverse(int b) { return b == C8_NAN ? 0.f : __uint_as_float((uint32_t)(254 - b) << 23); }
// 2^(b - 127), for bytes that the writer never makes too (0 is 2^-127, below float32's normal range); infinity for 255.
__device__ __forceinline__ float c8_power(uint32_t b) { return __uint_as_float(max(b << 23, 0x00400000u)); }
// the same, NaN for a vector that is not finite
__device__ __forceinline__ float c8_factor(int b) { return b == C8_NAN ? __uint_as_float(0x7FFFFFFFu) : c8_power((uint32_t)b); }

// two numbers to two codes (the first in the low byte), rounded to nearest, ties to even, saturating
__device__ __forceinline__ uint32_t c8_codes2(float x0, float x1) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;\n" : "=h"(r) : "f"(x0), "f"(x1));
  return r;
}
__device__ __forceinline__ uint32_t c8_codes4(float x0, float x1, float x2, float x3) { return c8_codes2(x0, x1) | (c8_codes2(x2, x3) << 16); }
// numbers of a vector that is not finite are multiplied by 0, which leaves NaN of them: no code of them is kept
__device__ __forceinline__ uint32_t c8_keep(uint32_t codes, int b) { return b == C8_NAN ? 0u : codes; }

// the two codes in the low (high) half of `w` as two float16 (exact)
__device__ __forceinline__ uint32_t c8_half2_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t c8_half2_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}\n" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ float2 c8_float2(uint32_t half2) { return __half22float2(*reinterpret_cast<const __half2*>(&half2)); }

// a / b of whole numbers, quotients below 2^20: a multiplication by the reciprocal, off by one at most, put right
__device__ __forceinline__ int div_small(int a, int b) {
  int q = (int)((float)a * __frcp_rn((float)b));
  const int r = a - q * b;
  if (r < 0) --q;
  if (r >= b) ++q;
  return q;
}

inline int c8_page_shift(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

}  // namespace ms
