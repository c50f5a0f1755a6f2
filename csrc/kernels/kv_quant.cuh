// Keys and values in 8 bits.  A page of 32 tokens of one kv head is e4m3 values [32][D] and one byte per token, 127 + e for the power
// of two 2^e that the token's row is multiplied by (255: the row stands for NaN, and its values are 0).  e is the smallest whole number
// for which the row's largest magnitude is at most 448 * 2^e, between kQ8MinLog2 and kQ8MaxLog2.
#pragma once
#include <cuda_fp8.h>
#include "common.cuh"

namespace nkb {

constexpr int kQ8Page = 32;
constexpr int kQ8MinLog2 = -64, kQ8MaxLog2 = 64;

// 64 bits to 32, rounded to odd: a later rounding to fewer bits gives what one rounding from 64 bits would have given.  Beyond the
// largest finite number it stays finite.
__device__ __forceinline__ float round_to_odd(double x) {
  const float f = __double2float_rz(x);
  return double(f) != x && x == x ? __int_as_float(__float_as_int(f) | 1) : f;
}

// e of a row whose largest magnitude is amax (finite)
__device__ __forceinline__ int q8_log2_scale(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);      // 448 is 1.75 * 2^8
  return min(max(e, kQ8MinLog2), kQ8MaxLog2);
}
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((127 + e) << 23); }    // -126 <= e <= 127

// a token's scale byte as the factor and its logarithm; bytes that no row has are taken to the nearest that one may have
__device__ __forceinline__ int q8_log2_of(int byte) { return min(max(byte - 127, kQ8MinLog2), kQ8MaxLog2); }
__device__ __forceinline__ float q8_factor_of(int byte) {
  return byte == 255 ? __int_as_float(0x7fc00000) : exp2_int(q8_log2_of(byte));
}

// two values to e4m3, nearest even, beyond 448 to 448; the first in the low byte
__device__ __forceinline__ uint16_t pack_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
// two e4m3 values as f16 (exact), the low byte first
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

}  // namespace nkb
