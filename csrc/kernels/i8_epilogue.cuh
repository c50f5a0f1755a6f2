// What becomes of a whole-number sum: times both scales, gated, + bias, + residual.  One set of operations, each rounded as it says and none contracted or
// flushed by a file's compiler flags, so that the kernels for few tokens, for a batch and for prompts give the same bits.
#pragma once
#include "common.cuh"

namespace nkb {

__device__ __forceinline__ float mul_rn(float a, float b) {
  float d;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float add_rn(float a, float b) {
  float d;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float2 mul2_rn(float2 a, float2 b) {
  uint64_t rd;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return reinterpret_cast<float2&>(rd);
}

// A sum times its scales; two of one token.
__device__ __forceinline__ float i8_scaled(int sum, float sx, float sw) { return mul_rn(mul_rn(float(sum), sx), sw); }
__device__ __forceinline__ float2 i8_scaled2(uint32_t a, uint32_t b, float2 sx, float sa, float sb) {
  return mul2_rn(mul2_rn(make_float2(float(int(a)), float(int(b))), sx), make_float2(sa, sb));
}

// 1 / (1 + 2^e) by the special-function unit, two steps of it off.
__device__ __forceinline__ float one_over_one_plus_exp2(float e) {
  float t, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(e));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(add_rn(1.f, t)));
  return r;
}
// The gate's exponent e with act(g) = g / (1 + 2^e).  SiLU: -g / ln 2; GELU in its tanh form, (1 + tanh w) / 2 = 1 / (1 + exp(-2 w)) with
// w = sqrt(2 / pi) (g + 0.044715 g^3): -2 w / ln 2.
__device__ __forceinline__ float gelu_exponent(float g) {
  return mul_rn(mul_rn(g, __fmaf_rn(mul_rn(g, g), 0.044715f, 1.f)), -2.302208198f);
}
// Gates times what they gate; act 0: SiLU, 1: GELU.
__device__ __forceinline__ float i8_gated(float g, float u, int act) {
  const float e = act ? gelu_exponent(g) : mul_rn(g, -1.4426950408889634f);
  return mul_rn(mul_rn(g, one_over_one_plus_exp2(e)), u);
}
__device__ __forceinline__ float2 i8_gated2(float2 g, float2 u, int act) {
  const float2 e = act ? make_float2(gelu_exponent(g.x), gelu_exponent(g.y)) : mul2_rn(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
  return mul2_rn(mul2_rn(g, make_float2(one_over_one_plus_exp2(e.x), one_over_one_plus_exp2(e.y))), u);
}

}  // namespace nkb
