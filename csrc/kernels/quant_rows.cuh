// Rows brought into 8-bit whole numbers, device code of quant_rows.cu and gemm_i8_few.cu (compiled without fast math): quant_rows.cu has the mathematics.
#pragma once
#include "common.cuh"

namespace nkb {

// Distance from a whole number beyond which a gated one is decided in 64 bits: half, less 127 times the error of a gated value in 32 bits and that of its
// quotient by the row's largest, 2 * 2^-24.  The value's is 28 * 2^-24 where gate and up are rounded sums (the exponential multiplies the gate's rounding by the gate, -20 at
// the least: gates below are in 64 bits from the start, kFar in quant_rows.cu), and below 2^-21 where both are given (the exponential, 1 +, the quotient,
// the product).
constexpr float kNearHalfGated = 0.5f - 1.f / 4096, kNearHalfGatedOnce = 0.5f - 1.f / (1 << 13);
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Bytes [by, by + 16) of 32; by: even, below 16.
__device__ __forceinline__ uint4 moved(const uint32_t (&v)[8], uint32_t by) {
  uint32_t u[7], t[5];
#pragma unroll
  for (int j = 0; j < 7; ++j) u[j] = by & 4u ? v[j + 1] : v[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) t[j] = by & 8u ? u[j + 2] : u[j];
  const uint32_t half = (by & 2u) * 8u;
  return make_uint4(__funnelshift_r(t[0], t[1], half), __funnelshift_r(t[1], t[2], half), __funnelshift_r(t[2], t[3], half), __funnelshift_r(t[3], t[4], half));
}
// The two pieces of sixteen bytes that 8 columns from p on lie in, where `inside` says that both lie within the rows' memory.
struct Pieces {
  uint4 lo, hi;
};
__device__ __forceinline__ Pieces fetch_pieces(const uint16_t* p, bool inside) {
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) & ~uintptr_t(15));
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  return {inside ? __ldg(q) : none, inside ? __ldg(q + 1) : none};
}
// 8 columns from `c` on of a row, as they lie in memory; columns past the width read as zeros.  VEC: rows start on 16 bytes; others column by column, or
// from the pieces.  (Through the read-only path: a thread's loads may then go ahead of its stores, which in place follow the loads of the same columns.)
__device__ __forceinline__ uint4 fetch8_each(const uint16_t* p, int columns) {
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < columns) w[j >> 1] |= uint32_t(__ldg(p + j)) << (16 * (j & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 from_pieces(const Pieces& t, const uint16_t* p, bool inside, int columns) {
  if (!inside) return fetch8_each(p, columns);
  const uint32_t v[8] = {t.lo.x, t.lo.y, t.lo.z, t.lo.w, t.hi.x, t.hi.y, t.hi.z, t.hi.w};
  return moved(v, uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u);
}
template <bool VEC>
__device__ __forceinline__ uint4 fetch8_bf16(const void* row, int c, int width) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + c;
  if (VEC && c + 8 <= width) return __ldg(reinterpret_cast<const uint4*>(p));
  return fetch8_each(p, width - c);
}
template <bool VEC>
__device__ __forceinline__ void fetch8_f32(const float* row, int c, int width, uint4 (&r)[2]) {
  if (VEC && c + 8 <= width) {
    r[0] = __ldg(reinterpret_cast<const uint4*>(row + c));
    r[1] = __ldg(reinterpret_cast<const uint4*>(row + c) + 1);
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = c + j < width ? __ldg(reinterpret_cast<const uint32_t*>(row) + c + j) : 0u;
  r[0] = make_uint4(w[0], w[1], w[2], w[3]);
  r[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void values8_bf16(const uint4& r, float (&v)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 f = unpack_bf16x2(w[e]);
    v[2 * e] = f.x;
    v[2 * e + 1] = f.y;
  }
}
__device__ __forceinline__ void values8_f32(const uint4 (&r)[2], float (&v)[8]) {
  const uint32_t w[8] = {r[0].x, r[0].y, r[0].z, r[0].w, r[1].x, r[1].y, r[1].z, r[1].w};
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
}
// The numbers of 8 columns by the exact comparison.  WIDE: x and m have 24 bits, the sides of the comparison 32.
template <bool WIDE>
__device__ __noinline__ uint2 exact8(const float (&x)[8], float m) {
  // a power of two that keeps 254 |x| and 127 / m inside the range of 32 bits
  const float f = m < 1e-18f ? 1.1805916207174113e21f : (m > 1e18f ? 8.470329472543003e-22f : 1.f);
  const float mf = m * f, inv = mf > 0.f ? 127.f / mf : 0.f;
  uint32_t packed[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float ax = fabsf(x[j]) * f, k = floorf(ax * inv);
    bool up;
    if constexpr (WIDE) {
      const double l = 254.0 * double(ax), r = (2.0 * double(k) + 1.0) * double(mf);
      up = l > r || (l == r && (int(k) & 1));
    } else {
      const float l = 254.f * ax, r = (2.f * k + 1.f) * mf;
      up = l > r || (l == r && (int(k) & 1));
    }
    const int q = int(k) + (up ? 1 : 0);
    packed[j >> 2] |= uint32_t((x[j] < 0.f ? -q : q) & 255) << (8 * (j & 3));
  }
  return make_uint2(packed[0], packed[1]);
}

// The numbers nearest to 127 x / m of 8 columns; inv: 127 / m.  odd: rows at an end of the range, by the comparison alone.
// 127 x / m + 1.5 * 2^23 rounds to a whole number k, whose lowest byte is then that of the sum.  inv is rounded, so beside a half k may be a neighbour's;
// what is left, r = 127 x - k m, says so: 127 x and k m have at most 24 bits, and r is exact.  Halves themselves are common (x = m / 2 is one: half a
// percent of a normal row in bf16, three of ten warps' pieces), so they are mended in place.  WIDE: x and m have 24 bits; r in 64 where it is near m / 2.
template <bool WIDE>
__device__ __forceinline__ uint2 numbers8(const float (&x)[8], float m, float inv, bool odd) {
  if (odd) {
    // (copies: what a call may reach has to lie in memory)
    float y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = x[j];
    return exact8<WIDE>(y, m);
  }
  uint32_t t[8];
  float r[8], most = 0.f;
  const float2 inv2 = make_float2(inv, inv), one = make_float2(12582912.f, 12582912.f), less = make_float2(-1.f, -1.f);
  const float2 m2 = make_float2(m, m), top = make_float2(127.f, 127.f);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {        // two columns an instruction
    const float2 v = make_float2(x[j], x[j + 1]), s = ffma2(v, inv2, one), left = ffma2(ffma2(s, less, one), m2, fmul2(v, top));
    t[j] = __float_as_uint(s.x);
    t[j + 1] = __float_as_uint(s.y);
    r[j] = left.x;
    r[j + 1] = left.y;
    most = fmax3(most, fabsf(left.x), fabsf(left.y));
  }
  if (2.f * most >= (WIDE ? m * (1.f - 1.f / 1024) : m)) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bool over;
      if constexpr (WIDE) {
        const double k = double(__uint_as_float(t[j]) - 12582912.f), e = 2.0 * fabs(127.0 * double(x[j]) - k * double(m));
        over = e > double(m) || (e == double(m) && (t[j] & 1u));
      } else {
        const float e = 2.f * fabsf(r[j]);
        over = e > m || (e == m && (t[j] & 1u));
      }
      if (over) t[j] += r[j] > 0.f ? 1u : 0xffffffffu;
    }
  }
  return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410));
}
__device__ __forceinline__ bool odd_row(float m) { return m < 1e-18f || m > 1e18f; }

}  // namespace nkb
