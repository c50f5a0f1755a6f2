// Rows brought into 8-bit whole numbers: q = the whole number nearest to 127 x / m with m = max|x| (ties to the even one), scale = m / 127.
//
// Mathematics.  The quotient is never formed.  With k = floor(127 |x| / m), wrong by one at most in 32 bits, |q| is k + 1 where
// 254 |x| > (2 k + 1) m, or where both are equal and k is odd, and k elsewhere; that also mends a k that is wrong by one.  Both sides have at
// most 24 bits where |x| and m have 16, so the comparison is exact in 32 bits for bf16 rows and for products of two bf16 numbers.
//   norm   The norm's factor r = 1 / sqrt(mean(h^2) + eps) is the same for the whole row: 127 (r h w) / max|r h w| = 127 (h w) / max|h w|.  So the numbers
//          come from the exact products h * w, and r enters the scale alone: no rounding of statistics can move a number to its neighbour.
//   gate   silu(g) * u is not exact in 32 bits.  Numbers within 2^-11 of a half (one in a thousand) and candidates for the row's maximum are worked out
//          once more in 64 bits; rows that are small altogether, and the clamped form, whose up + 1 may cancel, in 64 bits as a whole.
// A row with a value that is not finite gets the scale NaN and zeros; a row of zeros the scale 0.
//
// The numbers are thus the same for every order of the sums and every launch shape, and equal those of the CPU.
//
// Layout: a block per row, eight neighbouring columns per thread and turn, kept in registers between the pass for the maximum and the one that
// writes; rows too wide for the registers are computed twice.
#include "api.h"
#include "common.cuh"
#include "i8_args.h"

namespace nkb {

constexpr float kHalfNear = 1.f / 2048;      // of m: distance from a half below which a gated value is worked out in 64 bits
constexpr float kGateSmall = 1.f / (1 << 20);   // rows with a smaller maximum are gated in 64 bits: their 32-bit errors are not small beside it

__device__ __forceinline__ double gate64(double g, double u, float limit, float alpha) {
  if (limit > 0.f) {
    g = fmin(g, double(limit));
    u = fmin(fmax(u, -double(limit)), double(limit));
    return (u + 1.0) * g / (1.0 + exp(-double(alpha) * g));
  }
  return g / (1.0 + exp(-g)) * u;
}

// 8 columns from `c` on of a bf16 row; columns past the width read as zeros.  VEC: rows start on 16 bytes.
template <bool VEC>
__device__ __forceinline__ void load8_bf16(const __nv_bfloat16* row, int c, int width, float (&v)[8]) {
  if (VEC && c + 8 <= width) {
    const uint4 r = *reinterpret_cast<const uint4*>(row + c);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(w[e]);
      v[2 * e] = f.x;
      v[2 * e + 1] = f.y;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < width ? __bfloat162float(row[c + j]) : 0.f;
}
template <bool VEC>
__device__ __forceinline__ void load8_f32(const float* row, int c, int width, float (&v)[8]) {
  if (VEC && c + 8 <= width) {
    const float4 a = reinterpret_cast<const float4*>(row + c)[0], b = reinterpret_cast<const float4*>(row + c)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c + j < width ? row[c + j] : 0.f;
}

// Gate and up of 8 columns, summed in 64 bits.
template <int FORM, bool VEC>
__device__ __forceinline__ void load8_gate(const NkbQuantRows& a, long long row, int c, double (&g)[8], double (&u)[8]) {
  float v[8];
  if constexpr (FORM == NKB_ROW_GATE_BF16) {
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + row * a.x_ld;
    load8_bf16<VEC>(x, c, a.width, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = v[j];
    load8_bf16<VEC>(x + a.width, c, a.width, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = v[j];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = u[j] = 0.0;
    for (int s = 0; s < a.splits; ++s) {
      const float* p = a.partials + s * a.split_stride + row * a.x_ld;
      load8_f32<VEC>(p, c, a.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) g[j] += v[j];
      load8_f32<VEC>(p + a.width, c, a.width, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] += v[j];
    }
  }
  if (a.bias) {
    const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(a.bias);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (c + j >= a.width) continue;
      g[j] += __bfloat162float(b[c + j]);
      u[j] += __bfloat162float(b[a.width + c + j]);
    }
  }
}

// What the 8 columns from c on are rounded from.  Norm: stores the residual stream, and adds its squares to ss.
template <int FORM, bool VEC>
__device__ __forceinline__ void load8(const NkbQuantRows& a, long long row, int c, float (&v)[8], float& ss, bool store) {
  if constexpr (FORM == NKB_ROW_BF16) {
    load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(a.x) + row * a.x_ld, c, a.width, v);
  } else if constexpr (FORM == NKB_ROW_F32) {
    load8_f32<VEC>(reinterpret_cast<const float*>(a.x) + row * a.x_ld, c, a.width, v);
  } else if constexpr (FORM == NKB_ROW_NORM) {
    float r[8], w[8], x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = x[j] = 0.f;
    if (a.residual) load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(a.residual) + row * a.width, c, a.width, r);
    if (a.x) load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(a.x) + row * a.x_ld, c, a.width, x);
    load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(a.w), c, a.width, w);
    if (a.partials || a.bias) {
      // more than two addends: in 64 bits, so that the rounding to bf16 is the one of the sum
      double h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = double(x[j]) + double(r[j]);
      for (int s = 0; s < a.splits; ++s) {
        float p[8];
        load8_f32<VEC>(a.partials + s * a.split_stride + row * a.x_ld, c, a.width, p);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += p[j];
      }
      if (a.bias) {
        float b[8];
        load8_bf16<VEC>(reinterpret_cast<const __nv_bfloat16*>(a.bias), c, a.width, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] += b[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __bfloat162float(__double2bfloat16(h[j]));
    } else {
      // the sum of two bf16 numbers in 32 bits is never a tie of bf16 that the sum itself is not
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = __bfloat162float(__float2bfloat16(x[j] + r[j]));
    }
    if (store && a.residual_out) {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.residual_out) + row * a.width + c;
      if (VEC && c + 8 <= a.width) {
        *reinterpret_cast<uint4*>(o) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                                                  pack_bf16x2(x[6], x[7]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < a.width) o[j] = __float2bfloat16(x[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(x[j], x[j], ss);
      v[j] = x[j] * w[j];
    }
  } else {
    double g[8], u[8];
    load8_gate<FORM, VEC>(a, row, c, g, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (a.limit > 0.f) {
        v[j] = float(gate64(g[j], u[j], a.limit, a.alpha));
      } else {
        const float gf = float(g[j]);
        v[j] = gf / (1.f + expf(-gf)) * float(u[j]);
      }
    }
  }
}

template <int FORM, bool VEC, int IT>
__global__ void __launch_bounds__(1024) quant_rows_kernel(const NkbQuantRows a) {
  constexpr bool kGate = FORM == NKB_ROW_GATE_BF16 || FORM == NKB_ROW_GATE_F32;
  constexpr bool kKeep = IT > 0;
  __shared__ uint32_t s_top[32];
  __shared__ float s_ss[32];
  __shared__ unsigned long long s_top64;
  const long long row = blockIdx.x;
  const int chunks = (a.width + 7) / 8, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) s_top64 = 0ull;
  griddep_wait();
  griddep_launch();
  float v[kKeep ? IT : 1][8];
  uint32_t top = 0;                       // bits of the largest magnitude: infinities and NaN lie above all numbers
  float ss = 0.f;
  if constexpr (kKeep) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int ch = threadIdx.x + it * blockDim.x;
      if (ch >= chunks) break;
      load8<FORM, VEC>(a, row, ch * 8, v[it], ss, true);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[it][j]) & 0x7fffffffu);
    }
  } else {
    for (int ch = threadIdx.x; ch < chunks; ch += blockDim.x) {
      load8<FORM, VEC>(a, row, ch * 8, v[0], ss, true);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[0][j]) & 0x7fffffffu);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (FORM == NKB_ROW_NORM) ss = warp_sum(ss);
  if (lane == 0) {
    s_top[warp] = top;
    s_ss[warp] = ss;
  }
  __syncthreads();
  const int warps = blockDim.x >> 5;
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[lane] : 0u);
  float m = __uint_as_float(top);
  bool in64 = false;                      // gate: the whole row in 64 bits
  double m64 = m;
  if constexpr (kGate) {
    in64 = a.limit > 0.f || m < kGateSmall;
    if (top < 0x7f800000u) {
      // the exact maximum, of the values that may be it
      const float near = in64 ? 0.f : m * (1.f - 1.f / (1 << 18));
      double best = 0.0;
      for (int it = 0;; ++it) {
        const int ch = threadIdx.x + it * blockDim.x;
        if (ch >= chunks || (kKeep && it >= IT)) break;
        float mine = 0.f;
        if constexpr (kKeep) {
#pragma unroll
          for (int i = 0; i < IT; ++i)
            if (i == it)
#pragma unroll
              for (int j = 0; j < 8; ++j) mine = fmaxf(mine, fabsf(v[i][j]));
        } else {
          float none = 0.f;
          load8<FORM, VEC>(a, row, ch * 8, v[0], none, false);
#pragma unroll
          for (int j = 0; j < 8; ++j) mine = fmaxf(mine, fabsf(v[0][j]));
        }
        if (mine >= near) {
          double g[8], u[8];
          load8_gate<FORM, VEC>(a, row, ch * 8, g, u);
#pragma unroll
          for (int j = 0; j < 8; ++j) best = fmax(best, fabs(gate64(g[j], u[j], a.limit, a.alpha)));
        }
      }
      if (best > 0.0) atomicMax(&s_top64, (unsigned long long)__double_as_longlong(best));
      __syncthreads();
      m64 = __longlong_as_double((long long)s_top64);
      m = float(m64);
    }
  }
  const bool fine = top < 0x7f800000u;
  if (threadIdx.x == 0) {
    float scale = kGate ? float(m64 / 127.0) : m / 127.f;
    if constexpr (FORM == NKB_ROW_NORM) {
      float total = 0.f;
      for (int i = 0; i < warps; ++i) total += s_ss[i];
      scale *= rsqrtf(total / float(a.width) + a.eps);
    }
    a.scale[row] = fine ? scale : __uint_as_float(0x7fffffffu);
  }
  // a power of two that keeps 254 |x| and 127 / m inside the range of 32 bits
  const float f = m < 1e-18f ? 1.1805916207174113e21f : (m > 1e18f ? 8.470329472543003e-22f : 1.f);
  const float mf = m * f, inv = mf > 0.f ? 127.f / mf : 0.f;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.values) + row * a.q_ld;
  auto finish = [&](float (&x)[8], int ch) {
    uint32_t packed[2] = {0u, 0u};
    uint32_t again = 0;                   // columns to be worked out in 64 bits
    if (fine && !in64) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float ax = fabsf(x[j]) * f;
        float k = floorf(ax * inv);
        const float l = 254.f * ax, r = (2.f * k + 1.f) * mf;
        bool up = l > r || (l == r && (int(k) & 1));
        if constexpr (FORM == NKB_ROW_F32) {
          if (fabsf(l - r) <= kHalfNear * mf) {      // 24-bit numbers: the sides have 32 bits
            const double l64 = 254.0 * double(ax), r64 = (2.0 * double(k) + 1.0) * double(mf);
            up = l64 > r64 || (l64 == r64 && (int(k) & 1));
          }
        }
        if constexpr (kGate) {
          if (fabsf(l - r) <= kHalfNear * mf) again |= 1u << j;
        }
        const int q = int(k) + (up ? 1 : 0);
        packed[j >> 2] |= uint32_t((x[j] < 0.f ? -q : q) & 255) << (8 * (j & 3));
      }
    }
    if constexpr (kGate) {
      if (fine && in64) again = m64 > 0.0 ? 255u : 0u;
      if (again) {
        double g[8], u[8];
        load8_gate<FORM, VEC>(a, row, ch * 8, g, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (!((again >> j) & 1)) continue;
          const double y = gate64(g[j], u[j], a.limit, a.alpha);
          const int q = int(rint(127.0 * (y / m64)));
          packed[j >> 2] = (packed[j >> 2] & ~(255u << (8 * (j & 3)))) | uint32_t(q & 255) << (8 * (j & 3));
        }
      }
    }
    *reinterpret_cast<uint2*>(out + ch * 8) = make_uint2(packed[0], packed[1]);
    // (rows end on sixteen bytes)
    if (ch == chunks - 1 && (chunks & 1)) *reinterpret_cast<uint2*>(out + ch * 8 + 8) = make_uint2(0u, 0u);
  };
  if constexpr (kKeep) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int ch = threadIdx.x + it * blockDim.x;
      if (ch >= chunks) break;
      finish(v[it], ch);
    }
  } else {
    for (int ch = threadIdx.x; ch < chunks; ch += blockDim.x) {
      float none = 0.f;
      load8<FORM, VEC>(a, row, ch * 8, v[0], none, false);
      finish(v[0], ch);
    }
  }
}

template <int FORM, bool VEC>
static int launch_rows(const NkbQuantRows& a) {
  const int chunks = (a.width + 7) / 8;
  auto go = [&](auto kernel, int threads) {
    return launch_pdl(kernel, dim3(unsigned(a.rows)), dim3(unsigned(threads)), 0, reinterpret_cast<cudaStream_t>(a.stream), a);
  };
  auto warps = [](int n) { return (n + 31) / 32 * 32; };
  if (chunks <= 1024) return go(quant_rows_kernel<FORM, VEC, 1>, warps(chunks));
  if (chunks <= 2048) return go(quant_rows_kernel<FORM, VEC, 2>, warps((chunks + 1) / 2));
  return go(quant_rows_kernel<FORM, VEC, 0>, 1024);
}

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_quant_rows(const void* packed) {
  const NkbQuantRows& a = *reinterpret_cast<const NkbQuantRows*>(packed);
  if (a.rows <= 0) return 0;
  if (a.width <= 0 || a.splits < 0 || a.q_ld < (a.width + 15) / 16 * 16 || (a.q_ld & 15)) return -2;
  uintptr_t at = reinterpret_cast<uintptr_t>(a.values);
  if (at & 15) return -2;
  for (const void* p : {a.x, (const void*)a.partials, a.bias, a.residual, a.w, (const void*)a.residual_out})
    at |= reinterpret_cast<uintptr_t>(p);
  const bool gate = a.form == NKB_ROW_GATE_BF16 || a.form == NKB_ROW_GATE_F32;
  const bool rows_of_width = a.form == NKB_ROW_NORM || gate;
  const bool vec = (at & 15) == 0 && (a.x_ld & 7) == 0 && (a.split_stride & 3) == 0 && (!rows_of_width || (a.width & 7) == 0);
  switch (a.form) {
    case NKB_ROW_BF16: return vec ? launch_rows<NKB_ROW_BF16, true>(a) : launch_rows<NKB_ROW_BF16, false>(a);
    case NKB_ROW_F32: return vec ? launch_rows<NKB_ROW_F32, true>(a) : launch_rows<NKB_ROW_F32, false>(a);
    case NKB_ROW_NORM: return vec ? launch_rows<NKB_ROW_NORM, true>(a) : launch_rows<NKB_ROW_NORM, false>(a);
    case NKB_ROW_GATE_BF16: return vec ? launch_rows<NKB_ROW_GATE_BF16, true>(a) : launch_rows<NKB_ROW_GATE_BF16, false>(a);
    case NKB_ROW_GATE_F32: return vec ? launch_rows<NKB_ROW_GATE_F32, true>(a) : launch_rows<NKB_ROW_GATE_F32, false>(a);
  }
  return -2;
}
