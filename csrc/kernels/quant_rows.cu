// Rows brought into 8-bit whole numbers: q = the whole number nearest to 127 x / m with m = max|x| (ties to the even one), scale = m / 127.
//
// Mathematics.  The quotient is never formed.  With k = floor(127 |x| / m), wrong by one at most in 32 bits, |q| is k + 1 where
// 254 |x| > (2 k + 1) m, or where both are equal and k is odd, and k elsewhere; that also mends a k that is wrong by one.  Both sides have at
// most 24 bits where |x| and m have 16, so the comparison is exact in 32 bits for bf16 rows and for products of two bf16 numbers.  The form that runs
// (numbers8 in quant_rows.cuh) takes the nearest k by a rounding constant and looks at what is left of it, which is exact, too.
//   norm   The norm's factor r = 1 / sqrt(mean(h^2) + eps) is the same for the whole row: 127 (r h w) / max|r h w| = 127 (h w) / max|h w|.  So the numbers
//          come from the exact products h * w, and r enters the scale alone: no rounding of statistics can move a number to its neighbour.  (Rows whose largest
//          product is below 2^-125 have products that 32 bits round, and may have a number's neighbour.)
//   gate   silu(g) * u is not exact in 32 bits.  Columns whose gate is far below zero (kFar), numbers within 2^-12 of a half (one in two thousand; 2^-13 where
//          gate and up are no sums) and candidates for the row's maximum are worked out once more in 64 bits; rows that are small altogether, and the clamped
//          form, whose up + 1 may cancel, in 64 bits as a whole.
// A row with a value that is not finite gets the scale NaN and zeros; a row of zeros the scale 0.
//
// The numbers are thus the same for every order of the sums and every launch shape, and equal those of the CPU.
//
// Layout: a CTA per row, or a cluster where there are few and long gated ones, whose parts meet through distributed shared memory; eight neighbouring
// columns per thread and turn, kept in registers between the pass for the maximum and the one that writes; rows too wide for them are
// computed twice.
//
// us in a graph (bytes at 6544 GB/s): bf16 rows as they are, 64 x 4096 1.7, 16384 x 4096 57 (31), 16384 x 14336 226 (108); fp32 4096 x 4096 14.4 (12.8),
// 16384 x 4096 52 (51); a norm of one, two, four and eight sums of 64 x 4096 2.9, 3.2, 5.3, 7.6, of 128 x 4096 3.3, 4.2, 5.5, 7.9.
#include "api.h"
#include "i8_args.h"
#include "quant_rows.cuh"

namespace nkb {

constexpr float kGateSmall = 1.f / (1 << 20);   // rows with a smaller maximum are gated in 64 bits: their 32-bit errors are not small beside it

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ float fmin3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ double gate64(double g, double u, float limit, float alpha) {
  if (limit > 0.f) {
    g = fmin(g, double(limit));
    u = fmin(fmax(u, -double(limit)), double(limit));
    return (u + 1.0) * g / (1.0 + exp(-double(alpha) * g));
  }
  return g / (1.0 + exp(-g)) * u;
}

template <bool VEC>
__device__ __forceinline__ void load8_bf16(const void* row, int c, int width, float (&v)[8]) {
  values8_bf16(fetch8_bf16<VEC>(row, c, width), v);
}
template <bool VEC>
__device__ __forceinline__ void load8_f32(const float* row, int c, int width, float (&v)[8]) {
  uint4 r[2];
  fetch8_f32<VEC>(row, c, width, r);
  values8_f32(r, v);
}

// What 8 columns are made of, fetched ahead: bf16 and fp32 rows; norm: x, residual and the norm's weights; gate and up (of the first partial sum).
template <int FORM>
struct Raw8 {
  static constexpr int kN = FORM == NKB_ROW_BF16 ? 1 : FORM == NKB_ROW_NORM ? 3 : FORM == NKB_ROW_GATE_F32 ? 4 : 2;
  uint4 r[kN];
};
template <int FORM, bool VEC>
__device__ __forceinline__ void fetch8(const NkbQuantRows& a, long long row, int c, Raw8<FORM>& o, bool weights) {
  const uint4 none = make_uint4(0u, 0u, 0u, 0u);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x) + row * a.x_ld;
  const uint16_t* y = FORM == NKB_ROW_NORM ? reinterpret_cast<const uint16_t*>(a.residual) + row * a.width : x + a.width;       // up, or the stream
  if constexpr (!VEC && (FORM == NKB_ROW_BF16 || FORM == NKB_ROW_NORM || FORM == NKB_ROW_GATE_BF16)) {
    // All loads first.  Pieces are read where they have columns of the same tensor around them: the row's own, or the next and the last one's.
    const int n = a.width - c;
    const bool apart = a.x_ld >= a.width, next = row + 1 < a.rows;
    const bool fx = a.x && n >= 8 && (c >= 8 || (apart && row > 0)) && (n >= 16 || (apart && next));
    const bool fy = FORM == NKB_ROW_NORM ? a.residual && n >= 8 && (c >= 8 || row > 0) && (n >= 16 || next)
                                         : FORM == NKB_ROW_GATE_BF16 && n >= 8 && (n >= 16 || (apart && next));
    const bool fw = FORM == NKB_ROW_NORM && weights && c >= 8 && n >= 16;
    const uint16_t* w = reinterpret_cast<const uint16_t*>(a.w);
    const Pieces px = fetch_pieces(x + c, fx), py = fetch_pieces(y + c, fy), pw = fetch_pieces(w + c, fw);
    o.r[0] = a.x ? from_pieces(px, x + c, fx, n) : none;
    if constexpr (FORM == NKB_ROW_GATE_BF16) o.r[1] = from_pieces(py, y + c, fy, n);
    if constexpr (FORM == NKB_ROW_NORM) {
      o.r[1] = a.residual ? from_pieces(py, y + c, fy, n) : none;
      if (weights) o.r[2] = from_pieces(pw, w + c, fw, n);        // (a thread's columns are the same in every row)
    }
  } else if constexpr (FORM == NKB_ROW_BF16) {
    o.r[0] = fetch8_bf16<VEC>(x, c, a.width);
  } else if constexpr (FORM == NKB_ROW_F32) {
    fetch8_f32<VEC>(reinterpret_cast<const float*>(a.x) + row * a.x_ld, c, a.width, o.r);
  } else if constexpr (FORM == NKB_ROW_NORM) {
    o.r[0] = a.x ? fetch8_bf16<VEC>(x, c, a.width) : none;
    o.r[1] = a.residual ? fetch8_bf16<VEC>(y, c, a.width) : none;
    if (weights) o.r[2] = fetch8_bf16<VEC>(a.w, c, a.width);
  } else if constexpr (FORM == NKB_ROW_GATE_BF16) {
    o.r[0] = fetch8_bf16<VEC>(x, c, a.width);
    o.r[1] = fetch8_bf16<VEC>(y, c, a.width);
  } else {
    const float* p = a.partials + row * a.x_ld;
    uint4 g[2], u[2];
    fetch8_f32<VEC>(p, c, a.width, g);
    fetch8_f32<VEC>(p + a.width, c, a.width, u);
    o.r[0] = g[0];
    o.r[1] = g[1];
    o.r[2] = u[0];
    o.r[3] = u[1];
  }
}

// Off by 2^-23 at most.
__device__ __forceinline__ float reciprocal(float v) {
  float d;
  asm("rcp.approx.f32 %0, %1;" : "=f"(d) : "f"(v));
  return d;
}

// Whether gate and up are what memory has, and no rounded sums or clamped ones.
__device__ __forceinline__ bool gates_given(const NkbQuantRows& a) { return !a.bias && a.limit <= 0.f && a.splits <= 1; }
// Below these arguments of the sigmoid the 32-bit error of a gated value is not what numbers are decided by: the exponential multiplies the rounding of a sum by its
// argument (at -20 the value is off by 28 * 2^-24, a number by 2^-12.2; at -88 by 96 * 2^-24, less than half of the margin for the row's maximum), and beyond -88 it
// leaves the range of 32 bits.  A thread that has such a gate takes its columns in 64 bits.  Sums have some at times: only where gate times up is so large (kLift) that the
// column is more than 2^-28.4, four tenths of a unit of any row that is not in 64 bits as a whole; otherwise its number is zero, however far off the value.
constexpr float kFar = -20.f, kFarGiven = -80.f, kLift = 1.5f;
__device__ __forceinline__ float far_edge(const NkbQuantRows& a) { return gates_given(a) ? kFarGiven : kFar; }

// Gate times up of one column in 64 bits.
template <int FORM>
__device__ __noinline__ double gate_exact(const NkbQuantRows& a, long long row, int c) {
  double g = 0.0, u = 0.0;
  if constexpr (FORM == NKB_ROW_GATE_BF16) {
    const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x) + row * a.x_ld;
    g = __bfloat162float(x[c]);
    u = __bfloat162float(x[a.width + c]);
  } else {
    for (int s = 0; s < a.splits; ++s) {
      const float* p = a.partials + s * a.split_stride + row * a.x_ld;
      g += p[c];
      u += p[a.width + c];
    }
  }
  if (a.bias) {
    const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(a.bias);
    g += __bfloat162float(b[c]);
    u += __bfloat162float(b[a.width + c]);
  }
  return gate64(g, u, a.limit, a.alpha);
}

// s + e += v, nothing lost: the rounding error of every addition of 32 bits is a number of 32 bits, kept in e.
__device__ __forceinline__ void add_pair(float& s, float& e, float v) {
  const float t = s + v, w = t - s;
  e += (s - (t - w)) + (v - w);
  s = t;
}

// Gate and up of 8 columns, each rounded once from its sum (up to the 2^-48 of pairs).
template <int FORM, bool VEC>
__device__ __forceinline__ void load8_gate(const NkbQuantRows& a, long long row, int c, const Raw8<FORM>& raw, float (&g)[8], float (&u)[8]) {
  if constexpr (FORM == NKB_ROW_GATE_BF16) {
    values8_bf16(raw.r[0], g);
    values8_bf16(raw.r[1], u);
    if (!a.bias) return;
  } else {
    const uint4 rg[2] = {raw.r[0], raw.r[1]}, ru[2] = {raw.r[2], raw.r[3]};
    values8_f32(rg, g);
    values8_f32(ru, u);
    if (a.splits == 1 && !a.bias) return;
  }
  float ge[8], ue[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) ge[j] = ue[j] = 0.f;
  if constexpr (FORM == NKB_ROW_GATE_F32) {
    for (int s = 1; s < a.splits; ++s) {
      const float* p = a.partials + s * a.split_stride + row * a.x_ld;
      float v[8], w[8];
      load8_f32<VEC>(p, c, a.width, v);
      load8_f32<VEC>(p + a.width, c, a.width, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        add_pair(g[j], ge[j], v[j]);
        add_pair(u[j], ue[j], w[j]);
      }
    }
  }
  if (a.bias) {
    const __nv_bfloat16* b = reinterpret_cast<const __nv_bfloat16*>(a.bias);
    float v[8];
    load8_bf16<VEC>(b, c, a.width, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) add_pair(g[j], ge[j], v[j]);
    load8_bf16<VEC>(b + a.width, c, a.width, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) add_pair(u[j], ue[j], v[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    // (beside an infinite sum the errors are NaN)
    g[j] = fabsf(g[j]) < INFINITY ? g[j] + ge[j] : g[j];
    u[j] = fabsf(u[j]) < INFINITY ? u[j] + ue[j] : u[j];
  }
}

// 8 columns of a row of `width`, one more to the right in the next lane: rows that do not start on sixteen bytes are stored in pieces that do, which a lane makes
// of its own columns and its neighbour's.  All lanes with columns come here together.
__device__ __forceinline__ void store8_moved(__nv_bfloat16* row, int c, int width, const uint32_t (&h)[4]) {
  const int lane = threadIdx.x & 31, n = min(32, (width + 7) / 8 - (c / 8 - lane));
  const uint32_t mask = n >= 32 ? ~0u : (1u << n) - 1u;
  __nv_bfloat16* o = row + c;
  const uint32_t over = uint32_t(reinterpret_cast<uintptr_t>(o)) & 15u;        // (the same in all lanes)
  int from = 0, to = 8;             // columns that are stored one by one
  if (over == 0) {
    if (c + 8 <= width) {
      *reinterpret_cast<uint4*>(o) = make_uint4(h[0], h[1], h[2], h[3]);
      return;
    }
  } else {
    uint32_t v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = h[j];
      v[4 + j] = __shfl_down_sync(mask, h[j], 1);
    }
    const int skip = int(16u - over) / 2;
    if (lane > 0 && c + 8 <= width) from = skip;
    if (lane + 1 < n && c + 16 <= width) {
      *reinterpret_cast<uint4*>(o + skip) = moved(v, 16u - over);
      to = skip;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j >= from && j < to && c + j < width) reinterpret_cast<uint16_t*>(o)[j] = uint16_t(h[j >> 1] >> (16 * (j & 1)));
}

// What the 8 columns from c on are rounded from.  Norm: stores the residual stream, and adds its squares to ss.  Gate: lowers least to the least argument of the
// sigmoid (of sums: where up lifts it again).
template <int FORM, bool VEC>
__device__ __forceinline__ void load8(const NkbQuantRows& a, long long row, int c, const Raw8<FORM>& raw, float (&v)[8], float& ss, float& least) {
  if constexpr (FORM == NKB_ROW_BF16) {
    values8_bf16(raw.r[0], v);
  } else if constexpr (FORM == NKB_ROW_F32) {
    values8_f32(raw.r, v);
  } else if constexpr (FORM == NKB_ROW_NORM) {
    float r[8], w[8], x[8];
    values8_bf16(raw.r[0], x);
    values8_bf16(raw.r[1], r);
    values8_bf16(raw.r[2], w);
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
      for (int j = 0; j < 8; ++j) x[j] += r[j];
    }
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
      const float2 f = unpack_bf16x2(h[e]);
      x[2 * e] = f.x;
      x[2 * e + 1] = f.y;
    }
    if (a.residual_out) {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.residual_out) + row * a.width;
      if constexpr (!VEC) {
        store8_moved(o, c, a.width, h);
      } else if (c + 8 <= a.width) {
        *reinterpret_cast<uint4*>(o + c) = make_uint4(h[0], h[1], h[2], h[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (c + j < a.width) o[c + j] = __float2bfloat16(x[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      ss = fmaf(x[j], x[j], ss);
      v[j] = x[j] * w[j];
    }
  } else {
    float g[8], u[8], low = 0.f;
    load8_gate<FORM, VEC>(a, row, c, raw, g, u);
    if (a.limit > 0.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g[j] = min_nan(g[j], a.limit);
        u[j] = max_nan(min_nan(u[j], a.limit), -a.limit) + 1.f;
        const float z = a.alpha * g[j];
        low = fminf(low, z);
        v[j] = __fdividef(g[j], 1.f + expf(-z)) * u[j];        // (in this order: the product of both may leave the range)
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; j += 2) low = fmin3(low, g[j], g[j + 1]);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = g[j] * reciprocal(1.f + expf(-g[j])) * u[j];
    }
    if constexpr (FORM == NKB_ROW_GATE_BF16) {
      least = fminf(least, low);
    } else if (low < far_edge(a)) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((a.limit > 0.f ? a.alpha * g[j] : g[j]) < far_edge(a) && fabsf(g[j] * u[j]) > kLift) least = -INFINITY;
    }
    // columns past the width read as zeros
    if (c + 8 > a.width) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j >= a.width) v[j] = 0.f;
    }
  }
}

// What a CTA of a cluster tells the others about its part of the row.
struct RowPart {
  unsigned long long top64;
  uint32_t top;
};

// Registers of a thread: as few as the chunks that it keeps and has on their way leave room for, since more warps hide more of the loads and barriers.
constexpr int row_registers(int form, int it) {
  if (it == 1) return form == NKB_ROW_GATE_F32 ? 128 : 64;
  if (it == 2) return form == NKB_ROW_GATE_F32 ? 128 : 72;
  if (it == 4) return form == NKB_ROW_BF16 ? 64 : 128;
  return 128;
}

// Grid: a CTA per row, or (CLUSTER, gated rows) a cluster along x per row y.  IT: chunks of eight columns that a thread keeps, 0: none, they are read twice.
template <int FORM, bool VEC, int IT, bool CLUSTER>
__global__ void __maxnreg__(row_registers(FORM, IT)) quant_rows_kernel(const NkbQuantRows a) {
  constexpr bool kGate = FORM == NKB_ROW_GATE_BF16 || FORM == NKB_ROW_GATE_F32;
  constexpr bool kKeep = IT > 0;
  static_assert(!CLUSTER || kGate, "only gated rows are divided");
  __shared__ uint32_t s_top[2][16];
  __shared__ float s_ss[2][16];
  __shared__ unsigned long long s_top64[2];
  __shared__ RowPart s_part;
  const int all = (a.width + 7) / 8, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int each = CLUSTER ? (all + gridDim.x - 1) / gridDim.x : all;
  const int chunk0 = CLUSTER ? blockIdx.x * each : 0, chunks = min(all, chunk0 + each);      // [chunk0, chunks)
  if (threadIdx.x == 0) s_top64[0] = 0ull;
  griddep_wait();
  if (!a.late) griddep_launch();
  Raw8<FORM> raw[kKeep ? IT : 1];
  auto fetch = [&](long long row, bool first) {
#pragma unroll
    for (int it = 0; it < (kKeep ? IT : 0); ++it) {
      const int ch = chunk0 + threadIdx.x + it * blockDim.x;
      if (ch < chunks) fetch8<FORM, VEC>(a, row, ch * 8, raw[it], first);
    }
  };
  long long row = CLUSTER ? blockIdx.y : blockIdx.x;
  fetch(row, true);
  // (of the shared words one set is filled while the other may still be read: one barrier a row, two of gated ones)
  for (int turn = 0; row < a.rows; row += CLUSTER ? a.rows : gridDim.x, turn ^= 1) {
  float v[kKeep ? IT : 1][8];
  float big = 0.f, ss = 0.f;              // largest magnitude, NaN if there is one
  float least = 0.f;
  uint32_t big16 = 0;
  if constexpr (kKeep) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int ch = chunk0 + threadIdx.x + it * blockDim.x;
      if (ch >= chunks) continue;
      load8<FORM, VEC>(a, row, ch * 8, raw[it], v[it], ss, least);
      if constexpr (FORM == NKB_ROW_BF16) {
        // magnitudes of bf16 are ordered as their bits are: two to a word
        const uint4 w = raw[it].r[0];
        big16 = __vimax3_s16x2(big16, w.x & 0x7fff7fffu, w.y & 0x7fff7fffu);
        big16 = __vimax3_s16x2(big16, w.z & 0x7fff7fffu, w.w & 0x7fff7fffu);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) big = max_nan(big, fabsf(v[it][j]));
      }
    }
    // the next row's loads are on their way while this one is finished
    if (!CLUSTER && row + gridDim.x < a.rows) fetch(row + gridDim.x, false);
  } else {
    for (int ch = chunk0 + threadIdx.x; ch < chunks; ch += blockDim.x) {
      fetch8<FORM, VEC>(a, row, ch * 8, raw[0], true);
      load8<FORM, VEC>(a, row, ch * 8, raw[0], v[0], ss, least);
#pragma unroll
      for (int j = 0; j < 8; ++j) big = max_nan(big, fabsf(v[0][j]));
    }
  }
  const bool far = kGate && least < far_edge(a);        // this thread's columns are worked out in 64 bits
  // wide rows: the columns once more.  The residual stream may lie in the place of what it was made of.
  NkbQuantRows again_a = a;
  if (!kKeep && FORM == NKB_ROW_NORM && a.residual_out) {
    again_a.x = a.residual_out;
    again_a.x_ld = a.width;
    again_a.residual = again_a.residual_out = nullptr;
    again_a.partials = nullptr;
    again_a.bias = nullptr;
    again_a.splits = 0;
  }
  auto once_more = [&](int ch) {
    float none = 0.f;
    if constexpr (FORM == NKB_ROW_NORM) {
      // (written by this block before its barrier: not through the read-only path)
      const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(again_a.x) + row * again_a.x_ld;
      if (a.residual_out) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (ch * 8 + j < a.width)
            w[j >> 1] |= uint32_t(*reinterpret_cast<const volatile uint16_t*>(h + ch * 8 + j)) << (16 * (j & 1));
        raw[0].r[0] = make_uint4(w[0], w[1], w[2], w[3]);
        raw[0].r[1] = make_uint4(0u, 0u, 0u, 0u);
        raw[0].r[2] = fetch8_bf16<VEC>(a.w, ch * 8, a.width);
        load8<FORM, VEC>(again_a, row, ch * 8, raw[0], v[0], none, none);
        return;
      }
    }
    fetch8<FORM, VEC>(again_a, row, ch * 8, raw[0], true);
    load8<FORM, VEC>(again_a, row, ch * 8, raw[0], v[0], none, none);
  };
  if (kKeep && FORM == NKB_ROW_BF16) big = __uint_as_float(max(big16 << 16, big16 & 0xffff0000u));
  uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big));      // infinities and NaN lie above all numbers
  if constexpr (FORM == NKB_ROW_NORM) ss = warp_sum(ss);
  if (lane == 0) {
    s_top[turn][warp] = top;
    s_ss[turn][warp] = ss;
  }
  __syncthreads();
  if (kGate && threadIdx.x == 0) s_top64[turn ^ 1] = 0ull;
  top = __reduce_max_sync(0xffffffffu, lane < warps ? s_top[turn][lane] : 0u);
  if constexpr (FORM == NKB_ROW_NORM) ss = warp_sum(lane < warps ? s_ss[turn][lane] : 0.f);
  auto small = [&](float m) { return m < kGateSmall || m < a.limit * a.limit / 16.f || m > 1e18f; };
  double m64 = 0.0;
  if constexpr (kGate) {
    // the exact maximum of this CTA's columns, of the values that may be it
    if (top < 0x7f800000u) {
      const float mine = __uint_as_float(top), near = small(mine) ? 0.f : mine * (1.f - 1.f / (1 << 16));
      double best = 0.0;
#pragma unroll
      for (int it = 0; it < (kKeep ? IT : 1 << 30); ++it) {
        const int ch = chunk0 + threadIdx.x + it * blockDim.x;
        if (ch >= chunks) break;
        if constexpr (!kKeep) once_more(ch);
        uint32_t some = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) some |= (far || fabsf(v[kKeep ? it : 0][j]) >= near) && ch * 8 + j < a.width ? 1u << j : 0u;
#pragma unroll 1
        for (; some; some &= some - 1u) best = fmax(best, fabs(gate_exact<FORM>(a, row, ch * 8 + __ffs(some) - 1)));
      }
      if (best > 0.0) atomicMax(&s_top64[turn], (unsigned long long)__double_as_longlong(best));
    }
    __syncthreads();
    m64 = __longlong_as_double((long long)s_top64[turn]);
  }
  if constexpr (CLUSTER) {
    if (threadIdx.x == 0) {
      s_part.top = top;
      s_part.top64 = (unsigned long long)__double_as_longlong(m64);
    }
    cluster_sync_all();
    uint32_t t = 0;
    unsigned long long o = 0;
    if (lane < int(gridDim.x)) {
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(t) : "r"(map_to_cta(&s_part.top, lane)) : "memory");
      asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(o) : "r"(map_to_cta(&s_part.top64, lane)) : "memory");
    }
    top = __reduce_max_sync(0xffffffffu, t);
    m64 = __longlong_as_double((long long)o);
#pragma unroll
    for (int i = 4; i > 0; i >>= 1) m64 = fmax(m64, __shfl_xor_sync(0xffffffffu, m64, i));
    m64 = __shfl_sync(0xffffffffu, m64, 0);
  }
  const bool fine = top < 0x7f800000u;
  const float m = kGate ? float(m64) : __uint_as_float(top);
  const bool in64 = kGate && (small(__uint_as_float(top)) || m > 1e18f);       // the whole row in 64 bits
  if (threadIdx.x == 0 && (!CLUSTER || blockIdx.x == 0)) {
    float scale = kGate ? float(m64 / 127.0) : m / 127.f;
    if constexpr (FORM == NKB_ROW_NORM) scale *= rsqrtf(ss / float(a.width) + a.eps);
    a.scale[row] = fine ? scale : __uint_as_float(0x7fffffffu);
  }
  const float near_half = gates_given(a) ? kNearHalfGatedOnce : kNearHalfGated;
  // Rows whose m or 127 / m is at an end of the range: every number by the comparison, scaled by a power of two.
  const bool odd = odd_row(m);
  const float inv = odd ? 0.f : 127.f / m;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.values) + row * a.q_ld;
  auto finish = [&](float (&x)[8], int ch) {
    uint32_t packed[2] = {0u, 0u};
    if constexpr (!kGate) {
      if (fine) {
        const uint2 q = numbers8<FORM == NKB_ROW_F32>(x, m, inv, odd);
        packed[0] = q.x;
        packed[1] = q.y;
      }
    } else if (fine) {
      uint32_t t[8], again = 0;           // as numbers8, and columns beside a half in 64 bits
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float s = fmaf(x[j], inv, 12582912.f);
        t[j] = __float_as_uint(s);
        again |= fabsf(fmaf(x[j], inv, 12582912.f - s)) > near_half ? 1u << j : 0u;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        packed[i] = __byte_perm(__byte_perm(t[4 * i], t[4 * i + 1], 0x0040), __byte_perm(t[4 * i + 2], t[4 * i + 3], 0x0040), 0x5410);
      if (in64 || far) again = m64 > 0.0 ? 255u : 0u;
#pragma unroll 1
      for (; again; again &= again - 1u) {
        const int j = __ffs(again) - 1;
        if (ch * 8 + j >= a.width) break;
        const double y = gate_exact<FORM>(a, row, ch * 8 + j);
        const uint32_t q = uint32_t(int(rint(127.0 * (y / m64))) & 255), at = 8 * (j & 3);
        if (j < 4) packed[0] = (packed[0] & ~(255u << at)) | q << at;
        else packed[1] = (packed[1] & ~(255u << at)) | q << at;
      }
    }
    *reinterpret_cast<uint2*>(out + ch * 8) = make_uint2(packed[0], packed[1]);
    // (rows end on sixteen bytes)
    if (ch == all - 1 && (all & 1)) *reinterpret_cast<uint2*>(out + ch * 8 + 8) = make_uint2(0u, 0u);
  };
  if constexpr (kKeep) {
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int ch = chunk0 + threadIdx.x + it * blockDim.x;
      if (ch >= chunks) break;
      finish(v[it], ch);
    }
  } else {
    for (int ch = chunk0 + threadIdx.x; ch < chunks; ch += blockDim.x) {
      once_more(ch);
      finish(v[0], ch);
    }
  }
  }
  if constexpr (CLUSTER) cluster_sync_all();        // shared memory stays until every CTA of the cluster has read it
}

// CTAs of a gated row: doubled while a row's part stays 1024 columns and all parts have an SM of their own.  Two partial sums of 2 x 14336, us, with 1, 2 and 4
// CTAs: 64 rows 21.4, 13.0, 15.5; 16 rows 17.1, 10.9, 7.1 (8: 6.5).  Other rows have a few instructions a column, and the cluster's start and barriers cost more than
// its parts gain: 64 behind a norm 5.2, 6.9, 5.9, as they are 3.7, 4.0, 4.1.
static int row_ctas(int rows, int chunks) {
  int c = 1;
  while (c < 8 && chunks > 512 && (long long)rows * c * 2 <= num_sms() && chunks / (2 * c) >= 128) c *= 2;
  return c;
}

// Blocks of that many threads, IT chunks each, that an SM holds at once.
template <int FORM, bool VEC, int IT>
static int resident(unsigned threads) {
  constexpr int kMaxDev = 64;
  static int known[kMaxDev][17] = {};
  int dev = -1, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return 1;
  int& k = known[dev][threads / 32];
  if (k == 0) k = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, quant_rows_kernel<FORM, VEC, IT, false>, int(threads), 0) == cudaSuccess && n > 0 ? n : 1;
  return k;
}

// Rows for several rounds: a block goes from row to row, its next row's loads on their way while it finishes one, as many blocks as the SMs hold.
// Fewer rows than that: -5.
template <int FORM, bool VEC, int IT>
static int launch_many(const NkbQuantRows& a, int chunks) {
  const unsigned threads = unsigned(((chunks + IT - 1) / IT + 31) / 32 * 32);
  if (threads > 512) return -5;
  const int blocks = num_sms() * resident<FORM, VEC, IT>(threads);
  if (a.rows < 2 * blocks) return -5;
  return launch_pdl(quant_rows_kernel<FORM, VEC, IT, false>, dim3(unsigned(blocks)), dim3(threads), 0, reinterpret_cast<cudaStream_t>(a.stream), a);
}

template <int FORM, bool VEC>
static int launch_rows(const NkbQuantRows& a) {
  const int chunks = (a.width + 7) / 8;
  auto warps = [](int n) { return unsigned((n + 31) / 32 * 32); };
  const cudaStream_t stream = reinterpret_cast<cudaStream_t>(a.stream);
  if constexpr (VEC && (FORM == NKB_ROW_GATE_BF16 || FORM == NKB_ROW_GATE_F32)) {
    const int c = row_ctas(a.rows, chunks);
    if (c > 1) {
      const int part = (chunks + c - 1) / c;
      const dim3 grid(unsigned(c), unsigned(a.rows));
      if (part <= 512) return launch_pdl_cluster(quant_rows_kernel<FORM, VEC, 1, true>, grid, dim3(warps(part)), 0, stream, c, a);
      if (part <= 1024) return launch_pdl_cluster(quant_rows_kernel<FORM, VEC, 2, true>, grid, dim3(warps((part + 1) / 2)), 0, stream, c, a);
    }
  }
  // (not normed rows off sixteen bytes, which hold two pieces for each load: 15262 x 2557 184 us so, 114 in a block of its own each; gated 14565 x 930 54, 56)
  if ((VEC || FORM != NKB_ROW_NORM) && chunks > 32 && chunks <= 2048) {
    constexpr int kFew = FORM == NKB_ROW_BF16 || FORM == NKB_ROW_NORM ? 4 : 2;
    int rc = kFew == 2 && chunks <= 1024 ? launch_many<FORM, VEC, kFew>(a, chunks) : launch_many<FORM, VEC, 4>(a, chunks);
    if (rc != -5) return rc;
  }
  const dim3 grid(unsigned(a.rows));
  if (chunks <= 512) return launch_pdl(quant_rows_kernel<FORM, VEC, 1, false>, grid, dim3(warps(chunks)), 0, stream, a);
  if (chunks <= 2048) return launch_pdl(quant_rows_kernel<FORM, VEC, 4, false>, grid, dim3(warps((chunks + 3) / 4)), 0, stream, a);
  return launch_pdl(quant_rows_kernel<FORM, VEC, 0, false>, grid, dim3(512), 0, stream, a);
}

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_quant_rows(const void* packed) {
  const NkbQuantRows& a = *reinterpret_cast<const NkbQuantRows*>(packed);
  if (!status_word() && nkb_init() != 0) return -1;
  if (a.rows <= 0) return 0;
  if (a.width <= 0 || a.splits < 0 || a.q_ld < (a.width + 15) / 16 * 16 || (a.q_ld & 15)) return -2;
  uintptr_t at = reinterpret_cast<uintptr_t>(a.values);
  if (at & 15) return -2;
  for (const void* p : {a.x, (const void*)a.partials, a.bias, a.residual, a.w, (const void*)a.residual_out})
    at |= reinterpret_cast<uintptr_t>(p);
  const bool gate = a.form == NKB_ROW_GATE_BF16 || a.form == NKB_ROW_GATE_F32;
  const bool rows_of_width = a.form == NKB_ROW_NORM || gate;
  // (of gated fp32 rows the up half starts on sixteen bytes with every fourth column already, a bias's with every eighth)
  const int whole = a.form == NKB_ROW_GATE_F32 && !a.bias ? 3 : 7;
  const bool vec = (at & 15) == 0 && (a.x_ld & whole) == 0 && (a.split_stride & 3) == 0 && (!rows_of_width || (a.width & whole) == 0);
  switch (a.form) {
    case NKB_ROW_BF16: return vec ? launch_rows<NKB_ROW_BF16, true>(a) : launch_rows<NKB_ROW_BF16, false>(a);
    case NKB_ROW_F32: return vec ? launch_rows<NKB_ROW_F32, true>(a) : launch_rows<NKB_ROW_F32, false>(a);
    case NKB_ROW_NORM: return vec ? launch_rows<NKB_ROW_NORM, true>(a) : launch_rows<NKB_ROW_NORM, false>(a);
    case NKB_ROW_GATE_BF16: return vec ? launch_rows<NKB_ROW_GATE_BF16, true>(a) : launch_rows<NKB_ROW_GATE_BF16, false>(a);
    case NKB_ROW_GATE_F32: return vec ? launch_rows<NKB_ROW_GATE_F32, true>(a) : launch_rows<NKB_ROW_GATE_F32, false>(a);
  }
  return -2;
}
