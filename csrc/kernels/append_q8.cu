// Queries, keys and values of new tokens from the fused QKV projection: split-K partials summed, bias, per-head RMSNorm, rotate-halves
// RoPE; queries leave as bf16, keys and values go to their places in 8-bit pages (kv_quant.cuh).  The counterpart of
// rope_kv_append (elementwise.cu) for a quantised cache.
//
// Keys and values are computed in 64 bits, so that their one rounding to e4m3 does not depend on the order of operations.
//
// Measured with 32 heads of 128 on 8: one token from 8 partial sums 3.1 us (latency), 16384 tokens from bf16 77.3 us (58.1 at the copy
// bandwidth of 6.56 TB/s; 80 for bf16 pages), 390 of 32 heads on 4 with norms 5.4 us (1.2; a chain of latencies, two square roots in it).
#include "api.h"
#include "kv_quant.cuh"

namespace nkb {

struct AppendQ8Params {
  const __nv_bfloat16* qkv;
  const float* partials;
  int splits;
  long long split_stride;
  const __nv_bfloat16* bias;
  const int *positions, *slots;
  const float* cos_sin;
  const __nv_bfloat16 *q_norm_w, *k_norm_w;
  double eps;
  __nv_bfloat16* q_out;
  uint8_t *k_values, *k_scales, *v_values, *v_scales;
  int tokens, nq, nkv, max_pos;
  long long slots_end;              // slots of the pool
};

// One warp per (token, head); a lane has PER elements of the head's first half and those that turn with them.
template <int D>
__global__ void __launch_bounds__(256) append_q8_kernel(const AppendQ8Params p) {
  constexpr int PER = D / 64;
  const int heads = p.nq + 2 * p.nkv;
  const long long gw = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  if (gw >= (long long)p.tokens * heads) return;
  const int t = int(gw / heads), h = int(gw % heads);
  const bool is_q = h < p.nq, is_k = !is_q && h < p.nq + p.nkv;
  const long long base = (long long)t * heads * D + (long long)h * D;
  double lo[PER], hi[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane * PER + j;
    double a = 0., b = 0.;
    if (p.partials) {
      for (int s = 0; s < p.splits; ++s) {
        a += double(p.partials[s * p.split_stride + base + i]);
        b += double(p.partials[s * p.split_stride + base + D / 2 + i]);
      }
    } else {
      a = double(__bfloat162float(p.qkv[base + i]));
      b = double(__bfloat162float(p.qkv[base + D / 2 + i]));
    }
    if (p.bias) {
      a += double(__bfloat162float(p.bias[h * D + i]));
      b += double(__bfloat162float(p.bias[h * D + D / 2 + i]));
    }
    lo[j] = a;
    hi[j] = b;
  }
  if (is_q || is_k) {
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : p.k_norm_w;
    if (nw) {
      double ss = 0.;
#pragma unroll
      for (int j = 0; j < PER; ++j) ss += lo[j] * lo[j] + hi[j] * hi[j];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const double inv = 1. / sqrt(ss / double(D) + p.eps);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = lane * PER + j;
        lo[j] = lo[j] * inv * double(__bfloat162float(nw[i]));
        hi[j] = hi[j] * inv * double(__bfloat162float(nw[D / 2 + i]));
      }
    }
    if (p.cos_sin) {
      const int pos = min(max(p.positions[t], 0), p.max_pos - 1);
      const float* cs = p.cos_sin + (long long)pos * D;  // [cos(d/2) | sin(d/2)]
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int i = lane * PER + j;
        const double c = cs[i], s = cs[D / 2 + i], a = lo[j], b = hi[j];
        lo[j] = a * c - b * s;
        hi[j] = b * c + a * s;
      }
    }
  }
  float x[2 * PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    x[j] = round_to_odd(lo[j]);
    x[PER + j] = round_to_odd(hi[j]);
  }
  if (is_q) {
    __nv_bfloat16* dst = p.q_out + ((long long)t * p.nq + h) * D;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      dst[lane * PER + j] = __float2bfloat16(x[j]);
      dst[D / 2 + lane * PER + j] = __float2bfloat16(x[PER + j]);
    }
    return;
  }
  const long long slot = p.slots ? p.slots[t] : -1;
  if (slot < 0 || slot >= p.slots_end) return;
  float amax = 0.f;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 2 * PER; ++j) {
    fine = fine && isfinite(x[j]);
    amax = fmaxf(amax, fabsf(x[j]));
  }
  fine = __all_sync(0xffffffffu, fine);
  amax = warp_max(amax);
  const int e = q8_log2_scale(amax);
  const float inv = fine ? exp2_int(-e) : 0.f;
  const long long row = (slot / kQ8Page * p.nkv + (is_k ? h - p.nq : h - p.nq - p.nkv)) * kQ8Page + slot % kQ8Page;
  uint8_t* dst = (is_k ? p.k_values : p.v_values) + row * D;
#pragma unroll
  for (int j = 0; j < 2 * PER; ++j) x[j] = fine ? x[j] * inv : 0.f;
  if constexpr (PER == 2) {
    *reinterpret_cast<uint16_t*>(dst + lane * 2) = pack_e4m3x2(x[0], x[1]);
    *reinterpret_cast<uint16_t*>(dst + D / 2 + lane * 2) = pack_e4m3x2(x[2], x[3]);
  } else {
    const uint16_t v = pack_e4m3x2(x[0], x[1]);
    dst[lane] = uint8_t(v);
    dst[D / 2 + lane] = uint8_t(v >> 8);
  }
  if (lane == 0) (is_k ? p.k_scales : p.v_scales)[row] = uint8_t(fine ? 127 + e : 255);
}

// a * c - d * s from 32-bit numbers, rounded to odd like round_to_odd of the same in 64 bits: products and their difference with what each
// rounding leaves (a product's rest is one multiply-add; the difference's by Knuth's two-sum).  What the products leave may be more than a
// step of their difference, so it is added before the rounding to odd (Dekker's sum, whose rest is wrong only where the products cancel, and
// the result becomes zero beside the head's other half).  Finite where the inputs are.
__device__ __forceinline__ float turn_to_odd(float a, float c, float d, float s) {
  constexpr float kMost = 3.402823466e38f;
  // (intrinsics: the compiler must not merge these)
  const float p = __fmul_rn(a, c), pe = __fmaf_rn(a, c, -p), q = __fmul_rn(d, s), qe = __fmaf_rn(d, s, -q);
  const float x = __fsub_rn(p, q), v = __fsub_rn(x, p);
  const float rest = __fadd_rn(__fsub_rn(__fsub_rn(p, __fsub_rn(x, v)), __fadd_rn(q, v)), __fsub_rn(pe, qe));
  const float y = __fadd_rn(x, rest), least = __fsub_rn(rest, __fsub_rn(y, x));
  const float top = fminf(fmaxf(fabsf(x) <= kMost ? y : x, -kMost), kMost);
  int bits = __float_as_int(top);
  if (least != 0.f && top != 0.f) {
    if ((least < 0.f) != (top < 0.f)) --bits;      // the sum lies nearer zero: the number before
    bits |= 1;
  }
  return __int_as_float(bits);
}

// The same in pieces of sixteen bytes: D / 16 lanes share a head, each with eight elements of its first half and the eight that turn with
// them.  A warp takes 512 / D heads of a token at a time, `run` times, the next ones' inputs on their way.  Every pointer on 16 bytes,
// split_stride a multiple of four.
//
// Bound by memory from some thousand tokens on, and next by what goes through L1: cos and sin are twice the bytes of a head's input, so a run
// loads them once.  Then come instructions: 64-bit arithmetic and conversions run at a fraction of the 32-bit
// rate, so keys of a bf16 projection without norm and bias turn in pairs of 32-bit numbers, and such values need no sum at all.
template <int D, bool PARTIALS>
__global__ void __launch_bounds__(256, PARTIALS ? 2 : 3) append8_q8_kernel(const AppendQ8Params p, int run) {
  constexpr int L = D / 16, kHeads = 32 / L;
  const int heads = p.nq + 2 * p.nkv, runs = (heads + kHeads * run - 1) / (kHeads * run);
  const int i0 = (threadIdx.x % L) * 8;
  const uint32_t mine = ((1u << L) - 1u) << ((threadIdx.x & 31) / L * L);      // the lanes of this head
  griddep_wait();
  griddep_launch();
  const uint32_t unit = blockIdx.x * 8 + threadIdx.x / 32;
  const int t = int(unit / uint32_t(runs)), first = int(unit - uint32_t(t) * runs) * run * kHeads, h1 = min(first + run * kHeads, heads);
  const int h0 = first + (threadIdx.x & 31) / L;
  if (t >= p.tokens) return;
  uint4 raw[2], raw_n[2];
  auto load = [&](int h, uint4 (&r)[2]) {
    if (!PARTIALS && h < h1) {
      const __nv_bfloat16* src = p.qkv + ((long long)t * heads + h) * D + i0;
      r[0] = *reinterpret_cast<const uint4*>(src);
      r[1] = *reinterpret_cast<const uint4*>(src + D / 2);
    }
  };
  load(h0, raw_n);
  const long long slot = p.slots && h1 > p.nq ? p.slots[t] : -1;
  float c[8], sn[8];
  if (p.cos_sin && h0 < p.nq + p.nkv) {
    const float* cs = p.cos_sin + (long long)min(max(p.positions[t], 0), p.max_pos - 1) * D + i0;  // [cos(d/2) | sin(d/2)]
#pragma unroll
    for (int j = 0; j < 8; j += 4) {
      *reinterpret_cast<float4*>(c + j) = *reinterpret_cast<const float4*>(cs + j);
      *reinterpret_cast<float4*>(sn + j) = *reinterpret_cast<const float4*>(cs + D / 2 + j);
    }
  }
  auto floats = [](const uint4& r, float* o) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(w[e]);
      o[2 * e] = f.x;
      o[2 * e + 1] = f.y;
    }
  };
  auto get16 = [&](const __nv_bfloat16* src, float* o) {         // this lane's elements of a head's row
    floats(*reinterpret_cast<const uint4*>(src + i0), o);
    floats(*reinterpret_cast<const uint4*>(src + D / 2 + i0), o + 8);
  };
  const auto at = [&](int j) { return i0 + (j < 8 ? j : D / 2 + j - 8); };
#pragma unroll 1
  for (int h = h0; h < h1; h += kHeads) {
    raw[0] = raw_n[0];
    raw[1] = raw_n[1];
    load(h + kHeads, raw_n);
    const long long row0 = ((long long)t * heads + h) * D + i0;
    const bool is_q = h < p.nq, is_k = !is_q && h < p.nq + p.nkv, turn = p.cos_sin && h < p.nq + p.nkv;
    float x[16];                         // queries, and what goes to the pages; at first bf16 inputs, exactly
    double y[PARTIALS ? 16 : 1];         // sums of partials
    if constexpr (PARTIALS) {
#pragma unroll
      for (int j = 0; j < 16; ++j) y[j] = 0.;
#pragma unroll 2
      for (int s = 0; s < p.splits; ++s) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 v = *reinterpret_cast<const float4*>(p.partials + s * p.split_stride + row0 + (j < 8 ? j : D / 2 + j - 8));
          y[j] += double(v.x);
          y[j + 1] += double(v.y);
          y[j + 2] += double(v.z);
          y[j + 3] += double(v.w);
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = float(y[j]);
    } else {
      floats(raw[0], x);
      floats(raw[1], x + 8);
    }
    // the input with its bias in 64 bits
    const auto in64 = [&](int j) {
      double v;
      if constexpr (PARTIALS) v = y[j];
      else v = double(x[j]);
      return p.bias ? v + double(__bfloat162float(p.bias[h * D + at(j)])) : v;
    };
    const __nv_bfloat16* nw = is_q ? p.q_norm_w : (is_k ? p.k_norm_w : nullptr);
    double inv = 1.;
    if (is_q) {
      if (p.bias) {
        float b[16];
        get16(p.bias + h * D, b);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] += b[j];
      }
      if (nw) {
        float ss = 0.f, w[16];
        get16(nw, w);
#pragma unroll
        for (int j = 0; j < 16; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int m = L / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(mine, ss, m);
        float f = 1.f / sqrtf(ss / float(D) + float(p.eps));
        if (!(ss > 1e-30f && ss <= 1e38f)) {       // squares beyond 32 bits (a head's lanes agree)
          double wide = 0.;
#pragma unroll
          for (int j = 0; j < 16; ++j) wide += double(x[j]) * double(x[j]);
#pragma unroll
          for (int m = L / 2; m > 0; m >>= 1) wide += __shfl_xor_sync(mine, wide, m);
          f = float(1. / sqrt(wide / double(D) + p.eps));
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = x[j] * f * w[j];
      }
      if (turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = x[j], d = x[8 + j];
          x[j] = a * c[j] - d * sn[j];
          x[8 + j] = d * c[j] + a * sn[j];
        }
      }
      __nv_bfloat16* dst = p.q_out + ((long long)t * p.nq + h) * D + i0;
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
      *reinterpret_cast<uint4*>(dst + D / 2) =
          make_uint4(pack_bf16x2(x[8], x[9]), pack_bf16x2(x[10], x[11]), pack_bf16x2(x[12], x[13]), pack_bf16x2(x[14], x[15]));
      continue;
    }
    bool fine = true;
    if (PARTIALS || p.bias || nw) {
      if (nw) {
        double ss = 0.;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const double v = in64(j);
          ss += v * v;
        }
#pragma unroll
        for (int m = L / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(mine, ss, m);
        inv = 1. / sqrt(ss / double(D) + p.eps);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        double a = in64(j), d = in64(8 + j);
        if (nw) {
          a = a * inv * double(__bfloat162float(nw[at(j)]));
          d = d * inv * double(__bfloat162float(nw[at(8 + j)]));
        }
        if (is_k && turn) {
          const double co = c[j], si = sn[j], a0 = a;
          a = a0 * co - d * si;
          d = d * co + a0 * si;
        }
        x[j] = round_to_odd(a);
        x[8 + j] = round_to_odd(d);
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) fine = fine && isfinite(x[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) fine = fine && isfinite(x[j]);
      if (is_k && turn) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = x[j], d = x[8 + j];
          fine = fine && isfinite(c[j]) && isfinite(sn[j]);
          x[j] = turn_to_odd(a, c[j], d, sn[j]);
          x[8 + j] = turn_to_odd(d, c[j], -a, sn[j]);
        }
      }
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
    for (int m = L / 2; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mine, amax, m));
    fine = __all_sync(mine, fine);
    if (slot < 0 || slot >= p.slots_end) continue;
    const int e = q8_log2_scale(amax);
    const float down = exp2_int(-e);
    const long long row = (slot / kQ8Page * p.nkv + (is_k ? h - p.nq : h - p.nq - p.nkv)) * kQ8Page + slot % kQ8Page;
    uint8_t* dst = (is_k ? p.k_values : p.v_values) + row * D + i0;
    uint32_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      v[j] = fine ? pack_e4m3x2(x[4 * j] * down, x[4 * j + 1] * down) | uint32_t(pack_e4m3x2(x[4 * j + 2] * down, x[4 * j + 3] * down)) << 16 : 0u;
    *reinterpret_cast<uint2*>(dst) = make_uint2(v[0], v[1]);
    *reinterpret_cast<uint2*>(dst + D / 2) = make_uint2(v[2], v[3]);
    if (i0 == 0) (is_k ? p.k_scales : p.v_scales)[row] = uint8_t(fine ? 127 + e : 255);
  }
}

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_q8_append(const NkbQ8Append* arg) {
  const NkbQ8Append& g = *arg;
  const int tokens = g.tokens, nq = g.nq, nkv = g.nkv, head_dim = g.head_dim;
  const void* qkv_bf16 = g.qkv;
  const float* qkv_partials = g.partials;
  if (tokens <= 0) return 0;
  if (nq < 1 || nkv < 1 || (!qkv_bf16 && (!qkv_partials || g.splits < 1)) || (g.cos_sin && (!g.positions || g.max_pos < 1))) return -2;
  if (!status_word() && nkb_init() != 0) return -1;
  AppendQ8Params p{};
  p.qkv = (const __nv_bfloat16*)qkv_bf16;
  p.partials = qkv_partials;
  p.splits = g.splits;
  p.split_stride = g.split_stride;
  p.bias = (const __nv_bfloat16*)g.bias;
  p.positions = g.positions;
  p.slots = g.slots;
  p.cos_sin = g.cos_sin;
  p.q_norm_w = (const __nv_bfloat16*)g.q_norm_w;
  p.k_norm_w = (const __nv_bfloat16*)g.k_norm_w;
  p.eps = g.eps;
  p.q_out = (__nv_bfloat16*)g.q_out;
  p.k_values = (uint8_t*)g.k_values;
  p.k_scales = (uint8_t*)g.k_scales;
  p.v_values = (uint8_t*)g.v_values;
  p.v_scales = (uint8_t*)g.v_scales;
  p.tokens = tokens; p.nq = nq; p.nkv = nkv; p.max_pos = g.max_pos;
  p.slots_end = (long long)g.num_blocks * kQ8Page;
  uintptr_t at = 0;
  for (const void* a : {qkv_bf16, (const void*)qkv_partials, g.bias, (const void*)g.cos_sin, g.q_norm_w, g.k_norm_w, (const void*)g.q_out,
                        (const void*)g.k_values, (const void*)g.v_values})
    at |= reinterpret_cast<uintptr_t>(a);
  // A few tokens are bound by latency and keep a warp per head: 64 of them from partial sums 3.3 us and 4.1 in pieces, 128 5.7 and 5.5, 255 from
  // bf16 4.3 and 3.05.
  const bool pieces = tokens >= (qkv_partials ? 128 : 64) && (at & 15) == 0 && (!qkv_partials || (g.split_stride & 3) == 0);
  const long long heads = (long long)tokens * (nq + 2 * nkv);
  if (heads > 0x7fffffffll) return -2;
  // runs so long that all warps are resident at once
  const int steps = (nq + 2 * nkv + 512 / head_dim - 1) / (512 / head_dim);
  const long long resident = num_sms() * (qkv_partials ? 16 : 24), need = ((long long)tokens * steps + resident - 1) / resident;
  const long long run = need > steps ? steps : need;
  const long long blocks = ((pieces ? tokens * ((steps + run - 1) / run) : heads) + 7) / 8;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(g.stream);
  const dim3 grid = dim3(unsigned(blocks));
#define NKB_APPEND(D)                                                                                                                 \
  return pieces ? launch_pdl(qkv_partials ? append8_q8_kernel<D, true> : append8_q8_kernel<D, false>, grid, dim3(256), 0, s, p, int(run)) \
                : launch_pdl(append_q8_kernel<D>, grid, dim3(256), 0, s, p)
  if (head_dim == 128) NKB_APPEND(128);
  if (head_dim == 64) NKB_APPEND(64);
#undef NKB_APPEND
  return -2;
}
