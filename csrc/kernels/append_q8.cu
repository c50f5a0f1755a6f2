// Queries, keys and values of new tokens from the fused QKV projection: split-K partials summed, bias, per-head RMSNorm, rotate-halves
// RoPE; queries leave as bf16, keys and values go to their places in 8-bit pages (kv_quant.cuh).  The counterpart of
// rope_kv_append (elementwise.cu) for a quantised cache.
//
// Keys and values are computed in 64 bits, so that their one rounding to e4m3 does not depend on the order of operations.
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

// The same in pieces of sixteen bytes: D / 16 lanes share a head, each with eight elements of its first half and the eight that turn with
// them.  Every pointer on 16 bytes, split_stride a multiple of four.
template <int D, bool PARTIALS>
__global__ void __launch_bounds__(256, PARTIALS ? 2 : 4) append8_q8_kernel(const AppendQ8Params p) {
  constexpr int L = D / 16;
  constexpr uint32_t kAll = 0xffffffffu;
  const int heads = p.nq + 2 * p.nkv;
  const long long units = (long long)p.tokens * heads, unit = (blockIdx.x * (long long)blockDim.x + threadIdx.x) / L;
  const int i0 = (threadIdx.x % L) * 8;
  griddep_wait();
  griddep_launch();
  // a warp's lanes leave together or stay for the sums: units past the end repeat the last one and store nothing
  const bool on = unit < units;
  const long long u = on ? unit : units - 1;
  const int t = int(u / heads), h = int(u % heads);
  const bool is_q = h < p.nq, is_k = !is_q && h < p.nq + p.nkv;
  const long long base = (long long)t * heads * D + (long long)h * D + i0;
  auto get8 = [](const __nv_bfloat16* src, float* o) {
    const uint4 r = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 f = unpack_bf16x2(w[e]);
      o[2 * e] = f.x;
      o[2 * e + 1] = f.y;
    }
  };
  float x[16];                           // queries, and what goes to the pages; at first bf16 inputs, exactly
  double y[PARTIALS ? 16 : 1];           // sums of partials
  if constexpr (PARTIALS) {
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = 0.;
#pragma unroll 2
    for (int s = 0; s < p.splits; ++s) {
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p.partials + s * p.split_stride + base + (j < 8 ? j : D / 2 + j - 8));
        y[j] += double(v.x);
        y[j + 1] += double(v.y);
        y[j + 2] += double(v.z);
        y[j + 3] += double(v.w);
      }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = float(y[j]);
  } else {
    get8(p.qkv + base, x);
    get8(p.qkv + base + D / 2, x + 8);
  }
  const auto at = [&](int j) { return i0 + (j < 8 ? j : D / 2 + j - 8); };
  // the input with its bias in 64 bits
  const auto in64 = [&](int j) {
    double v;
    if constexpr (PARTIALS) v = y[j];
    else v = double(x[j]);
    return p.bias ? v + double(__bfloat162float(p.bias[h * D + at(j)])) : v;
  };
  const __nv_bfloat16* nw = is_q ? p.q_norm_w : (is_k ? p.k_norm_w : nullptr);
  const float* cs = nullptr;             // [cos(d/2) | sin(d/2)]
  if ((is_q || is_k) && p.cos_sin) cs = p.cos_sin + (long long)min(max(p.positions[t], 0), p.max_pos - 1) * D + i0;
  if (is_q && p.bias) {
    float b[16];
    get8(p.bias + h * D + i0, b);
    get8(p.bias + h * D + D / 2 + i0, b + 8);
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] += b[j];
  }
  double inv = 1.;
  if (p.q_norm_w || p.k_norm_w) {
    double ss = 0.;
    if (is_q) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) s += x[j] * x[j];
      ss = double(s);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const double v = in64(j);
        ss += v * v;
      }
    }
#pragma unroll
    for (int m = L / 2; m > 0; m >>= 1) ss += __shfl_xor_sync(kAll, ss, m);
    if (nw) inv = 1. / sqrt(ss / double(D) + p.eps);
  }
  if (is_q) {
    if (nw) {
      float w[16];
      get8(nw + i0, w);
      get8(nw + D / 2 + i0, w + 8);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = x[j] * float(inv) * w[j];
    }
    if (cs) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const float4 c4 = *reinterpret_cast<const float4*>(cs + j), s4 = *reinterpret_cast<const float4*>(cs + D / 2 + j);
        const float c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float a = x[j + k], d = x[8 + j + k];
          x[j + k] = a * c[k] - d * sn[k];
          x[8 + j + k] = d * c[k] + a * sn[k];
        }
      }
    }
    if (!on) return;
    __nv_bfloat16* dst = p.q_out + ((long long)t * p.nq + h) * D + i0;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    *reinterpret_cast<uint4*>(dst + D / 2) =
        make_uint4(pack_bf16x2(x[8], x[9]), pack_bf16x2(x[10], x[11]), pack_bf16x2(x[12], x[13]), pack_bf16x2(x[14], x[15]));
    return;
  }
  if (is_k || PARTIALS || p.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      double a = in64(j), d = in64(8 + j);
      if (nw) {
        a = a * inv * double(__bfloat162float(nw[at(j)]));
        d = d * inv * double(__bfloat162float(nw[at(8 + j)]));
      }
      if (cs) {
        const double c = cs[j], sn = cs[D / 2 + j], a0 = a;
        a = a0 * c - d * sn;
        d = d * c + a0 * sn;
      }
      x[j] = round_to_odd(a);
      x[8 + j] = round_to_odd(d);
    }
  }
  float amax = 0.f;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    fine = fine && isfinite(x[j]);
    amax = fmaxf(amax, fabsf(x[j]));
  }
  // the lanes of this head (those of queries have left)
  const uint32_t mine = ((1u << L) - 1u) << ((threadIdx.x & 31) / L * L);
#pragma unroll
  for (int m = L / 2; m > 0; m >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mine, amax, m));
  fine = __all_sync(mine, fine);
  const long long slot = p.slots ? p.slots[t] : -1;
  if (!on || slot < 0 || slot >= p.slots_end) return;
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

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_q8_append(const void* qkv_bf16, const float* qkv_partials, int splits, long long split_stride, const void* bias,
                             const int* positions, const int* slots, const float* cos_sin, const void* q_norm_w, const void* k_norm_w,
                             double eps, void* q_out, void* k_values, void* k_scales, void* v_values, void* v_scales, int tokens, int nq,
                             int nkv, int head_dim, int max_pos, int num_blocks, void* stream) {
  if (tokens <= 0) return 0;
  AppendQ8Params p{};
  p.qkv = (const __nv_bfloat16*)qkv_bf16;
  p.partials = qkv_partials;
  p.splits = splits;
  p.split_stride = split_stride;
  p.bias = (const __nv_bfloat16*)bias;
  p.positions = positions;
  p.slots = slots;
  p.cos_sin = cos_sin;
  p.q_norm_w = (const __nv_bfloat16*)q_norm_w;
  p.k_norm_w = (const __nv_bfloat16*)k_norm_w;
  p.eps = eps;
  p.q_out = (__nv_bfloat16*)q_out;
  p.k_values = (uint8_t*)k_values;
  p.k_scales = (uint8_t*)k_scales;
  p.v_values = (uint8_t*)v_values;
  p.v_scales = (uint8_t*)v_scales;
  p.tokens = tokens; p.nq = nq; p.nkv = nkv; p.max_pos = max_pos;
  p.slots_end = (long long)num_blocks * kQ8Page;
  uintptr_t at = 0;
  for (const void* a : {qkv_bf16, (const void*)qkv_partials, bias, (const void*)cos_sin, q_norm_w, k_norm_w, (const void*)q_out,
                        (const void*)k_values, (const void*)v_values})
    at |= reinterpret_cast<uintptr_t>(a);
  const bool pieces = tokens >= 256 && (at & 15) == 0 && (!qkv_partials || (split_stride & 3) == 0);
  const long long heads = (long long)tokens * (nq + 2 * nkv);
  if (heads > 0x7fffffffll) return -2;
  const dim3 blocks(unsigned(pieces ? (heads * (head_dim / 16) + 255) / 256 : (heads + 7) / 8));
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define NKB_APPEND(D) \
  return launch_pdl(pieces ? (qkv_partials ? append8_q8_kernel<D, true> : append8_q8_kernel<D, false>) : append_q8_kernel<D>, blocks, dim3(256), 0, s, p)
  if (head_dim == 128) NKB_APPEND(128);
  if (head_dim == 64) NKB_APPEND(64);
#undef NKB_APPEND
  return -2;
}
