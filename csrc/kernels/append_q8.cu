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
  const long long warps = (long long)tokens * (nq + 2 * nkv), blocks = (warps + 7) / 8;
  if (blocks > 0x7fffffffll) return -2;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_pdl(append_q8_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, s, p);
  if (head_dim == 64) return launch_pdl(append_q8_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, s, p);
  return -2;
}
