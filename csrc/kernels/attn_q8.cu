// Attention over 8-bit pages (kv_quant.cuh), any number of new tokens per sequence: a warp per (query, head) walks the keys that the
// query sees, a page at a time.
//
//   o = sum_j exp(s_j) 2^{v_j} v8_j / sum_j exp(s_j),   s_j = scale * 2^{k_j} (q . k8_j)
//
// with 2^{k_j}, 2^{v_j} the tokens' scales.  Running maximum, sum and result in 32 bits.  A row that sees nothing is zero.
#include "api.h"
#include "kv_quant.cuh"
#include <math.h>

namespace nkb {

struct AttnQ8Params {
  const __nv_bfloat16* q;
  const uint8_t *k_values, *k_scales, *v_values, *v_scales;
  const int *block_table, *q_start, *q_lens, *context_lens;
  __nv_bfloat16* out;
  const float* sinks;
  int total_q, max_q_len, nq, nkv, num_blocks, table_width, causal, window, chunk;
  long long table_stride;
  float scale_log2;
};

template <int D>
__global__ void __launch_bounds__(256) attn_q8_simple_kernel(const AttnQ8Params p) {
  constexpr int PER = D / 32;
  const int lane = threadIdx.x & 31, i = blockIdx.x * 8 + (threadIdx.x >> 5), head = blockIdx.y, b = blockIdx.z;
  griddep_wait();
  griddep_launch();
  const int n = p.q_lens ? p.q_lens[b] : p.max_q_len;
  const long long row = (p.q_start ? p.q_start[b] : (long long)b * p.max_q_len) + i;
  if (i >= n || row < 0 || row >= p.total_q) return;
  const int ctx = min(p.context_lens[b], p.table_width * kQ8Page), pos = ctx - n + i, kvh = head / (p.nq / p.nkv);
  const int hi = p.causal ? min(ctx - 1, pos) : ctx - 1, lo = nkb_first_visible(pos, p.window, p.chunk);
  float q[PER], o[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    q[j] = __bfloat162float(p.q[(row * p.nq + head) * D + lane * PER + j]) * p.scale_log2;
    o[j] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int page = lo / kQ8Page; page * kQ8Page <= hi; ++page) {
    const int blk = p.block_table[b * p.table_stride + page];
    const bool in = blk >= 0 && blk < p.num_blocks;
    const long long at = ((in ? (long long)blk : 0) * p.nkv + kvh) * kQ8Page;
    for (int j = max(lo - page * kQ8Page, 0); j <= min(hi - page * kQ8Page, kQ8Page - 1); ++j) {
      const float kf = in ? q8_factor_of(p.k_scales[at + j]) : 0.f, vf = in ? q8_factor_of(p.v_scales[at + j]) : 0.f;
      float s = 0.f, v[PER];
#pragma unroll
      for (int d = 0; d < PER; d += 2) {
        const long long x = (at + j) * D + lane * PER + d;
        const __half2_raw kr = __nv_cvt_fp8x2_to_halfraw2(*reinterpret_cast<const uint16_t*>(p.k_values + x), __NV_E4M3);
        const __half2_raw vr = __nv_cvt_fp8x2_to_halfraw2(*reinterpret_cast<const uint16_t*>(p.v_values + x), __NV_E4M3);
        const float2 k2 = __half22float2(kr), v2 = __half22float2(vr);
        s = fmaf(q[d], k2.x, fmaf(q[d + 1], k2.y, s));
        v[d] = v2.x;
        v[d + 1] = v2.y;
      }
      s = warp_sum(s) * kf;
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn, keep = exp2f(m - base), w = exp2f(s - base);
      m = mn;
      l = l * keep + w;
#pragma unroll
      for (int d = 0; d < PER; ++d) o[d] = o[d] * keep + w * vf * (in ? v[d] : 0.f);
    }
  }
  if (p.sinks) {
    const float sk = p.sinks[head] * 1.4426950408889634f, m2 = fmaxf(m, sk), keep = m == -INFINITY ? 0.f : exp2f(m - m2);
    l = l * keep + exp2f(sk - m2);
#pragma unroll
    for (int d = 0; d < PER; ++d) o[d] *= keep;
  }
#pragma unroll
  for (int d = 0; d < PER; ++d) p.out[(row * p.nq + head) * D + lane * PER + d] = __float2bfloat16(l == 0.f ? 0.f : o[d] / l);
}

}  // namespace nkb

using namespace nkb;

// q_start and q_lens null: every sequence has max_q_len new tokens, one behind another
extern "C" int nkb_q8_attn_simple(const void* q, const void* k_values, const void* k_scales, const void* v_values, const void* v_scales,
                                  const int* block_table, const int* q_start, const int* q_lens, const int* context_lens, void* out,
                                  int batch, int total_q, int max_q_len, int nq, int nkv, int head_dim, int num_blocks, int table_width,
                                  long long table_stride, float scale, int causal, int window, int chunk, const float* sinks,
                                  void* stream) {
  if (batch <= 0 || total_q <= 0) return 0;
  if (batch > 65535 || nq > 65535 || nkv < 1 || nq % nkv) return -2;
  AttnQ8Params p{};
  p.q = (const __nv_bfloat16*)q;
  p.k_values = (const uint8_t*)k_values; p.k_scales = (const uint8_t*)k_scales;
  p.v_values = (const uint8_t*)v_values; p.v_scales = (const uint8_t*)v_scales;
  p.block_table = block_table; p.q_start = q_start; p.q_lens = q_lens; p.context_lens = context_lens;
  p.out = (__nv_bfloat16*)out;
  p.sinks = sinks;
  p.total_q = total_q; p.max_q_len = max_q_len; p.nq = nq; p.nkv = nkv; p.num_blocks = num_blocks; p.table_width = table_width;
  p.causal = causal; p.window = window; p.chunk = chunk;
  p.table_stride = table_stride;
  p.scale_log2 = scale * 1.4426950408889634f;
  const dim3 grid((max_q_len + 7) / 8, nq, batch);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_pdl(attn_q8_simple_kernel<128>, grid, dim3(256), 0, s, p);
  if (head_dim == 64) return launch_pdl(attn_q8_simple_kernel<64>, grid, dim3(256), 0, s, p);
  return -2;
}
