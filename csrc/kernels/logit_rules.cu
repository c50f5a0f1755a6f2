// Rules on logits: penalties for repeated tokens, biases and masks; the logits that are left, or the most likely token.
//
// Mathematics, per row, for the tokens that the rules name, in 64 bits and rounded once:
//   seen (in the prompt or the answer):  l = l > 0 ? l / repetition : l * repetition
//   n times among the answer's tokens:   l -= frequency * n;  l -= presence where n > 0
//   biases:                              l += the sum of the token's entries, in their order
//   mask bit zero:                       l = -inf
// Most tokens are named by none: they pass as they are, and in place they are not even read.
//
// A slice of the vocabulary per CTA.  Its counts lie in shared memory, one word per token (bit 31: seen, bit 30: has a bias, below: times in the answer), filled
// from the row's whole list of tokens, so there is no state to keep beside that list, no hashing, and no limit on its length; whole numbers, so the
// order of the counting changes nothing.  Then one pass over the slice's logits.  The most likely token of a row's slices is found by the CTAs of a cluster
// through distributed shared memory: no workspace that calls could share, and ties go to the lowest index.
#include "api.h"
#include "common.cuh"
#include "rules_args.h"

namespace nkb {

constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u, kTimes = 0x3fffffffu;
constexpr int kSliceMost = 24576;       // tokens whose counts are held at a time (96 KB)
constexpr int kRuleThreads = 512;

struct RuleRow {
  double rep, freq, pres;
  const int* bias_ids;
  const float* bias_values;
  int biases;
};

__device__ __noinline__ float ruled(const RuleRow& r, float l0, uint32_t c, int token) {
  double l = l0;
  if (c & kSeen) {
    l = l > 0.0 ? l / r.rep : l * r.rep;
    const uint32_t n = c & kTimes;
    l -= r.freq * double(n);
    if (n) l -= r.pres;
  }
  if (c & kBiased) {
    double sum = 0.0;
    for (int i = 0; i < r.biases; ++i)
      if (r.bias_ids[i] == token) sum += double(r.bias_values[i]);
    l += sum;
  }
  return float(l);
}

template <bool F32>
__device__ __forceinline__ float rule_logit(const void* p, long long i) {
  return F32 ? reinterpret_cast<const float*>(p)[i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}

// Grid: x = slices of a row (a cluster where ids are wanted), y strides over the rows.
template <bool F32, bool VEC>
__global__ void __launch_bounds__(kRuleThreads) logit_rules_kernel(const NkbLogitRules a, int slice) {
  extern __shared__ __align__(16) uint32_t counts[];
  __shared__ float s_best[kRuleThreads / 32];
  __shared__ int s_at[kRuleThreads / 32];
  __shared__ int2 s_mine;               // best of this CTA's slice: bits of the value, token
  constexpr int kPer = 8;               // tokens of a piece
  constexpr int kBytes = F32 ? 4 : 2;
  griddep_wait();
  griddep_launch();
  const int row = blockIdx.y, tid = threadIdx.x;
  const int first = blockIdx.x * slice, last = min(a.vocab, first + slice);
  const int len = a.tokens ? min(a.lens[row], a.width) : 0;
  const int prompt = a.prompts && a.tokens ? a.prompts[row] : 0;
  int* tokens = a.tokens ? a.tokens + row * a.tokens_ld : nullptr;
  const bool fresh = a.ids && len > 0;
  const int newest = fresh ? a.ids[row] : 0;
  if (fresh && blockIdx.x == 0 && tid == 0) tokens[len - 1] = newest;      // (the others take it from ids)
  RuleRow r;
  r.rep = a.repetition ? double(a.repetition[row]) : 1.0;
  r.freq = a.frequency ? double(a.frequency[row]) : 0.0;
  r.pres = a.presence ? double(a.presence[row]) : 0.0;
  r.bias_ids = a.bias_ids + row * a.bias_ld;
  r.bias_values = a.bias_values + row * a.bias_ld;
  r.biases = a.biases;
  const bool counted = len > 0 && (r.rep != 1.0 || r.freq != 0.0 || r.pres != 0.0);
  const int mrow = a.mask_rows ? a.mask_rows[row] : row;
  const int* mask = a.mask && mrow >= 0 && mrow < a.mask_count ? a.mask + mrow * a.mask_ld : nullptr;
  const uint8_t* in = reinterpret_cast<const uint8_t*>(a.logits) + (long long)row * a.ld * kBytes;
  uint8_t* out = reinterpret_cast<uint8_t*>(a.out) + (a.out ? (long long)row * a.out_ld * kBytes : 0);
  const bool in_place = a.out && out == in;
  const bool named = counted || a.biases > 0;
  float best = -INFINITY;
  int at = 0x7fffffff;

  for (int lo = first; lo < last; lo += kSliceMost) {
    const int hi = min(last, lo + kSliceMost);
    if (named) {
      for (int i = tid; i < (hi - lo + 3) / 4; i += kRuleThreads) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
      __syncthreads();
      if (counted) {
        for (int i = tid; i < len; i += kRuleThreads) {
          const int t = (fresh && i == len - 1 ? newest : tokens[i]) - lo;
          if (t < 0 || t >= hi - lo) continue;
          atomicOr(&counts[t], kSeen);
          if (i >= prompt) atomicAdd(&counts[t], 1u);
        }
      }
      for (int i = tid; i < a.biases; i += kRuleThreads) {
        const int t = r.bias_ids[i] - lo;
        if (t >= 0 && t < hi - lo) atomicOr(&counts[t], kBiased);
      }
      __syncthreads();
    }
    for (int p = tid; p < (hi - lo + kPer - 1) / kPer; p += kRuleThreads) {
      const int t0 = lo + p * kPer, n = min(kPer, hi - t0);
      uint32_t c[kPer];
      uint32_t any = 0;
      if (named) {
        const uint4 c0 = reinterpret_cast<const uint4*>(counts)[2 * p], c1 = reinterpret_cast<const uint4*>(counts)[2 * p + 1];
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w;
        c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
#pragma unroll
        for (int j = 0; j < kPer; ++j) any |= j < n ? c[j] : 0u;
      }
      const uint32_t left = mask ? (uint32_t(mask[t0 >> 5]) >> (t0 & 31)) & 255u : 255u;
      if (in_place && !any && left == 255u && !a.out_ids) continue;
      float l[kPer];
      if (VEC && n == kPer) {
        if constexpr (F32) {
          const float4 x = reinterpret_cast<const float4*>(in + t0 * 4ll)[0], y = reinterpret_cast<const float4*>(in + t0 * 4ll)[1];
          l[0] = x.x; l[1] = x.y; l[2] = x.z; l[3] = x.w;
          l[4] = y.x; l[5] = y.y; l[6] = y.z; l[7] = y.w;
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(in + t0 * 2ll);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = unpack_bf16x2(w[e]);
            l[2 * e] = f.x;
            l[2 * e + 1] = f.y;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) l[j] = j < n ? rule_logit<F32>(in, t0 + j) : 0.f;
      }
      if (any) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j < n && c[j]) l[j] = ruled(r, l[j], c[j], t0 + j);
      }
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (!((left >> j) & 1u)) l[j] = -INFINITY;
      if (a.out) {
        if (VEC && n == kPer) {
          if constexpr (F32) {
            reinterpret_cast<float4*>(out + t0 * 4ll)[0] = make_float4(l[0], l[1], l[2], l[3]);
            reinterpret_cast<float4*>(out + t0 * 4ll)[1] = make_float4(l[4], l[5], l[6], l[7]);
          } else {
            *reinterpret_cast<uint4*>(out + t0 * 2ll) = make_uint4(pack_bf16x2(l[0], l[1]), pack_bf16x2(l[2], l[3]), pack_bf16x2(l[4], l[5]),
                                                                   pack_bf16x2(l[6], l[7]));
          }
        } else {
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (j < n) {
              if constexpr (F32) reinterpret_cast<float*>(out)[t0 + j] = l[j];
              else reinterpret_cast<__nv_bfloat16*>(out)[t0 + j] = __float2bfloat16(l[j]);
            }
        }
      }
      if (a.out_ids) {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j < n && l[j] > best) {            // pieces of a thread come in ascending order; a NaN loses against every number
            best = l[j];
            at = t0 + j;
          }
      }
    }
    if (named) __syncthreads();
  }
  if (!a.out_ids) return;
  auto better = [&](float v, int i) {
    if (v > best || (v == best && i < at)) {
      best = v;
      at = i;
    }
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best, o);
    const int i = __shfl_xor_sync(0xffffffffu, at, o);
    better(v, i);
  }
  if ((tid & 31) == 0) {
    s_best[tid >> 5] = best;
    s_at[tid >> 5] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kRuleThreads / 32; ++w) better(s_best[w], s_at[w]);
    s_mine = make_int2(__float_as_int(best), at);
  }
  if (gridDim.x > 1) {
    cluster_sync_all();
    if (blockIdx.x == 0 && tid == 0)
      for (unsigned c = 1; c < gridDim.x; ++c) {
        int v, i;
        asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v), "=r"(i) : "r"(map_to_cta(&s_mine, c)) : "memory");
        better(__int_as_float(v), i);
      }
    cluster_sync_all();               // shared memory stays until it has been read
  }
  if (blockIdx.x == 0 && tid == 0) a.out_ids[row] = best == -INFINITY ? -1 : at;
}

template <bool F32, bool VEC>
static int launch_rules(const NkbLogitRules& a) {
  // slices: a cluster of up to eight where ids are wanted, otherwise as many as give every SM some two CTAs
  int slices = (2 * num_sms() + a.rows - 1) / a.rows;
  if (a.out_ids && slices > 8) slices = 8;
  int fewest = (a.vocab + kSliceMost - 1) / kSliceMost;         // (a slice that has more runs in several turns)
  if (a.out_ids && fewest > 8) fewest = 8;
  if (slices < fewest) slices = fewest;
  int slice = ((a.vocab + slices - 1) / slices + 511) / 512 * 512;
  slices = (a.vocab + slice - 1) / slice;
  const int smem = (slice < kSliceMost ? slice : kSliceMost) * 4;
  constexpr int kMaxDev = 64;
  static bool ready[kMaxDev] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(logit_rules_kernel<F32, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceMost * 4);
    if (e != cudaSuccess) return int(e);
    ready[dev] = true;
  }
  return launch_pdl_cluster(logit_rules_kernel<F32, VEC>, dim3(unsigned(slices), unsigned(a.rows)), dim3(kRuleThreads), size_t(smem),
                            reinterpret_cast<cudaStream_t>(a.stream), a.out_ids ? slices : 1, a, slice);
}

}  // namespace nkb

using namespace nkb;

extern "C" int nkb_logit_rules(const void* packed) {
  const NkbLogitRules& a = *reinterpret_cast<const NkbLogitRules*>(packed);
  if (!status_word() && nkb_init() != 0) return -1;
  if (a.rows <= 0) return 0;
  if (a.vocab <= 0 || a.rows > 65535 || (!a.out && !a.out_ids) || a.biases < 0 || a.width < 0) return -2;
  if (a.tokens && !a.lens) return -2;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out);
  const bool vec = (at & 15) == 0 && ((a.ld | (a.out ? a.out_ld : 0)) & (a.fp32 ? 3 : 7)) == 0;
  if (a.fp32) return vec ? launch_rules<true, true>(a) : launch_rules<true, false>(a);
  return vec ? launch_rules<false, true>(a) : launch_rules<false, false>(a);
}
