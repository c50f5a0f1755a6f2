// Products of one or two tokens with weights in 8-bit whole numbers, on the CUDA cores: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] w[n, k].
//
// A weight is read once and multiplied with one or two rows: 16 bytes of it are 4 or 8 instructions (four products and sums each), while the memory
// gives an SM some 23 bytes per clock.  So the bytes bound it, and the tensor cores' tiles, of 128 features by 16 tokens at least, would only add a
// start, a ring and an end.  Rows that come in bf16 or fp32 are brought into 8 bits by every CTA for itself (quant_rows.cu has the mathematics; the same numbers), under
// the first weights' way from memory: a kernel, a launch and a buffer less.
//
// A warp per feature (gate and up: two), whose lanes read 16 bytes each, eight times ahead; sums over lanes by one integer reduction, so the order changes
// nothing and the results are those of the other kernels, bit by bit (i8_epilogue.cuh).
//
// us, bf16 rows, here and on the tensor cores: one token by 6144 x 4096 6.7 and 9.4 (the bytes' floor 3.9), by 4096 x 4096 5.2 and 8.2, by 4096 x 14336 14.5 and
// 17.0, by 2 x 14336 x 4096 22.4 and 26.7; two tokens 9.5 and 9.8, 6.5 and 8.5, 18.1 and 17.1, 24.4 and 26.9.  Three and four rows were slower in every CTA's own
// way into 8 bits (four by 6144 x 4096 13.4 and 9.3), and in 8 bits already no faster (8.2 and 7.3).
#include "api.h"
#include "i8_args.h"
#include "i8_epilogue.cuh"
#include "quant_rows.cuh"

namespace nkb {

constexpr int kFewThreads = 512, kFewWarps = kFewThreads / 32;
constexpr int kFewAhead = 8;              // pieces of 512 bytes of a feature on their way
constexpr int kFewBytes = 96 * 1024;      // of rows in shared memory

struct FewArgs {
  const void* x;                // int8 rows x_ld apart, or bf16 or fp32 ones
  const int8_t* w;
  const float *sx, *sw;         // sx: of int8 rows
  const __nv_bfloat16 *bias, *residual;
  void* out;
  long long x_ld, w_ld, ldo;
  int n, k, act, fp32, static_w, x_vec;
};

__device__ __forceinline__ uint4 ld_once(const int8_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// FORM: NKB_ROW_BF16, NKB_ROW_F32, or -1 for rows in 8 bits.
template <int M, int FORM, bool GATED>
__global__ void __launch_bounds__(kFewThreads, 2) i8_few_kernel(const FewArgs a) {
  extern __shared__ __align__(16) uint8_t xq[];          // [M][padded], zeros behind k
  __shared__ float s_scale[M];
  __shared__ uint32_t s_top[M][kFewWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pieces = (a.k + 511) / 512, padded = pieces * 512;
  const int total = gridDim.x * kFewWarps;
  int n = blockIdx.x * kFewWarps + warp;
  uint4 w[kFewAhead];
  auto load = [&](const int8_t* row, int p0) {
#pragma unroll
    for (int i = 0; i < kFewAhead; ++i) {
      const int at = (p0 + i) * 512 + lane * 16;
      w[i] = at < a.k ? ld_once(row + at) : make_uint4(0u, 0u, 0u, 0u);        // (a row's sixteen bytes lie within its pitch)
    }
  };
  // weights that no kernel before this one writes are on their way before its end
  const bool ahead = a.static_w && n < a.n;
  if (ahead) load(a.w + n * a.w_ld, 0);
  griddep_wait();
  griddep_launch();
  if constexpr (FORM < 0) {
    for (int i = threadIdx.x; i < M * (padded / 16); i += kFewThreads) {
      const int m = i / (padded / 16), at = (i - m * (padded / 16)) * 16;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (at < a.k) {
        v = *reinterpret_cast<const uint4*>(reinterpret_cast<const int8_t*>(a.x) + m * a.x_ld + at);
        uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int left = a.k - at - 4 * e;       // numbers of this word
          if (left < 4) q[e] = left <= 0 ? 0u : q[e] & ((1u << (8 * left)) - 1u);
        }
        v = make_uint4(q[0], q[1], q[2], q[3]);
      }
      *reinterpret_cast<uint4*>(xq + m * padded + at) = v;
    }
    if (threadIdx.x < M) s_scale[threadIdx.x] = a.sx[threadIdx.x];
  } else {
    auto fetch = [&](int m, int c, float (&v)[8]) {
      if constexpr (FORM == NKB_ROW_BF16) {
        const __nv_bfloat16* row = reinterpret_cast<const __nv_bfloat16*>(a.x) + m * a.x_ld;
        values8_bf16(a.x_vec ? fetch8_bf16<true>(row, c, a.k) : fetch8_bf16<false>(row, c, a.k), v);
      } else {
        const float* row = reinterpret_cast<const float*>(a.x) + m * a.x_ld;
        uint4 r[2];
        if (a.x_vec) fetch8_f32<true>(row, c, a.k, r);
        else fetch8_f32<false>(row, c, a.k, r);
        values8_f32(r, v);
      }
    };
    float v[8];
#pragma unroll 1
    for (int m = 0; m < M; ++m) {
      float big = 0.f;
      for (int c = threadIdx.x * 8; c < a.k; c += kFewThreads * 8) {
        fetch(m, c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) big = max_nan(big, fabsf(v[j]));
      }
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
      if (lane == 0) s_top[m][warp] = top;
    }
    __syncthreads();
#pragma unroll 1
    for (int m = 0; m < M; ++m) {
      const uint32_t top = __reduce_max_sync(0xffffffffu, lane < kFewWarps ? s_top[m][lane] : 0u);
      const bool fine = top < 0x7f800000u;
      const float t = __uint_as_float(top);
      if (threadIdx.x == 0) s_scale[m] = fine ? t / 127.f : __uint_as_float(0x7fffffffu);
      const bool odd = odd_row(t);
      const float inv = odd ? 0.f : 127.f / t;
      for (int c = threadIdx.x * 8; c < padded; c += kFewThreads * 8) {
        uint2 q = make_uint2(0u, 0u);
        if (c < a.k && fine) {
          fetch(m, c, v);                 // (past k: zeros)
          q = numbers8<FORM == NKB_ROW_F32>(v, t, inv, odd);
        }
        *reinterpret_cast<uint2*>(xq + m * padded + c) = q;
      }
    }
  }
  __syncthreads();
  float sx = 0.f;
  if (lane < M) sx = s_scale[lane];

  bool loaded = ahead;
  for (; n < a.n; n += total) {
    int sum[GATED ? 2 : 1][M];
#pragma unroll
    for (int half = 0; half < (GATED ? 2 : 1); ++half) {
      const int8_t* row = a.w + (long long)(half * a.n + n) * a.w_ld;
      int acc[M];
#pragma unroll
      for (int m = 0; m < M; ++m) acc[m] = 0;
      for (int p0 = 0; p0 < pieces; p0 += kFewAhead) {
        if (!loaded) load(row, p0);
        loaded = false;
#pragma unroll
        for (int i = 0; i < kFewAhead; ++i) {
          if (p0 + i >= pieces) break;
          const int* wi = reinterpret_cast<const int*>(&w[i]);
#pragma unroll
          for (int m = 0; m < M; ++m) {
            const int4 x = *reinterpret_cast<const int4*>(xq + m * padded + (p0 + i) * 512 + lane * 16);
            acc[m] = __dp4a(wi[0], x.x, acc[m]);
            acc[m] = __dp4a(wi[1], x.y, acc[m]);
            acc[m] = __dp4a(wi[2], x.z, acc[m]);
            acc[m] = __dp4a(wi[3], x.w, acc[m]);
          }
        }
      }
#pragma unroll
      for (int m = 0; m < M; ++m) sum[half][m] = __reduce_add_sync(0xffffffffu, acc[m]);
    }
    int mine = 0, up = 0;
#pragma unroll
    for (int m = 0; m < M; ++m)
      if (lane == m) {
        mine = sum[0][m];
        if (GATED) up = sum[GATED ? 1 : 0][m];
      }
    if (lane < M) {
      float y = i8_scaled(mine, sx, __ldg(a.sw + n));
      const long long at = lane * a.ldo + n;
      if constexpr (GATED) {
        y = i8_gated(y, i8_scaled(up, sx, __ldg(a.sw + a.n + n)), a.act);
      } else {
        if (a.bias) y = add_rn(y, __bfloat162float(a.bias[n]));
        if (a.residual) y = add_rn(y, __bfloat162float(a.residual[at]));
      }
      if (a.fp32) reinterpret_cast<float*>(a.out)[at] = y;
      else reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16(y);
    }
  }
}

template <int M, int FORM, bool GATED>
static int launch_few(const FewArgs& a, void* stream) {
  constexpr int kMaxDev = 64;
  static bool ready[kMaxDev] = {false};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) return -1;
  if (!ready[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(i8_few_kernel<M, FORM, GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewBytes);
    if (e != cudaSuccess) return int(e);
    ready[dev] = true;
  }
  const int ctas = (a.n + kFewWarps - 1) / kFewWarps, most = 2 * num_sms();
  return launch_pdl(i8_few_kernel<M, FORM, GATED>, dim3(unsigned(ctas < most ? ctas : most)), dim3(kFewThreads), size_t(M) * ((a.k + 511) / 512 * 512),
                    reinterpret_cast<cudaStream_t>(stream), a);
}

template <int M, int FORM>
static int few_gated(const FewArgs& a, bool gated, void* stream) {
  return gated ? launch_few<M, FORM, true>(a, stream) : launch_few<M, FORM, false>(a, stream);
}
template <int FORM>
static int few_rows(const FewArgs& a, int m, bool gated, void* stream) {
  switch (m) {
    case 1: return few_gated<1, FORM>(a, gated, stream);
    case 2: return few_gated<2, FORM>(a, gated, stream);
  }
  return -2;
}

}  // namespace nkb

using namespace nkb;

// Whole products of one or two rows; rows: how x is brought into 8 bits (null: it is).  -5: not for this kernel (more rows, or more of them than shared
// memory has room for).
extern "C" int nkb_gemm_i8_few(const void* rows, const void* packed) {
  const NkbGemmI8& g = *reinterpret_cast<const NkbGemmI8*>(packed);
  if (g.m < 1 || g.m > 2 || g.splits || (long long)g.m * ((g.k + 511) / 512 * 512) > kFewBytes) return -5;
  if (!status_word() && nkb_init() != 0) return -1;
  if (g.n <= 0) return 0;
  if (g.k <= 0 || (g.ldw & 15) || g.ldw < g.k || g.ldo < g.n || (reinterpret_cast<uintptr_t>(g.w) & 15)) return -2;
  if (!rows && ((g.ldx & 15) || g.ldx < g.k || (reinterpret_cast<uintptr_t>(g.x) & 15))) return -2;
  if (g.gated && (g.bias || g.residual || g.fp32)) return -2;
  FewArgs a{};
  int form = -1;
  if (rows) {
    const NkbQuantRows& r = *reinterpret_cast<const NkbQuantRows*>(rows);
    form = r.form;
    a.x = r.x;
    a.x_ld = r.x_ld;
    a.x_vec = (reinterpret_cast<uintptr_t>(r.x) & 15) == 0 && (r.x_ld & 7) == 0;
  } else {
    a.x = g.x;
    a.x_ld = g.ldx;
  }
  a.w = reinterpret_cast<const int8_t*>(g.w);
  a.w_ld = g.ldw;
  a.sx = g.x_scale;
  a.sw = g.w_scale;
  a.bias = reinterpret_cast<const __nv_bfloat16*>(g.bias);
  a.residual = reinterpret_cast<const __nv_bfloat16*>(g.residual);
  a.out = g.out;
  a.ldo = g.ldo;
  a.n = g.n;
  a.k = g.k;
  a.act = g.act;
  a.fp32 = g.fp32;
  a.static_w = g.static_w;
  if (form < 0) return few_rows<-1>(a, g.m, g.gated, g.stream);
  if (form == NKB_ROW_BF16) return few_rows<NKB_ROW_BF16>(a, g.m, g.gated, g.stream);
  if (form == NKB_ROW_F32) return few_rows<NKB_ROW_F32>(a, g.m, g.gated, g.stream);
  return -2;
}
