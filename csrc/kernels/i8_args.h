// Arguments of the operators on rows and weights held as 8-bit whole numbers (quant_rows.cu, gemm_i8.cu).  The caller packs them in this order;
// sizes are multiples of eight bytes.
#pragma once

// What a row is made of before it is brought into 8 bits.
enum NkbRowForm {
  NKB_ROW_BF16 = 0,       // x bf16
  NKB_ROW_F32 = 1,        // x fp32
  NKB_ROW_NORM = 2,       // h = partial sums + x + bias + residual, rounded to bf16; the row is h * w, with the RMS norm's factor in its scale
  NKB_ROW_GATE_BF16 = 3,  // x bf16 [2 width]: act(gate) * up
  NKB_ROW_GATE_F32 = 4,   // the same of the sum of fp32 partial sums, with a bias
};

struct NkbQuantRows {
  const void* x;                // rows x_ld elements apart; null: none (norm)
  const float* partials;        // [splits][rows], rows x_ld apart; null: none
  const void* bias;             // bf16 [width], gate: [2 width]; null: none
  const void* residual;         // bf16, rows of `width`; null: none
  const void* w;                // bf16 [width] (norm)
  void* residual_out;           // bf16, rows of `width`; null: not stored
  void* values;                 // int8, rows q_ld apart; q_ld at least the width rounded up to 16, which is written with zeros
  float* scale;                 // [rows]
  void* stream;
  long long x_ld, q_ld, split_stride;
  int form, rows, width, splits;
  float eps, limit, alpha;      // limit > 0: (up + 1) * gate * sigmoid(alpha * gate) of clamped gate and up
  int late;                     // the kernel behind this one starts after its end: it may take the rows for weights, which it fetches ahead of its wait
};

// y = x w^T of whole numbers, times both scales.
struct NkbGemmI8 {
  const void *x, *w;            // int8 [m, k] and [n, k] (gated: [2 n, k], gate rows and then up rows)
  const float *x_scale, *w_scale;
  const void* bias;             // bf16 [n], null: none (not gated)
  const void* residual;         // bf16 [m, n] with rows ldo apart, null: none (not gated)
  void* out;                    // [m, n]
  void* stream;
  long long ldx, ldw, ldo, split_stride;
  int m, n, k;
  int gated, act;               // act 0: SiLU, 1: GELU (tanh form)
  int fp32;                     // results in 32 bits
  int splits;                   // > 0: that many partial sums in 32 bits, split s at out + s * split_stride; 0: whole results
  int static_w;                 // w is not written by the kernel before this one
};
