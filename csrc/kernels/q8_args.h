// Arguments of the operators on 8-bit pages (kv_quant.cuh has the format).  The caller packs them in this order; both sizes are multiples of
// eight bytes.
#pragma once

// Append: queries, keys and values of `tokens` new tokens from the fused QKV projection [tokens][(nq + 2 nkv) * head_dim], bf16 or split-K
// partial sums.
struct NkbQ8Append {
  const void* qkv;                       // bf16, or null
  const float* partials;                 // [splits][tokens][...]
  const void* bias;                      // bf16, or null
  const int *positions, *slots;          // slots (null: none): places in the pages, negative or past them: nothing is stored
  const float* cos_sin;                  // [max_pos][cos(head_dim / 2) | sin(head_dim / 2)], or null
  const void *q_norm_w, *k_norm_w;       // bf16 [head_dim], or null
  void* q_out;                           // bf16 [tokens][nq * head_dim]
  void *k_values, *k_scales, *v_values, *v_scales;
  void* stream;
  long long split_stride;
  double eps;
  int splits, tokens, nq, nkv, head_dim, max_pos, num_blocks, unused;
};

// Attention of the newest tokens of `batch` sequences over their pages.
struct NkbQ8Attn {
  const void* q;                         // bf16 [total_q][nq * head_dim]
  const void *k_values, *k_scales, *v_values, *v_scales;
  const int* block_table;                // [batch][table_width], rows table_stride apart; blocks outside the pool read as zeros
  const int *q_start, *q_lens;           // first row and rows of a sequence (prompts)
  const int* context_lens;               // tokens of a sequence, the new ones counted
  void* out;
  const float* sinks;                    // [nq], or null
  // Workspace as large as the functions below say.  The first kQ8Counters words are zero before the first call, and a call leaves them at zero;
  // not shared by calls that may run at the same time.
  float* scratch;
  void* stream;
  long long table_stride;
  long long scratch_floats;              // what there is of it; a call that wants more is refused
  int batch, total_q, q_len;             // q_len: new tokens of every sequence (prompts: at most)
  int nq, nkv, head_dim, num_blocks, table_width, causal, window, chunk, num_splits;
  float scale;
  int unused;
};
constexpr int kQ8Counters = 16384;
