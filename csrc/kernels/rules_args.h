// Arguments of the rules on logits (logit_rules.cu).  The caller packs them in this order; the size is a multiple of eight bytes.
#pragma once

struct NkbLogitRules {
  const void* logits;            // [rows, vocab], bf16 or fp32
  void* out;                     // the same type, may be the logits themselves; null: none
  int* out_ids;                  // [rows]: the most likely token, -1 where none is left; null: none
  int* tokens;                   // [rows][width] ids of a row in their order; null: none
  const int *lens, *prompts;     // of a row's tokens, and those of its prompt among them (null: none); a length below one: no tokens
  const int* ids;                // [rows] the newest token, written to its place; null: it is there
  const float *repetition, *frequency, *presence;   // [rows], null: none
  const int* bias_ids;           // [rows][biases], negative: none
  const float* bias_values;
  const int* mask;               // [mask_count][words] bits, one per token, zero: not allowed; null: none
  const int* mask_rows;          // [rows] mask of a row, outside the masks: none; null: row b has mask b
  void* stream;
  long long ld, out_ld, tokens_ld, bias_ld, mask_ld;
  int rows, vocab, width, biases, mask_count, fp32;
};
