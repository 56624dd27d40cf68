#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace air {

struct LogitRulesArgs {
  const void* logits;        // [B, V] f32 or bf16
  int bf16;
  int64_t ld_in, ld_out;
  float* out;                // [B, V] f32 (may be the f32 logits)
  int B, V;
  const uint8_t* counts;     // [S, V] occurrences so far (null: no penalties)
  const int* count_row;      // [B] row of counts (null: b), -1: none
  int64_t S;
  const float* repetition;   // [B] (null: 1)
  const float* frequency;    // [B] (null: 0)
  const float* presence;     // [B] (null: 0)
  const int* bias_ptr;       // [B + 1] (null: no biases)
  const int* bias_ids;
  const float* bias_vals;
  int64_t n_bias;            // entries of bias_ids / bias_vals
  const uint32_t* mask;      // [B, ceil(V / 32)] allow bits (null: all allowed)
  int* err;
};

void launch_logit_rules(const LogitRulesArgs& a, cudaStream_t st);

}  // namespace air
