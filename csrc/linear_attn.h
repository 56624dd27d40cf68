// Linear attention with one decay per head (recurrent decoder layers).
//   S_t = exp(g_t) S_{t-1} + v_t k_t^T,   o_t = scale * S_t q_t      (S [dv, dk], per head, f32)
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace air {

struct LinAttnArgs {
  const void *q, *k, *v;            // [T, heads, d] rows of bf16 or f32 (inner stride 1)
  void* out;                        // [T, H, dv], the type of q
  int64_t qs_t, qs_h, ks_t, ks_h, vs_t, vs_h, os_t, os_h;   // token / head strides in elements
  int q_div, k_div, v_div;          // state heads that share one q / k / v head
  const float* decay;               // g: [T, H], or [H] with decay_t = 0
  int64_t decay_t;
  const int* cu;                    // [N + 1] token offsets of the packed sequences
  int whole;                        // cu null: 1 one sequence of all T tokens, 0 one token per sequence
  const int* slots;                 // [N] state row of each sequence, -1: none (null: row n)
  const int* has_state;             // [N] 0: start from zeros (null: has_state_all)
  int has_state_all;
  int zero_pad;                     // 1: a sequence without a state row writes zeros
  float* state;                     // [S, H, dv, dk] f32, read and updated (null: from zeros, not kept)
  int64_t S;
  int N, T, H, dk, dv;
  float scale;
  int* err;
};

// Any dk <= 256 and any dv: token by token.
void launch_linear_scan(const LinAttnArgs& a, bool f32, cudaStream_t st);
// One token per sequence, dk in {64, 128}, dv a multiple of 8, 16-byte aligned state.
bool linear_step_supported(const LinAttnArgs& a, bool f32);
void launch_linear_step(const LinAttnArgs& a, bool f32, cudaStream_t st);


// Blocks of 128 tokens on the tensor cores: bf16, dk and dv in {64, 128}, rows and strides of whole
// 16-byte units.
bool linear_blocks_supported(const LinAttnArgs& a, bool f32);
bool linear_blocks_worth(const LinAttnArgs& a);         // against launch_linear_scan, by size
// Floats of scratch that launch_linear_blocks needs (0: none).
int64_t linear_blocks_workspace(const LinAttnArgs& a, int sms);
const char* launch_linear_blocks(const LinAttnArgs& a, float* ws, int sms, cudaStream_t st);

}  // namespace air
