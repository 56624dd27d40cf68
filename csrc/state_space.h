// Operators of a state-space decoder: causal convolution, selective scan, block norm, token log probabilities.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace air {

// Packed sequences and their state rows, shared by the convolution and the scan.
struct SeqArgs {
  const int* cu;           // [N + 1] token offsets (null: one sequence of all T tokens, or with `step` one token each)
  const int* slots;        // [N] state row of each sequence, -1: none (null: row n)
  const int* has_state;    // [N] 0: start from zeros (null: has_state_all)
  int has_state_all;
  int step;                // 1: sequence n is token n, and one without a state row writes zeros
  int64_t S;               // state rows (0: no state)
  int N, T;
  int* err;
};

struct ConvArgs {
  SeqArgs seq;
  const void* x;           // [T, D] bf16 or f32
  void* out;               // [T, D], the type of x
  int64_t xs, os;          // token strides in elements
  const float* w;          // [D, W]
  const float* bias;       // [D] (null: none)
  void* state;             // [S, W - 1, D], the type of x: the last inputs, the newest in the last row (null: none)
  int D, W, silu;
};
// 2 <= W <= 4. vec = 8, 4, 2 or 1 divides D, the rows of x, out and state are aligned to vec elements, w to 16 bytes.
const char* launch_causal_conv(const ConvArgs& a, bool f32, int vec, cudaStream_t st);

struct ScanArgs {
  SeqArgs seq;
  const void *x, *dt, *z;  // [T, D] bf16 or f32 (z null: no gate)
  const void *B, *C;       // [T, G, N] of the same type, the states contiguous
  void* out;               // [T, D] of the same type
  int64_t xs, ds, zs, os;  // token strides in elements
  int64_t bs_t, bs_g, cs_t, cs_g;
  const float* A;          // [D, N]
  const float *skip, *dt_bias;   // [D] (null: none)
  float* state;            // [S, D, N] f32 (null: from zeros, not kept)
  int D, G, N, softplus;
};
constexpr int kScanMaxStates = 256;
// Sequences token by token, a few threads per channel: any shape.
void launch_scan_tokens(const ScanArgs& a, bool f32, cudaStream_t st);

// Prompts in tiles of tokens, at most 64 states: the number of tiles, their tokens, whether SMs have two blocks each and the
// floats of scratch.
struct ScanPlan {
  int tiles, tile;
  bool pairs;
  int64_t floats;
};
bool scan_tiles_worth(const ScanArgs& a);       // against launch_scan_tokens, by size
ScanPlan scan_plan(const ScanArgs& a, int sms);
const char* launch_scan_tiles(const ScanArgs& a, const ScanPlan& p, float* ws, bool f32, cudaStream_t st);

struct BlockNormArgs {
  const void* y;           // [T, K] bf16 or f32
  const void* gate;        // [T, K] of y's type (null: none); ldg = 0: one row for all tokens
  const void* resid;       // [T, K] f32 or bf16 (null: none)
  void* resid_out;         // [T, K] of resid's type: resid + scale * h (null: not written)
  void* out;               // [T, K] bf16 or f32 (null: not written)
  const float *w, *post;   // [K] norm weights before the next block and after this one (null: no such norm)
  const float* scale_row;  // [K] (null: `scale`)
  float scale, w_offset, eps;
  int64_t ldy, ldg, ldr, ldro, ldo;
  int T, K;
  int y_bf16, r_bf16, o_bf16;
  int act;                 // of the gate: 0 SiLU, 1 sigmoid, 2 none
};
constexpr int kBlockNormMaxK = 32768;
// vec = 4, 2 or 1 divides K and all rows are aligned to vec elements.
const char* launch_block_norm(const BlockNormArgs& a, int vec, cudaStream_t st);

struct TokenLogprobArgs {
  const void* logits;      // [T, V] bf16 or f32
  int64_t ld;
  const int* tokens;       // [T], -1: none (null: none at all)
  float *logprob, *entropy;   // [T]
  float* top_lp;           // [T, k]
  int* top_id;             // [T, k]
  int T, V, k;
  int* err;
};
constexpr int kLogprobMaxTop = 32;
void launch_token_logprobs(const TokenLogprobArgs& a, bool f32, cudaStream_t st);

}  // namespace air
