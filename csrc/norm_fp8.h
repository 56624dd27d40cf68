#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace air {

struct AddNormF8Args {
  const float* x;          // [T, K] f32 residual stream
  const void* y;           // [T, K] bf16 or f32 addend (null: none)
  int y_bf16;
  const float* w;          // [K] norm weight
  float w_offset, eps;
  float* resid;            // [T, K] x + y (null: not written; may be x)
  void* out_bf16;          // [T, K] the norm's output (null: not written)
  uint8_t* xq;             // [T, K] E4M3 codes
  float* xs;               // [T] scale of each row
  int64_t ldx, ldy, ldr, ldo;
  int T, K;
};

constexpr int kAddNormMaxK = 32768;
// K a multiple of 8, rows of x / resid 16-byte and of y / codes 8-byte aligned. null on success.
const char* launch_add_rmsnorm_fp8(const AddNormF8Args& a, cudaStream_t st);

}  // namespace air
