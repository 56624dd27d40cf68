// Checks that the torch <-> kernel adapters share.
#pragma once
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <string>
#include <utility>

namespace air_bind {

using at::Tensor;
using c10::optional;

// Numbers enter messages through std::to_string: formatting them with a string stream inside the
// extension crashed with this image's torch and libstdc++.
inline std::string str(int64_t n) { return std::to_string(n); }

inline void same_device(const Tensor& t, const Tensor& as, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == as.device(), what, " must be on the same CUDA device as the first operand");
}
inline void post(const char* what) {
  cudaError_t e = cudaGetLastError();
  TORCH_CHECK(e == cudaSuccess, what, ": ", cudaGetErrorString(e));
}
// Rows of an output (two or three dimensions) share no memory: expanded or interleaved ones would be written by
// several blocks at once.
inline void distinct_rows(const Tensor& t, const char* op, const char* what) {
  const auto sizes = t.sizes(), strides = t.strides();
  const int last = (int)sizes.size() - 1;
  int a = 0, b = last - 1;                            // the outer dimension and the next
  if (sizes[b] > 1 && (sizes[a] <= 1 || strides[a] < strides[b])) std::swap(a, b);
  const int64_t inner = sizes[b] > 1 && b != a ? (sizes[b] - 1) * strides[b] : 0;
  const bool ok = (sizes[b] <= 1 || b == a || strides[b] >= sizes[last]) &&
                  (sizes[a] <= 1 || strides[a] >= inner + sizes[last]);
  TORCH_CHECK(ok || t.numel() == 0, op, ": the rows of ", what, " overlap or interleave in memory");
}
// The caller's output, or a new one.
inline Tensor or_new(const optional<Tensor>& out, at::IntArrayRef sizes, const Tensor& as, at::ScalarType type) {
  if (out.has_value()) return *out;
  TORCH_CHECK(as.is_cuda(), "the operands must be CUDA tensors");
  return at::empty(sizes, as.options().dtype(type));
}

}  // namespace air_bind
