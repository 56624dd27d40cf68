// Log probabilities from logits, one pass a row:
//   lse = log sum_v exp(x_v),  logprob = x_token - lse,  entropy = lse - sum_v p_v x_v,
// and the k most likely tokens (ties: the lowest index first). Sums stay f32 around the row's maximum.
#include "state_space.cuh"

namespace air {

namespace {

constexpr int kLpThreads = 256;

// Order of the alternatives as one number: the value's bits mapped to rising unsigned ones, then the index inverted.
AIR_DEVICE unsigned long long rank_key(float v, int i) {
  const uint32_t b = __float_as_uint(v);
  return (unsigned long long)(b ^ (b >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~i;
}
AIR_DEVICE float key_value(unsigned long long k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xffffffffu));
}

AIR_DEVICE unsigned long long block_max_key(unsigned long long v, unsigned long long* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kLpThreads / 32; ++w) v = max(v, red[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const TokenLogprobArgs a) {
  __shared__ float red[32];
  __shared__ unsigned long long redk[kLpThreads / 32];
  const int64_t t = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + t * a.ld;
  float m = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < a.V; i += kLpThreads) {
    const float v = to_f(x[i]);
    nan |= v != v || v == INFINITY;
    m = fmaxf(m, v);
  }
  m = block_max(m, red);
  nan = __syncthreads_or(nan);
  const bool none = m == -INFINITY;
  float s = 0.f, e = 0.f;
  for (int i = threadIdx.x; i < a.V; i += kLpThreads) {
    const float u = to_f(x[i]) - m, p = expf(u);
    s += p;
    if (p > 0.f) e = fmaf(p, u, e);
  }
  s = block_sum(s, red);
  __syncthreads();
  e = block_sum(e, red);
  const float ls = logf(s);
  auto logprob = [&](float v) { return nan ? NAN : v == -INFINITY ? -INFINITY : v - m - ls; };
  if (threadIdx.x == 0) {
    const int tok = a.tokens ? a.tokens[t] : -1;
    if (tok < -1 || tok >= a.V) set_error(a.err, kErrBounds);
    a.logprob[t] = tok < 0 || tok >= a.V ? 0.f : logprob(to_f(x[tok]));
    a.entropy[t] = nan ? NAN : none ? 0.f : ls - e / s;
  }
  unsigned long long below = ~0ull;
  for (int r = 0; r < a.k; ++r) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < a.V && !nan; i += kLpThreads) {
      const float v = to_f(x[i]);
      const unsigned long long key = v == -INFINITY ? 0 : rank_key(v == 0.f ? 0.f : v, i);
      if (key < below) best = max(best, key);
    }
    below = best = block_max_key(best, redk);
    if (threadIdx.x == 0) {
      a.top_id[t * a.k + r] = best ? (int)~(uint32_t)best : -1;
      a.top_lp[t * a.k + r] = nan ? NAN : best ? logprob(key_value(best)) : -INFINITY;
    }
  }
}

}  // namespace

void launch_token_logprobs(const TokenLogprobArgs& a, bool f32, cudaStream_t st) {
  if (a.T == 0) return;
  if (f32) token_logprobs_kernel<float><<<a.T, kLpThreads, 0, st>>>(a);
  else token_logprobs_kernel<__nv_bfloat16><<<a.T, kLpThreads, 0, st>>>(a);
}

}  // namespace air
