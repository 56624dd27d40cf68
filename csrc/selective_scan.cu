// Selective state-space scan over packed sequences:
//   delta = softplus(dt + bias),  h[d, n] = exp(delta A[d, n]) h[d, n] + delta x B[n],
//   y[d] = (sum_n C[n] h[d, n] + D[d] x[d]) silu(z[d])
// h, delta, the sums and the gate stay f32; y is rounded once. The state is f32 in memory.
#include "state_space.cuh"

namespace air {

namespace {

constexpr int kTokThreads = 128;

// One token after the other, for single tokens and any shape: L lanes share a channel, S states each (the states of a
// lane are consecutive, so the lanes of a channel read its whole row of the pool). A warp works on 32 / L channels.
// Single tokens are bound by the pool: 8 bytes a state against a dozen instructions.
template <typename T, int L, int S>
__global__ void __launch_bounds__(kTokThreads) scan_tokens_kernel(const ScanArgs a, int blocks_d) {
  const int n = blockIdx.x / blocks_d;
  const int q = threadIdx.x % L;
  const int d = (blockIdx.x % blocks_d) * (kTokThreads / L) + threadIdx.x / L;
  const SeqRange s = seq_range(a.seq, n);
  const bool live = d < a.D;
  const int dd = live ? d : 0;                 // idle lanes compute channel 0 and write nothing
  const T* x = static_cast<const T*>(a.x) + dd;
  const T* dt = static_cast<const T*>(a.dt) + dd;
  const T* z = a.z ? static_cast<const T*>(a.z) + dd : nullptr;
  T* out = static_cast<T*>(a.out) + dd;
  float* st = s.slot >= 0 ? a.state + (s.slot * a.D + dd) * a.N : nullptr;
  if (a.seq.step && !st) {
    if (live && q == 0)
      for (int t = s.t0; t < s.t1; ++t) out[t * a.os] = from_f<T>(0.f);
    return;
  }
  const int64_t g = dd / (a.D / a.G);
  const T* B = static_cast<const T*>(a.B) + g * a.bs_g;
  const T* C = static_cast<const T*>(a.C) + g * a.cs_g;
  const bool whole = a.N % 4 == 0 && reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
  float A[S], h[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    const int c = q * S + i;
    A[i] = c < a.N ? a.A[(int64_t)dd * a.N + c] * kLog2e : 0.f;
    h[i] = 0.f;
  }
  if (s.init) {
#pragma unroll
    for (int i = 0; i < S; i += 4) {
      const int c = q * S + i;
      if (whole && c < a.N) load_v<float, 4>(st + c, h + i);
      else if (!whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < a.N) h[i + j] = st[c + j];
      }
    }
  }
  const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f, skip = a.skip ? a.skip[dd] : 0.f;
  for (int t = s.t0; t < s.t1; ++t) {
    const float xv = to_f(x[t * a.xs]);
    float delta = to_f(dt[t * a.ds]) + bias;
    if (a.softplus) delta = softplus_f(delta);
    const float dx = delta * xv;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int c = q * S + i;
      const float b = c < a.N ? to_f(B[t * a.bs_t + c]) : 0.f;
      const float cc = c < a.N ? to_f(C[t * a.cs_t + c]) : 0.f;
      h[i] = fmaf(decay_m1(delta * A[i]), h[i], fmaf(dx, b, h[i]));
      y = fmaf(cc, h[i], y);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (live && q == 0) {
      y = fmaf(skip, xv, y);
      if (z) y *= silu_f(to_f(z[t * a.zs]));
      out[t * a.os] = from_f<T>(y);
    }
  }
  if (st && live) {
#pragma unroll
    for (int i = 0; i < S; i += 4) {
      const int c = q * S + i;
      if (whole && c < a.N) store_v<float, 4>(st + c, h + i);
      else if (!whole) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < a.N) st[c + j] = h[i + j];
      }
    }
  }
}

template <typename T>
void tokens(const ScanArgs& a, cudaStream_t st) {
#define AIR_SCAN(L, S)                                                                 \
  {                                                                                    \
    const int bd = (a.D + kTokThreads / L - 1) / (kTokThreads / L);                    \
    scan_tokens_kernel<T, L, S><<<(unsigned)bd * a.seq.N, kTokThreads, 0, st>>>(a, bd); \
  }
  if (a.N <= 4) AIR_SCAN(1, 4)
  else if (a.N <= 8) AIR_SCAN(2, 4)
  else if (a.N <= 16) AIR_SCAN(4, 4)
  else if (a.N <= 32) AIR_SCAN(8, 4)
  else if (a.N <= 64) AIR_SCAN(16, 4)
  else if (a.N <= 128) AIR_SCAN(32, 4)
  else AIR_SCAN(32, 8)
#undef AIR_SCAN
}

}  // namespace

void launch_scan_tokens(const ScanArgs& a, bool f32, cudaStream_t st) {
  if (a.seq.N == 0) return;
  if (f32) tokens<float>(a, st);
  else tokens<__nv_bfloat16>(a, st);
}

}  // namespace air
