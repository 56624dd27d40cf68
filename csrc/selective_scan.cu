// Selective state-space scan over packed sequences:
//   delta = softplus(dt + bias),  h[d, n] = exp(delta A[d, n]) h[d, n] + delta x B[n],
//   y[d] = (sum_n C[n] h[d, n] + D[d] x[d]) silu(z[d])
// h, delta, the sums and the gate stay f32; y is rounded once. The state is f32 in memory.
#include <algorithm>

#include "state_space.cuh"

namespace air {

namespace {

constexpr int kTokThreads = 128;

// One token after the other, for any shape: more than 64 states, calls of short sequences, single tokens whose rows are not
// aligned. L lanes share a channel, S states each (the states of a lane are consecutive, so the lanes of a channel read its
// whole row of the pool). A warp works on 32 / L channels. Latency-bound: 0.8 us a token with 16 states of up to 1536
// channels and 128 of 1024, 1.4 with 16 of 4096 and 200 of 2048, which the tiles avoid.
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
      h[i] = decayed(delta * A[i], h[i], dx, b);
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

// Single tokens, `rows` of them a thread with A and the channel's parameters kept; the states of a lane are whole accesses
// (N a multiple of 4 or 8, aligned rows). 128 x 8192 with 16 states takes 33.6 us at a floor of 21.9: instructions, of
// which the work of a channel (step, gate, addresses) is shared by eight states a lane (four: 46 us). Up to four rows a
// thread (one: 57 us with four states a lane); two rows in flight cost more registers than they gain (44 us).
template <typename T, int L, int S>
__global__ void __launch_bounds__(kTokThreads) scan_step_kernel(const ScanArgs a, int blocks_d, int rows) {
  const int q = threadIdx.x % L, n0 = blockIdx.x / blocks_d * rows, n1 = min(n0 + rows, a.seq.N);
  const int d = (blockIdx.x % blocks_d) * (kTokThreads / L) + threadIdx.x / L;
  const bool live = d < a.D;
  const int dd = live ? d : 0;                 // idle lanes compute channel 0 and write nothing
  const int64_t g = dd / (a.D / a.G);
  const bool mine = q * S < a.N;               // the lane has states
  f2 A[S / 2];
  {
    float v[S] = {};
    if (mine) load_v<float, S>(a.A + (int64_t)dd * a.N + q * S, v);
#pragma unroll
    for (int i = 0; i < S / 2; ++i) A[i] = pack2(v[2 * i] * kLog2e, v[2 * i + 1] * kLog2e);
  }
  const float bias = a.dt_bias ? a.dt_bias[dd] : 0.f, skip = a.skip ? a.skip[dd] : 0.f;
  for (int64_t n = n0; n < n1; ++n) {
    const int64_t slot = state_row(a.seq, (int)n, d == 0);
    float* st = slot >= 0 ? a.state + (slot * a.D + dd) * a.N + q * S : nullptr;
    const float x = to_f(static_cast<const T*>(a.x)[n * a.xs + dd]);
    float delta = to_f(static_cast<const T*>(a.dt)[n * a.ds + dd]) + bias;
    const float z = a.z ? to_f(static_cast<const T*>(a.z)[n * a.zs + dd]) : 0.f;
    float h[S] = {}, B[S] = {}, C[S] = {};
    if (mine) {
      load_v<T, S>(static_cast<const T*>(a.B) + n * a.bs_t + g * a.bs_g + q * S, B);
      load_v<T, S>(static_cast<const T*>(a.C) + n * a.cs_t + g * a.cs_g + q * S, C);
      if (st) load_v<float, S>(st, h);
    }
    if (a.softplus) delta = softplus_f(delta);
    const float dx = delta * x;
    const f2 step = dup2(delta);
    f2 y2 = 0ull;
#pragma unroll
    for (int i = 0; i < S / 2; ++i) {
      float u0, u1;
      unpack2(mul2(step, A[i]), u0, u1);
      h[2 * i] = decayed(u0, h[2 * i], dx, B[2 * i]);
      h[2 * i + 1] = decayed(u1, h[2 * i + 1], dx, B[2 * i + 1]);
      y2 = fma2(pack2(C[2 * i], C[2 * i + 1]), pack2(h[2 * i], h[2 * i + 1]), y2);
    }
    float y, y_;
    unpack2(y2, y, y_);
    y += y_;
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (!live) continue;
    if (st && mine) store_v<float, S>(st, h);
    if (q == 0) {
      y = fmaf(skip, x, y);
      if (a.z) y *= silu_f(z);
      static_cast<T*>(a.out)[n * a.os + d] = from_f<T>(st ? y : 0.f);
    }
  }
}

template <typename T>
void steps(const ScanArgs& a, cudaStream_t st) {
#define AIR_STEP(L, S)                                                                                         \
  {                                                                                                            \
    const int64_t bd = (a.D + kTokThreads / L - 1) / (kTokThreads / L);                                        \
    const int64_t per = std::min<int64_t>(4, std::max<int64_t>(1, a.seq.N * bd / (148 * 16)));                \
    scan_step_kernel<T, L, S><<<(unsigned)(bd * ((a.seq.N + per - 1) / per)), kTokThreads, 0, st>>>(a, (int)bd, (int)per); \
  }
  // eight states a lane where they come in eights: what a lane does for its channel is shared by more of them
  if (a.N <= 4) AIR_STEP(1, 4)
  else if (a.N == 8) AIR_STEP(1, 8)
  else if (a.N == 12) AIR_STEP(4, 4)
  else if (a.N == 16) AIR_STEP(2, 8)
  else if (a.N <= 32 && a.N % 8 == 0) AIR_STEP(4, 8)
  else if (a.N <= 32) AIR_STEP(8, 4)
  else if (a.N <= 64 && a.N % 8 == 0) AIR_STEP(8, 8)
  else if (a.N <= 64) AIR_STEP(16, 4)
  else if (a.N <= 128) AIR_STEP(32, 4)
  else AIR_STEP(32, 8)
#undef AIR_STEP
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
  const int e = f32 ? 4 : 2, S = a.N > 128 || a.N % 8 == 0 ? 8 : 4;
  auto ok = [](const void* p, int64_t st, int64_t sg, int bytes, int size) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && st * size % bytes == 0 && sg * size % bytes == 0;
  };
  const bool vec = a.N % S == 0 && ok(a.A, 0, 0, 16, 4) && ok(a.state, 0, 0, 16, 4) && ok(a.B, a.bs_t, a.G > 1 ? a.bs_g : 0, S * e > 16 ? 16 : S * e, e) &&
                   ok(a.C, a.cs_t, a.G > 1 ? a.cs_g : 0, S * e > 16 ? 16 : S * e, e);
  if (a.seq.step && vec) {
    if (f32) steps<float>(a, st);
    else steps<__nv_bfloat16>(a, st);
    return;
  }
  if (f32) tokens<float>(a, st);
  else tokens<__nv_bfloat16>(a, st);
}

}  // namespace air
