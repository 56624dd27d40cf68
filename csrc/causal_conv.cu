// Short causal depthwise convolution over packed sequences:
//   y[t, d] = act(b[d] + sum_j w[d, j] x[t - W + 1 + j, d]),   W = 2 .. 4
// where the W - 1 inputs before a sequence's first token are those of its state row (or zeros); the row then gets the
// sequence's last W - 1 inputs. Sums stay f32 and are rounded once; the state holds inputs, unrounded.
//
// One launch has two kinds of blocks. Token runs: R consecutive packed tokens of a block of channels slide a window
// over x; they write the tokens that have their W - 1 predecessors in their own sequence, so they need no state.
// Sequences: the first W - 1 tokens and the state row, read and replaced by the same threads, so no block reads a row
// that another writes. x is read once but for W - 1 rows a run. Memory-bound: two element sizes of traffic for
// 2 W + 5 operations and two special functions.
#include "state_space.cuh"

namespace air {

namespace {

constexpr int kConvThreads = 128;
constexpr int kConvRun = 32;       // tokens a run, a bit each of a warp's vote

template <typename T, int W, int V>
struct Taps {
  float w[W][V], b[V];
  AIR_DEVICE Taps(const ConvArgs& a, int d) {
    float flat[V * W];
    if constexpr (V == 1) {
#pragma unroll
      for (int i = 0; i < W; ++i) flat[i] = a.w[(int64_t)d * W + i];
    } else {
#pragma unroll
      for (int i = 0; i < V * W; i += 4) load_v<float, 4>(a.w + (int64_t)d * W + i, flat + i);
    }
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) w[j][v] = flat[v * W + j];
    if (a.bias) {
      if constexpr (V == 1) b[0] = a.bias[d];
      else {
#pragma unroll
        for (int i = 0; i < V; i += 4) load_v<float, 4>(a.bias + d + i, b + i);
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) b[v] = 0.f;
    }
  }
  // rows[0 .. W - 1]: the token's window, oldest first
  template <class Row>
  AIR_DEVICE void apply(Row rows, int silu, T* out) const {
    float y[V];
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = b[v];
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = fmaf(w[j][v], rows(j)[v], y[v]);
    if (silu) {
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = silu_f(y[v]);
    }
    store_v<T, V>(out, y);
  }
};

// The first W - 1 tokens of sequence n and its state row, V channels a thread.
template <typename T, int W, int V>
AIR_DEVICE void conv_sequence(const ConvArgs& a, int n, int d) {
  constexpr int H = W - 1;
  const SeqRange s = seq_range(a.seq, n);
  if (d >= a.D) return;
  const T* x = static_cast<const T*>(a.x) + d;
  T* out = static_cast<T*>(a.out) + d;
  T* row = s.slot >= 0 ? static_cast<T*>(a.state) + s.slot * H * (int64_t)a.D + d : nullptr;
  if (a.seq.step && !row) {
    float zero[V] = {};
    for (int t = s.t0; t < s.t1; ++t) store_v<T, V>(out + t * a.os, zero);
    return;
  }
  const int len = s.t1 - s.t0;
  // ext: the state's rows, then the first H tokens
  float ext[2 * H][V], last[H][V];
#pragma unroll
  for (int i = 0; i < 2 * H; ++i) {
    const T* p = i < H ? (s.init ? row + (int64_t)i * a.D : nullptr) : i - H < len ? x + (int64_t)(s.t0 + i - H) * a.xs : nullptr;
    if (p) load_v<T, V>(p, ext[i]);
    else {
#pragma unroll
      for (int v = 0; v < V; ++v) ext[i][v] = 0.f;
    }
  }
  if (row) {
#pragma unroll
    for (int i = 0; i < H; ++i) {
      if (len >= H) load_v<T, V>(x + (int64_t)(s.t1 - H + i) * a.xs, last[i]);
      else {
#pragma unroll
        for (int k = 0; k < H; ++k) {                 // ext[len + i], with the index known to the compiler
          if (len == k) {
#pragma unroll
            for (int v = 0; v < V; ++v) last[i][v] = ext[k + i][v];
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < H; ++i) store_v<T, V>(row + (int64_t)i * a.D, last[i]);
  }
  const Taps<T, W, V> taps(a, d);
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (i < len) taps.apply([&](int j) -> const float* { return ext[i + j]; }, a.silu, out + (int64_t)(s.t0 + i) * a.os);
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const ConvArgs a, int blocks_d, int runs) {
  const int bd = blockIdx.x % blocks_d, unit = blockIdx.x / blocks_d;
  const int d = (bd * kConvThreads + threadIdx.x) * V;
  if (unit >= runs) {
    conv_sequence<T, W, V>(a, unit - runs, d);
    return;
  }
  constexpr int H = W - 1, B = 4;                 // rows in flight
  const int t0 = unit * kConvRun;
  const unsigned mask = tokens_inside<W>(a.seq, t0);
  if (d >= a.D || !mask) return;
  const T* x = static_cast<const T*>(a.x) + d;
  T* out = static_cast<T*>(a.out) + d;
  const Taps<T, W, V> taps(a, d);
  float win[H + B][V];
  auto row = [&](int t, float* f) {
    if (t >= 0 && t < a.seq.T) load_v<T, V>(x + (int64_t)t * a.xs, f);
    else {
#pragma unroll
      for (int v = 0; v < V; ++v) f[v] = 0.f;
    }
  };
#pragma unroll
  for (int i = 0; i < H; ++i) row(t0 - H + i, win[i]);
  for (int r = 0; r < kConvRun; r += B) {
    if (!(mask >> r)) return;
#pragma unroll
    for (int i = 0; i < B; ++i) row(t0 + r + i, win[H + i]);
#pragma unroll
    for (int i = 0; i < B; ++i)
      if (mask >> (r + i) & 1)
        taps.apply([&](int j) -> const float* { return win[i + j]; }, a.silu, out + (int64_t)(t0 + r + i) * a.os);
#pragma unroll
    for (int i = 0; i < H; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) win[i][v] = win[B + i][v];
  }
}

template <typename T, int W, int V>
const char* launch(const ConvArgs& a, cudaStream_t st) {
  const int64_t blocks_d = (a.D + (int64_t)kConvThreads * V - 1) / (kConvThreads * V);
  const int64_t runs = a.seq.step ? 0 : (a.seq.T + (int64_t)kConvRun - 1) / kConvRun;
  const int64_t grid = blocks_d * (runs + a.seq.N);
  if (grid >= (1ll << 31)) return "causal_conv: too many tokens, sequences or channels for one call";
  if (grid) causal_conv_kernel<T, W, V><<<(unsigned)grid, kConvThreads, 0, st>>>(a, (int)blocks_d, (int)runs);
  return nullptr;
}

}  // namespace

const char* launch_causal_conv(const ConvArgs& a, bool f32, bool vec, cudaStream_t st) {
#define AIR_CONV(N)                                                                               \
  if (a.W == N) return f32 ? (vec ? launch<float, N, 4>(a, st) : launch<float, N, 1>(a, st))      \
                           : (vec ? launch<__nv_bfloat16, N, 8>(a, st) : launch<__nv_bfloat16, N, 1>(a, st));
  AIR_CONV(2)
  AIR_CONV(3)
  AIR_CONV(4)
#undef AIR_CONV
  return "causal_conv: 2 to 4 taps";
}

}  // namespace air
