// Short causal depthwise convolution over packed sequences:
//   y[t, d] = act(b[d] + sum_j w[d, j] x[t - W + 1 + j, d]),   W = 2 .. 4
// where the W - 1 inputs before a sequence's first token are those of its state row (or zeros); the row then gets the
// sequence's last W - 1 inputs. Sums stay f32 and are rounded once; the state holds inputs, unrounded.
//
// A prompt launch has two kinds of blocks. Token runs: R consecutive packed tokens of a block of channels slide a window
// over x; they write the tokens that have their W - 1 predecessors in their own sequence, so they need no state.
// Sequences: the first W - 1 tokens and the state row, read and replaced by the same threads, so no block reads a row
// that another writes. x is read once but for W - 1 rows a run. Memory-bound: two element sizes of traffic for
// 2 W + 5 operations and two special functions; the arithmetic runs on pairs of channels (f32x2).
// 16384 x 8192 bf16 with two, three and four taps takes 87, 92 and 100 us (5.4 TB/s and more, floor 82; f32 8192 x 8192 85, 86
// and 87 us). Rows that are not whole 16-byte parts go in pairs or element by element: 163, 166 and 195 us in pairs, 182 to 193
// in single elements.
#include "state_space.cuh"

namespace air {

namespace {

constexpr int kConvThreads = 128;
constexpr int kConvRun = 32;       // tokens a run, a bit each of a warp's vote
constexpr int kGroups = 4;         // groups of rows in the ring

// V channels of a row as they lie in memory, and as pairs of f32 (one channel: a pair whose second half is unused).
template <typename T, int V>
struct alignas(V * sizeof(T)) Raw {
  T v[V];
};
template <int V>
struct Chan {
  static constexpr int P = (V + 1) / 2;
  f2 p[P];
  AIR_DEVICE void zero() {
#pragma unroll
    for (int i = 0; i < P; ++i) p[i] = 0ull;
  }
  template <typename T>
  AIR_DEVICE void from(const Raw<T, V>& r) {
#pragma unroll
    for (int i = 0; i < P; ++i) p[i] = pack2(to_f(r.v[2 * i]), V > 1 ? to_f(r.v[V > 1 ? 2 * i + 1 : 0]) : 0.f);
  }
};
template <typename T, int V>
AIR_DEVICE Raw<T, V> no_row() {
  Raw<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = from_f<T>(0.f);
  return r;
}

template <typename T, int W, int V>
struct Taps {
  Chan<V> w[W], b;
  AIR_DEVICE Taps(const ConvArgs& a, int d) {
    float flat[V * W], bias[V];
    if constexpr (V > 1 && V * W % 4 == 0) load_v<float, V * W>(a.w + (int64_t)d * W, flat);
    else {
#pragma unroll
      for (int i = 0; i < V * W; ++i) flat[i] = a.w[(int64_t)d * W + i];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias ? a.bias[d + v] : 0.f;
#pragma unroll
    for (int i = 0; i < Chan<V>::P; ++i) {
      const int c0 = 2 * i, c1 = V > 1 ? 2 * i + 1 : 0;
#pragma unroll
      for (int j = 0; j < W; ++j) w[j].p[i] = pack2(flat[c0 * W + j], flat[c1 * W + j]);
      b.p[i] = pack2(bias[c0], bias[c1]);
    }
  }
  // win(0 .. W - 1): the token's window, oldest first
  template <class Win>
  AIR_DEVICE void apply(Win win, int silu, T* out) const {
    Raw<T, V> r;
#pragma unroll
    for (int i = 0; i < Chan<V>::P; ++i) {
      f2 y = b.p[i];
#pragma unroll
      for (int j = 0; j < W; ++j) y = fma2(w[j].p[i], win(j).p[i], y);
      if (silu) y = silu2(y);
      float y0, y1;
      unpack2(y, y0, y1);
      r.v[2 * i] = from_f<T>(y0);
      if (V > 1) r.v[V > 1 ? 2 * i + 1 : 0] = from_f<T>(y1);
    }
    *reinterpret_cast<Raw<T, V>*>(out) = r;
  }
};

// The first W - 1 tokens of sequence n and its state row, V channels a thread.
template <typename T, int W, int V>
AIR_DEVICE void conv_sequence(const ConvArgs& a, int n, int d) {
  using R = Raw<T, V>;
  constexpr int H = W - 1;
  const SeqRange s = seq_range(a.seq, n);
  if (d >= a.D) return;
  const T* x = static_cast<const T*>(a.x) + d;
  T* out = static_cast<T*>(a.out) + d;
  T* row = s.slot >= 0 ? static_cast<T*>(a.state) + s.slot * H * (int64_t)a.D + d : nullptr;
  const int len = s.t1 - s.t0;
  const Taps<T, W, V> taps(a, d);
  // ext: the state's rows, then the first H tokens
  R ext[2 * H];
#pragma unroll
  for (int i = 0; i < 2 * H; ++i) {
    const T* p = i < H ? (s.init ? row + (int64_t)i * a.D : nullptr) : i - H < len ? x + (int64_t)(s.t0 + i - H) * a.xs : nullptr;
    ext[i] = p ? *reinterpret_cast<const R*>(p) : no_row<T, V>();
  }
  if (row) {
    R last[H];
#pragma unroll
    for (int i = 0; i < H; ++i) {
      if (len >= H) last[i] = *reinterpret_cast<const R*>(x + (int64_t)(s.t1 - H + i) * a.xs);
      else {
#pragma unroll
        for (int k = 0; k < H; ++k)                   // ext[len + i], with the index known to the compiler
          if (len == k) last[i] = ext[k + i];
      }
    }
#pragma unroll
    for (int i = 0; i < H; ++i) *reinterpret_cast<R*>(row + (int64_t)i * a.D) = last[i];
  }
  Chan<V> f[2 * H];
#pragma unroll
  for (int i = 0; i < 2 * H; ++i) f[i].from(ext[i]);
#pragma unroll
  for (int i = 0; i < H; ++i)
    if (i < len) taps.apply([&](int j) -> const Chan<V>& { return f[i + j]; }, a.silu, out + (int64_t)(s.t0 + i) * a.os);
}

// Single tokens, one a block: everything is asked for at once but for the state's row, whose number is read first.
// 256 x 8192 bf16 takes 9.0 us at a floor of 5.2 (several rows a thread, which read the taps once for all of them: 11.3;
// eight channels a thread: 15.6).
template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads) conv_step_kernel(const ConvArgs a, int blocks_d) {
  using R = Raw<T, V>;
  constexpr int H = W - 1;
  const int d = (blockIdx.x % blocks_d * kConvThreads + threadIdx.x) * V, n = blockIdx.x / blocks_d;
  if (d >= a.D) return;
  const Taps<T, W, V> taps(a, d);
  const int64_t slot = state_row(a.seq, n, d == 0);
  T* out = static_cast<T*>(a.out) + (int64_t)n * a.os + d;
  if (slot < 0) {
    *reinterpret_cast<R*>(out) = no_row<T, V>();
    return;
  }
  T* row = static_cast<T*>(a.state) + slot * H * (int64_t)a.D + d;
  R ext[W];
#pragma unroll
  for (int i = 0; i < H; ++i) ext[i] = *reinterpret_cast<const R*>(row + (int64_t)i * a.D);
  ext[H] = *reinterpret_cast<const R*>(static_cast<const T*>(a.x) + (int64_t)n * a.xs + d);
  Chan<V> f[W];
#pragma unroll
  for (int i = 0; i < W; ++i) f[i].from(ext[i]);
  taps.apply([&](int j) -> const Chan<V>& { return f[j]; }, a.silu, out);
#pragma unroll
  for (int i = 0; i < H; ++i) *reinterpret_cast<R*>(row + (int64_t)i * a.D) = ext[i + 1];
}

template <typename T, int W, int V>
__global__ void __launch_bounds__(kConvThreads, 4) causal_conv_kernel(const ConvArgs a, int blocks_d, int runs) {
  using R = Raw<T, V>;
  const int bd = blockIdx.x % blocks_d, unit = blockIdx.x / blocks_d;
  const int d = (bd * kConvThreads + threadIdx.x) * V;
  if (unit >= runs) {
    conv_sequence<T, W, V>(a, unit - runs, d);
    return;
  }
  // B rows a group. Whole 16-byte parts of rows are copied asynchronously, kGroups - 1 groups ahead, into a ring of shared
  // memory that is each thread's own, so nothing waits for other threads; narrower parts go through registers.
  constexpr bool async = V * sizeof(T) == 16;
  constexpr int H = W - 1, B = async ? 4 : 8, groups = kConvRun / B;
  __shared__ R ring[async ? kGroups : 1][async ? B : 1][kConvThreads];
  const int t0 = unit * kConvRun;
  const T* x = static_cast<const T*>(a.x) + d + (int64_t)t0 * a.xs;
  auto row = [&](int i) { return t0 + i >= 0 && t0 + i < a.seq.T ? *reinterpret_cast<const R*>(x + i * a.xs) : no_row<T, V>(); };
  R next[async ? 1 : B];
  Chan<V> win[H + B];
  auto fetch = [&](int g) {
    if constexpr (async) {
#pragma unroll
      for (int i = 0; i < B; ++i)
        if (g < groups && t0 + g * B + i < a.seq.T) copy_async<16>(&ring[g % kGroups][i][threadIdx.x], x + (g * B + i) * a.xs, true);
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else if (g < groups) {
#pragma unroll
      for (int i = 0; i < B; ++i) next[i] = row(g * B + i);
    }
  };
  if (d < a.D) {
#pragma unroll
    for (int g = 0; g < (async ? kGroups - 1 : 1); ++g) fetch(g);
#pragma unroll
    for (int i = 0; i < H; ++i) win[i].from(row(i - H));
  }
  const unsigned mask = tokens_inside<W>(a.seq, t0);
  if (d >= a.D) return;
  T* out = static_cast<T*>(a.out) + d + (int64_t)t0 * a.os;
  const Taps<T, W, V> taps(a, d);
  for (int g = 0; g < groups && mask >> g * B; ++g) {
    if constexpr (async) {
      fetch(g + kGroups - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
    }
#pragma unroll
    for (int i = 0; i < B; ++i) win[H + i].from(async ? ring[g % kGroups][i][threadIdx.x] : next[async ? 0 : i]);
    if constexpr (!async) fetch(g + 1);
#pragma unroll
    for (int i = 0; i < B; ++i)
      if (mask >> (g * B + i) & 1)
        taps.apply([&](int j) -> const Chan<V>& { return win[i + j]; }, a.silu, out + (int64_t)(g * B + i) * a.os);
#pragma unroll
    for (int i = 0; i < H; ++i) win[i] = win[B + i];
  }
  if constexpr (async) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int W, int V>
const char* launch(const ConvArgs& a, cudaStream_t st) {
  const int64_t blocks_d = (a.D + (int64_t)kConvThreads * V - 1) / (kConvThreads * V);
  const int64_t runs = a.seq.step ? 0 : (a.seq.T + (int64_t)kConvRun - 1) / kConvRun;
  const int64_t grid = blocks_d * (runs + a.seq.N);
  if (grid >= (1ll << 31)) return "causal_conv: too many tokens, sequences or channels for one call";
  if (!grid) return nullptr;
  if (a.seq.step) conv_step_kernel<T, W, V><<<(unsigned)grid, kConvThreads, 0, st>>>(a, (int)blocks_d);
  else causal_conv_kernel<T, W, V><<<(unsigned)grid, kConvThreads, 0, st>>>(a, (int)blocks_d, (int)runs);
  return nullptr;
}

}  // namespace

const char* launch_causal_conv(const ConvArgs& a, bool f32, int vec, cudaStream_t st) {
#define AIR_CONV_V(N, T) return vec * sizeof(T) >= 16 && !a.seq.step ? launch<T, N, 16 / sizeof(T)>(a, st) : vec >= 4 ? launch<T, N, 4>(a, st) : vec == 2 ? launch<T, N, 2>(a, st) : launch<T, N, 1>(a, st)
#define AIR_CONV(N)                     \
  if (a.W == N) {                       \
    if (f32) AIR_CONV_V(N, float);      \
    AIR_CONV_V(N, __nv_bfloat16);       \
  }
  AIR_CONV(2)
  AIR_CONV(3)
  AIR_CONV(4)
#undef AIR_CONV
#undef AIR_CONV_V
  return "causal_conv: 2 to 4 taps";
}

}  // namespace air
