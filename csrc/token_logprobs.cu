// Log probabilities from logits, one pass over a row:
//   lse = log sum_v exp(x_v),  logprob = x_token - lse,  entropy = lse - sum_v p_v x_v,
// and the k most likely tokens (ties: the lowest index first).
//
// A block (or a cluster of blocks, with few rows) streams its row in 16-byte accesses. Each thread keeps s = sum exp(d) and
// e = sum d exp(d) for d = x - ref, ref being its largest logit so far: four vectors are summed by themselves around the new
// maximum, then the sums before are moved there and added, so the exponential and four paired operations are what two
// elements cost, and a favourite's term, next to which small ones round, meets only a vector's worth of them and then
// sums. The threads' sums are f32, joined around the row's maximum: entropy = log s - e / s. Infinities below count as
// -1e30, whose exponential is an exact zero.
//
// The alternatives need no second pass over the row: the k-th largest of the threads' maxima is at most the k-th largest
// logit, so only the k threads whose maximum reaches it can hold one. Their elements (k / threads of the row, from L2) are
// read again by the whole block, the few that reach the bound are collected and ordered. A row with fewer than k logits
// above -1e29 is swept once more, for finite ones below.
//
// Memory-bound with many long rows: 2048 x 128256 bf16 takes 94 us without alternatives (5.6 TB/s, floor 80), 103 with one,
// 122 with five where every 16th row has three tokens left and is swept twice. One row of f32 takes 6.1 us without and 10.5 with 20.
#include <cooperative_groups.h>

#include "state_space.cuh"

namespace air {

namespace {

namespace cg = cooperative_groups;

constexpr float kMasked = -1e30f;          // stands for -inf in the sums
constexpr float kAllLow = -1e29f;          // a row whose maximum is below takes the plain path

using Key = unsigned long long;
// Order of the alternatives as one number: the value's bits mapped to rising unsigned ones, then the index inverted.
// Zeros of both signs are alike.
AIR_DEVICE uint32_t rank_bits(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
AIR_DEVICE Key rank_key(float v, int i) { return (Key)rank_bits(v) << 32 | (uint32_t)~i; }
AIR_DEVICE float key_value(Key k) {
  const uint32_t b = (uint32_t)(k >> 32);
  return __uint_as_float(b ^ (b >> 31 ? 0x80000000u : 0xffffffffu));
}
AIR_DEVICE int key_index(Key k) { return (int)~(uint32_t)k; }

// 16 bytes of a row as f32, infinities below as kMasked, NaN kept.
template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int E = 8;
  __nv_bfloat162 v[4];
  AIR_DEVICE void load(const __nv_bfloat16* p) {
    const uint4 u = ld_stream(p);
    v[0] = *reinterpret_cast<const __nv_bfloat162*>(&u.x);
    v[1] = *reinterpret_cast<const __nv_bfloat162*>(&u.y);
    v[2] = *reinterpret_cast<const __nv_bfloat162*>(&u.z);
    v[3] = *reinterpret_cast<const __nv_bfloat162*>(&u.w);
  }
  AIR_DEVICE void load_part(const __nv_bfloat16* p, int lo, int hi) {
    __nv_bfloat16 t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = i >= lo && i < hi ? p[i] : __float2bfloat16_rn(-INFINITY);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __nv_bfloat162(t[2 * i], t[2 * i + 1]);
  }
  AIR_DEVICE void clamp() {
    const __nv_bfloat162 m = __float2bfloat162_rn(kMasked);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __hmax2_nan(v[i], m);
  }
  AIR_DEVICE float max() const {
    const __nv_bfloat162 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  AIR_DEVICE void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u = *reinterpret_cast<const uint32_t*>(&v[i]);
      f[2 * i] = __uint_as_float(u << 16);
      f[2 * i + 1] = __uint_as_float(u & 0xffff0000u);
    }
  }
};
template <>
struct Vec<float> {
  static constexpr int E = 4;
  float v[4];
  AIR_DEVICE void load(const float* p) {
    const uint4 u = ld_stream(p);
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  }
  AIR_DEVICE void load_part(const float* p, int lo, int hi) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i >= lo && i < hi ? p[i] : -INFINITY;
  }
  AIR_DEVICE void clamp() {
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(v[i]) : "f"(kMasked));
  }
  AIR_DEVICE float max() const { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); }
  AIR_DEVICE void get(float (&f)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = v[i];
  }
};

// A row as aligned vectors: vector i holds elements i E - off .. of the row.
template <typename T>
struct Row {
  static constexpr int E = Vec<T>::E;
  const T* base;                           // 16-byte aligned, at or before the first element
  int off, V, vectors;
  AIR_DEVICE Row(const T* x, int n) : V(n) {
    off = (int)(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    base = x - off;
    vectors = (int)(((int64_t)n + off + E - 1) / E);
  }
  AIR_DEVICE Vec<T> operator()(int i) const {
    Vec<T> r;
    const int64_t first = (int64_t)i * E - off;
    if (first >= 0 && first + E <= V) r.load(base + (int64_t)i * E);
    else r.load_part(base + (int64_t)i * E, first < 0 ? off : 0, (int)min((int64_t)E, V - first));
    return r;
  }
};

struct Sums {
  float ref, s, e;                         // s = sum exp(d), e = sum d exp(d) for d = x - ref
  AIR_DEVICE void move(float to) {         // to >= ref
    const float d = ref - to, f = ref == -INFINITY ? 0.f : exp2f(d * kLog2e);
    e = f == 0.f ? 0.f : f * fmaf(d, s, e);      // d s may pass f32 where nothing is left
    s *= f;
    ref = to;
  }
};

template <typename T, int NT>
struct LpSmem {
  static constexpr int Keep = 256, Cap = Keep + NT * Vec<T>::E;    // a round of collect_rounds adds at most a vector a thread
  Key keys[Cap], best[kLogprobMaxTop];
  float maxima[NT];
  short chosen[NT];
  Sums warp[NT / 32], total, joined;
  float red[32];
  float bound;
  int count, n_chosen;
};

// keys[0 .. n) -> the k largest in order in best (0 where there are fewer): each key's place is the number of larger ones
template <int NT>
AIR_DEVICE void largest(const Key* keys, int n, int k, Key* best) {
  if (threadIdx.x < k) best[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const Key mine = keys[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += keys[j] > mine;
    if (above < k) best[above] = mine;
  }
  __syncthreads();
}

// A bound that at least k of NT values reach and hardly more: the k-th largest, rounded down to 16 bits. By one warp.
template <int NT>
AIR_DEVICE float kth_largest(const float* v, int k) {
  uint32_t mine[NT / 32], bound = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) mine[i] = rank_bits(v[(threadIdx.x & 31) + 32 * i]);
  for (int b = 31; b >= 16; --b) {
    const uint32_t t = bound | 1u << b;
    int n = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) n += mine[i] >= t;
    if (__reduce_add_sync(0xffffffffu, n) >= k) bound = t;
  }
  return __uint_as_float(bound ^ (bound >> 31 ? 0x80000000u : 0xffffffffu));
}

// The sums of up to 32 lanes, in all lanes.
AIR_DEVICE Sums warp_join(Sums r) {
  const float m = warp_max(r.ref);
  if (m > r.ref) r.move(m);
  return {m, warp_sum(r.s), warp_sum(r.e)};
}

// The sums of a row by one block, element by element around its true maximum, for rows that the stand-in for -inf would
// change: all logits below -1e29.
template <typename T, int NT>
__device__ Sums low_row(const T* x, int V, float* red) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += NT) m = fmaxf(m, to_f(x[i]));
  m = block_max(m, red);
  float s = 0.f, e = 0.f;
  for (int i = threadIdx.x; i < V && m > -INFINITY; i += NT) {
    const float u = to_f(x[i]) - m, p = expf(u);
    s += p;
    if (p > 0.f) e = fmaf(p, u, e);
  }
  s = block_sum(s, red);
  __syncthreads();
  e = block_sum(e, red);
  return {m, s, e};
}

// Collects the elements of the vectors at(0 .. items) that `take` wants into sm.keys, which may hold some already; never
// more than the k largest and a round's worth at a time. By the whole block.
template <typename T, int NT, class At, class Take>
__device__ __noinline__ void collect_rounds(LpSmem<T, NT>& sm, const Row<T>& row, int k, int items, At at, Take take) {
  constexpr int E = Vec<T>::E;
  Key above = 0;
  for (int w0 = 0; w0 < items; w0 += NT) {
    const int i = w0 + (int)threadIdx.x < items ? at(w0 + threadIdx.x) : -1;
    if (i >= 0) {
      float f[E];
      row(i).get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const Key key = rank_key(f[j], i * E - row.off + j);
        if (take(f[j]) && key > above) sm.keys[atomicAdd(&sm.count, 1)] = key;
      }
    }
    __syncthreads();
    const int n = sm.count;
    if (n > LpSmem<T, NT>::Keep) {                   // keep the k largest, and look for larger ones only
      largest<NT>(sm.keys, n, k, sm.best);
      above = sm.best[k - 1];
      if (threadIdx.x < k) sm.keys[threadIdx.x] = sm.best[threadIdx.x];
      if (threadIdx.x == 0) sm.count = k;
    }
    __syncthreads();
  }
}
// The same in one go, several vectors in flight and no barriers, and in rounds only if there are too many to hold.
template <typename T, int NT, class At, class Take>
AIR_DEVICE void collect(LpSmem<T, NT>& sm, const Row<T>& row, int k, int items, At at, Take take) {
  constexpr int E = Vec<T>::E, U = 4;
  const int before = sm.count;
  __syncthreads();
  for (int w0 = threadIdx.x; w0 < items; w0 += NT * U) {
    Vec<T> v[U];
    int i[U];
    bool whole = true;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      i[u] = w0 + u * NT < items ? at(w0 + u * NT) : -1;
      whole &= i[u] > 0 && i[u] < row.vectors - 1;
    }
    if (whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u].load(row.base + (int64_t)i[u] * E);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i[u] >= 0) v[u] = row(i[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i[u] < 0) continue;
      float f[E];
      v[u].get(f);
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) any |= take(f[j]);
      if (!any) continue;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        if (!take(f[j])) continue;
        const int n = atomicAdd(&sm.count, 1);
        if (n < LpSmem<T, NT>::Cap) sm.keys[n] = rank_key(f[j], i[u] * E - row.off + j);
      }
    }
  }
  __syncthreads();
  const int n = sm.count;
  __syncthreads();
  if (n > LpSmem<T, NT>::Cap) {
    if (threadIdx.x == 0) sm.count = before;
    __syncthreads();
    collect_rounds<T, NT>(sm, row, k, items, at, take);
  }
}

template <typename T, int NT, int CS>
__global__ void __launch_bounds__(NT) token_logprobs_kernel(const TokenLogprobArgs a) {
  using V = Vec<T>;
  constexpr int E = V::E, U = 4;                     // vectors in flight
  extern __shared__ __align__(16) uint8_t raw_smem[];
  LpSmem<T, NT>& sm = *reinterpret_cast<LpSmem<T, NT>*>(raw_smem);
  const int rank = CS > 1 ? (int)cg::this_cluster().block_rank() : 0;
  const int64_t t = blockIdx.x / CS;
  const Row<T> row(static_cast<const T*>(a.logits) + t * a.ld, a.V);
  const int per = (row.vectors + CS - 1) / CS;
  const int v0 = min(row.vectors, rank * per), v1 = min(row.vectors, v0 + per);

  float ref = kMasked;                               // the largest logit so far
  f2 s2 = 0ull, e2 = 0ull;                           // the sums in two halves
  auto join = [&]() {
    float s0, s1, e0, e1;
    unpack2(s2, s0, s1);
    unpack2(e2, e0, e1);
    return Sums{ref, s0 + s1, e0 + e1};
  };
  auto add = [&](V (&v)[U]) {
    float to = ref;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      v[j].clamp();
      to = fmaxf(to, v[j].max());
    }
    f2 gs = 0ull, ge = 0ull;
    const f2 back = dup2(-to);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float f[E];
      v[j].get(f);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const f2 d = add2(pack2(f[i], f[i + 1]), back);
        float u0, u1;
        unpack2(mul2(d, dup2(kLog2e)), u0, u1);
        const f2 p = pack2(exp2_fast(u0), exp2_fast(u1));
        gs = add2(gs, p);
        ge = fma2(d, p, ge);
      }
    }
    const float d = fmaxf(ref - to, -1000.f);        // far enough to be nothing, and d s stays in f32
    const f2 f = dup2(exp2_fast(d * kLog2e));
    e2 = fma2(f, fma2(dup2(d), s2, e2), ge);
    s2 = fma2(f, s2, gs);
    ref = to;
  };
  // whole vectors, several in flight; then what is left of them with one of the two at the row's ends, which may hold fewer
  // elements
  const int w0 = v0 + (v0 == 0), w1 = v1 - (v1 == row.vectors && v1 > w0);
  const T* p = row.base + (int64_t)(w0 + threadIdx.x) * E;
  int i = w0 + threadIdx.x;
  for (; i + (U - 1) * NT < w1; i += U * NT, p += U * NT * E) {
    V v[U];
#pragma unroll
    for (int j = 0; j < U; ++j) v[j].load(p + j * NT * E);
    add(v);
  }
  const int end = threadIdx.x == 0 && w0 > v0 && v1 > v0 ? v0 : threadIdx.x == NT - 1 && w1 < v1 ? w1 : -1;
  if (i < w1 || end >= 0) {
    V v[U];
#pragma unroll
    for (int j = 0; j < U - 1; ++j) {
      if (i + j * NT < w1) v[j].load(p + j * NT * E);
      else v[j].load_part(p, 0, 0);
    }
    if (end >= 0) v[U - 1] = row(end);
    else v[U - 1].load_part(p, 0, 0);
    add(v);
  }

  // ---- the block's maximum and sums, and a bound of its k largest
  {
    const Sums w = warp_join(join());
    if ((threadIdx.x & 31) == 0) sm.warp[threadIdx.x >> 5] = w;
    sm.maxima[threadIdx.x] = ref;
    if (threadIdx.x == 0) sm.n_chosen = sm.count = 0;
  }
  __syncthreads();
  if (a.k && threadIdx.x < 32) {
    const float b = kth_largest<NT>(sm.maxima, a.k);
    if (threadIdx.x == 0) sm.bound = fmaxf(b, kAllLow);
  } else if (threadIdx.x >= NT - 32) {
    const int lane = threadIdx.x & 31;
    const Sums w = warp_join(lane < NT / 32 ? sm.warp[lane] : Sums{-INFINITY, 0.f, 0.f});
    if (lane == 0) sm.total = w;
  }
  __syncthreads();

  // ---- the block's k largest
  if (a.k) {
    const float bound = sm.bound;
    if (ref >= bound) sm.chosen[atomicAdd(&sm.n_chosen, 1)] = (short)threadIdx.x;
    __syncthreads();
    const int each = (w1 - w0 + NT - 1) / NT + 1;    // a thread's vectors; the last place is for one of the row's ends
    collect<T, NT>(sm, row, a.k, sm.n_chosen * each,
                   [=, &sm](int w) {
                     const int who = sm.chosen[w / each], j = w % each, at = w0 + who + j * NT;
                     if (j < each - 1) return at < w1 ? at : -1;
                     return who == 0 && w0 > v0 && v1 > v0 ? v0 : who == NT - 1 && w1 < v1 ? w1 : -1;
                   },
                   [=](float f) { return f >= bound; });
    if (sm.count < a.k)                              // fewer than k: what is finite and lower still, if there is any
      collect<T, NT>(sm, row, a.k, v1 - v0, [=](int w) { return v0 + w; }, [=](float f) { return f < bound && f > -INFINITY; });
    largest<NT>(sm.keys, sm.count, a.k, sm.best);
  }

  // ---- the cluster's
  Sums all = sm.total;
  if constexpr (CS > 1) {
    auto cluster = cg::this_cluster();
    cluster.sync();
    if (rank == 0) {
      if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const Sums w = warp_join(lane < CS ? cluster.map_shared_rank(&sm, lane % CS)->total : Sums{-INFINITY, 0.f, 0.f});
        if (lane == 0) sm.joined = w;
      }
      for (int w = threadIdx.x; w < CS * a.k; w += NT) sm.keys[w] = cluster.map_shared_rank(&sm, w / a.k)->best[w % a.k];
      __syncthreads();
      all = sm.joined;
    }
    cluster.sync();                                  // the others' memory was read until here
    if (rank != 0) return;
    if (a.k) largest<NT>(sm.keys, CS * a.k, a.k, sm.best);
  }
  const bool nan = !(all.s < INFINITY);
  const int tok = a.tokens ? a.tokens[t] : -1;
  if (threadIdx.x == 0 && (tok < -1 || tok >= a.V)) set_error(a.err, kErrBounds);
  if (!nan && all.ref <= kAllLow) all = low_row<T, NT>(row.base + row.off, a.V, sm.red);
  const bool none = all.ref == -INFINITY;            // nothing is allowed
  const float ls = logf(all.s);
  auto logprob = [&](float v) { return nan ? NAN : v == -INFINITY ? -INFINITY : v - all.ref - ls; };
  if (threadIdx.x == 0) {
    a.logprob[t] = tok < 0 || tok >= a.V ? 0.f : logprob(to_f(row.base[row.off + (int64_t)tok]));
    a.entropy[t] = nan ? NAN : none ? 0.f : ls - all.e / all.s;
  }
  if (threadIdx.x < a.k) {
    const Key b = nan ? 0 : sm.best[threadIdx.x];
    a.top_id[t * a.k + threadIdx.x] = b ? key_index(b) : -1;
    a.top_lp[t * a.k + threadIdx.x] = nan ? NAN : b ? logprob(key_value(b)) : -INFINITY;
  }
}

template <typename T, int NT, int CS>
void launch(const TokenLogprobArgs& a, cudaStream_t st) {
  static unsigned long long done = 0;
  constexpr int bytes = sizeof(LpSmem<T, NT>);
  set_max_smem_per_device(token_logprobs_kernel<T, NT, CS>, bytes, done);
  cudaLaunchConfig_t c{};
  c.gridDim = dim3((unsigned)a.T * CS);
  c.blockDim = dim3(NT);
  c.dynamicSmemBytes = bytes;
  c.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {CS, 1, 1};
  c.attrs = &at;
  c.numAttrs = CS > 1 ? 1 : 0;
  cudaLaunchKernelEx(&c, token_logprobs_kernel<T, NT, CS>, a);
}

template <typename T>
void choose(const TokenLogprobArgs& a, cudaStream_t st) {
  // Blocks of 256 threads fill the device at four or five an SM. Rows that leave room are cut among clusters of up to 8 blocks (1
  // row of 128256: 10.5 us against 18.4 by one block; 100 rows: 16 against 27), or taken by larger blocks (400 rows: 39.7
  // against 40.3). Many short rows leave most threads of a block idle in the selection: 20000 x 5000 takes 85 us
  // with 64 threads, 112 with 128 and 199 with 256, 4000 x 16000 takes 50, 48 and 64; 300 x 10000 10.1, 8.2 and 8.8.
  const int64_t room = 148 * 5, vectors = a.V / Vec<T>::E;
  if (vectors <= 1024 && a.T > 1024) launch<T, 64, 1>(a, st);
  else if (vectors <= 2048 && a.T > 1024) launch<T, 128, 1>(a, st);
  else if (vectors <= 2048) launch<T, 256, 1>(a, st);
  else if (a.T * 8 <= room) launch<T, 256, 8>(a, st);
  else if (a.T * 4 <= room) launch<T, 256, 4>(a, st);
  else if (a.T * 2 <= room) launch<T, 256, 2>(a, st);
  else if (a.T <= 148 * 3) launch<T, 512, 1>(a, st);
  else launch<T, 256, 1>(a, st);
}

}  // namespace

void launch_token_logprobs(const TokenLogprobArgs& a, bool f32, cudaStream_t st) {
  if (a.T == 0) return;
  if (f32) choose<float>(a, st);
  else choose<__nv_bfloat16>(a, st);
}

}  // namespace air
