// Selective scan of packed prompts in tiles of tokens.
//   h = exp(delta A) h + delta x B,   y = (C . h + D x) silu(z)
//
// What bounds it: one exponential per token, channel and state (a warp's exponential takes 8 clocks of its scheduler, a
// paired multiply-add 2, both measured), against 8 bytes a token and channel: 64 channels of a token with 16 states are 33 ns
// of an SM's exponentials and 12 ns of its share of the memory bandwidth. So the special-function, multiply-add and issue
// slots are what counts: 8192 x 8192 x 16 bf16 takes 657 us where the exponentials alone would take 231 and the
// bytes 82; issue slots are busy 61 % on average (108 SMs have two blocks, 40 have one), the multiply-add pipe 51 %.
//
// A block has as many scan warps as helper warps, four of each (two blocks an SM). L lanes share a pair of channels, each
// with two states of both: the arithmetic runs on pairs of channels (f32x2), so the steps of a pair are one operand and y
// of the pair comes out as one. Stage by stage of TS tokens, through two sets of buffers, the helpers turn dt and x of the
// next stages into delta and delta x, and the lanes' parts of y of the last one into the output (sum, skip, gate,
// rounding), so all global accesses are theirs, copied asynchronously up to three stages ahead. Before the helpers, with each
// scan warp loading its own rows, the case above took 11.9 ms; with the helpers' loads through registers 1.45.
//
// The tokens of all sequences lie in one row of tiles of equal length; a block walks through its tile and loads or
// stores a state where a sequence starts or ends, so ragged batches are balanced. With few channels there are several
// tiles: a first pass then computes what each tile's last sequence adds to the next tile (the state from zero, or from the
// sequence's initial state, and the sum of delta), and the second pass starts from exp(A sum) times those of the tiles before.
// That pass adds 0.65 of the work over sequences that cross tiles, so the host cuts no more than pays (scan_plan).
// Up to 64 states; more go token by token (selective_scan.cu).
#include <algorithm>

#include "state_space.cuh"

namespace air {

namespace {

// What 2^u h + in (decayed) takes of M pairs, step by step over all of them: e = 2^u and p = (2^u - 1) / u beside slow decays. M
// independent chains, and the exponentials beside them.
template <int M>
AIR_DEVICE void decays(const f2* u, f2* p, f2* e) {
  const f2 c2 = dup2(kDecay2), c1 = dup2(kDecay1), c0 = dup2(kDecay0);
#pragma unroll
  for (int m = 0; m < M; ++m) {
    float ua, ub;
    unpack2(u[m], ua, ub);
    e[m] = pack2(exp2_fast(ua), exp2_fast(ub));
  }
#pragma unroll
  for (int m = 0; m < M; ++m) p[m] = fma2(c2, u[m], c1);
#pragma unroll
  for (int m = 0; m < M; ++m) p[m] = fma2(p[m], u[m], c0);
}
// One state of the pair, by one comparison: what multiplies h, and what of h is added. SELECT: h or zero, which the token's input
// is then added to in the same instruction. Otherwise the sum of h and `in`, the input by itself, whose product does not
// wait for the token before: an instruction more, a step less in the chain through h.
template <bool SELECT>
AIR_DEVICE void choose_decay(float u, float p, float h, float& e, float& in) {
  const bool slow = fabsf(u) <= kNearDecay;
  e = slow ? p * u : e;
  in = SELECT ? (slow ? h : 0.f) : slow ? in + h : in;
}
template <bool SELECT>
AIR_DEVICE f2 decayed2(f2 u, f2 p, f2 e, f2 h, f2 dx, f2 b) {
  float u0, u1, p0, p1, e0, e1, h0, h1, i0, i1;
  unpack2(u, u0, u1);
  unpack2(p, p0, p1);
  unpack2(e, e0, e1);
  unpack2(h, h0, h1);
  if (!SELECT) unpack2(mul2(dx, b), i0, i1);
  choose_decay<SELECT>(u0, p0, h0, e0, i0);
  choose_decay<SELECT>(u1, p1, h1, e1, i1);
  return fma2(pack2(e0, e1), h, SELECT ? fma2(dx, b, pack2(i0, i1)) : pack2(i0, i1));
}
// softplus_f of a pair
AIR_DEVICE f2 softplus2(float a, float b) {
  const f2 u = pack2(exp2_fast(fabsf(a) * -kLog2e), exp2_fast(fabsf(b) * -kLog2e));
  f2 p = fma2(dup2(0.00523269409f), u, dup2(-0.0295052398f));
  p = fma2(p, u, dup2(0.0782259554f));
  p = fma2(p, u, dup2(-0.136632457f));
  p = fma2(p, u, dup2(0.191060066f));
  p = fma2(p, u, dup2(-0.24842982f));
  p = fma2(p, u, dup2(0.333190978f));
  p = fma2(p, u, dup2(-0.499994934f));
  p = fma2(p, u, dup2(0.99999994f));
  return fma2(p, u, pack2(fmaxf(a, 0.f), fmaxf(b, 0.f)));
}

constexpr int kGroup = 2;           // tokens whose decays are computed together
// Hand-over of a stage's buffers: each has a barrier for "prepared" and one for "scanned"; the side that gives arrives,
// the side that takes waits.
template <int THREADS>
AIR_DEVICE void give(int barrier) { asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "n"(THREADS) : "memory"); }
template <int THREADS>
AIR_DEVICE void take(int barrier) { asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(THREADS) : "memory"); }
AIR_DEVICE int prepared(int k) { return 1 + (k & 1); }
AIR_DEVICE int scanned(int k) { return 3 + (k & 1); }

template <int L>
struct Shape {
  // Threads that scan, and as many helpers. Two blocks an SM of 128 + 128, or, where many lanes share a pair and a block of
  // that size would have few channels to share B and C, one of 256 + 256 (8000 x 2048 with 64 states: 590 against 758 us).
  static constexpr int SCAN = L <= 16 ? 128 : 256, HELP = SCAN, THREADS = SCAN + HELP, BLOCKS = 256 / SCAN;
  static constexpr int CH = 2 * SCAN / L, CP = CH / 2;   // channels a block, and pairs
  static constexpr int TS = L <= 4 ? 8 : 16;             // tokens a stage
  static constexpr int NP = 2 * L;                       // states, padded
  static constexpr int E = CH * TS / HELP > 1 ? CH * TS / HELP : 2;   // channels of a helper's access
  static constexpr int HT = CH / E;                      // helpers a token
};
constexpr int kRing = 4, kAhead = 3; // stages of raw rows: up to `kAhead` being fetched, two prepared
template <typename T, int L>
struct Smem {
  using S = Shape<L>;
  static constexpr int BC = S::TS * S::NP * 2 / 4;       // groups of four values of B and C a stage
  alignas(16) float4 step[2][S::TS][S::CP];              // delta of the pair, delta x of the pair
  alignas(16) float4 bc[2][S::TS][L];                    // B and C of a lane's two states
  alignas(16) float2 y[2][S::TS][S::CP * L];             // the lanes' parts of y of the pair
  // x, dt, z: each helper's own part, with room for the words that rows of bf16 at odd addresses start and end in
  static constexpr int W = sizeof(T) == 2 ? 2 * S::E : S::E;
  alignas(16) T rows[kRing][3][S::HELP][W];
  alignas(16) T raw_bc[kRing][BC][4];
};
// Where a pair lies in `step` and a lane's part in `y`: helpers write or read E channels each, and without the exchange
// the eight helpers of a quarter of a warp would all go to the same banks.
template <int E>
AIR_DEVICE int step_slot(int cp) { return cp ^ (cp >> 3 & (E / 2 - 1)); }
template <int L, int E>
AIR_DEVICE int y_slot(int cp, int q) {
  const int i = cp * L + q, helper = cp / (E / 2);
  return i ^ (helper & 7) << 1;
}

// The part of a sequence from token t on: [t, hi) of sequence n, or tokens of no (sound) sequence (n = -1).
struct Segment {
  int n, lo, hi;
};
AIR_DEVICE Segment segment_at(const SeqArgs& a, int t) {
  if (!a.cu) return {0, 0, a.T};
  if (a.N == 0) return {-1, 0, a.T};
  const int n = seq_of_token(a.cu, a.N, t);
  const int lo = a.cu[n], hi = a.cu[n + 1];
  if (t < lo) return {-1, t, min(lo, a.T)};
  if (t >= hi) return {-1, t, a.T};                      // past the last sequence
  if (lo < 0 || hi > a.T) return {-1, t, min(hi, a.T)};
  return {n, lo, hi};
}

struct TileArgs {
  int tiles, tile;         // tiles, tokens of each (the last one may have fewer)
  int blocks_g;            // blocks of channels a group
  float* h;                // [tiles][D][N] what the tile's last sequence leaves for the next tile
  float* init;             // [tiles][D][N] that sequence's initial state, if it starts in the tile
  float* sum;              // [tiles][D] sum of delta over its tokens in the tile
};

// ---- helpers: delta and delta x of a stage, B and C, and the output from y. A helper fetches, prepares and finishes the
// same E channels of the same token of each stage, and the same groups of four values of B and C.
// VEC: its part of a row is one aligned access.
template <typename T, int L, bool FIRST, bool VEC>
struct Helper {
  using S = Shape<L>;
  using M = Smem<T, L>;
  static constexpr int E = S::E, NB = (M::BC + S::HELP - 1) / S::HELP;
  const ScanArgs& a;
  M& sm;
  const int tid, tok, c;            // helper: token of the stage, first channel in the block
  const int live;                   // channels there are from c on, up to E
  const bool vec_bc;                // B and C can be copied in whole accesses
  const int t1;
  int tf, tb[NB];                   // tokens of the next fetch
  const T *x, *dt, *z, *bc[NB];     // and its rows
  T* out;                           // row of the next output
  int64_t bc_stride[NB];
  bool has_bc[NB];                  // padded states have none
  int ring;                         // stages fetched, as a place in the ring
  float bias[E], skip[E];
  int odd[3];                       // where a row's part starts in its first 4-byte word (the same at every stage: TS is even)

  AIR_DEVICE Helper(const ScanArgs& a_, M& s, int64_t d0, int64_t g, int left, bool v, int t0, int end)
      : a(a_), sm(s), tid(threadIdx.x - S::SCAN), tok(tid / S::HT), c(tid % S::HT * E),
        live(tok < S::TS ? max(0, min(E, left - c)) : 0), vec_bc(v), t1(end), tf(t0 + tok), ring(0) {
    const int64_t d = d0 + c;
    x = static_cast<const T*>(a.x) + (int64_t)tf * a.xs + d;
    dt = static_cast<const T*>(a.dt) + (int64_t)tf * a.ds + d;
    z = a.z ? static_cast<const T*>(a.z) + (int64_t)tf * a.zs + d : nullptr;
    out = static_cast<T*>(a.out) + (int64_t)tf * a.os + d;
    odd[0] = odd_half(x);
    odd[1] = odd_half(dt);
    odd[2] = odd_half(z);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      bias[i] = a.dt_bias && i < live ? a.dt_bias[d + i] : 0.f;
      skip[i] = a.skip && i < live ? a.skip[d + i] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {  // four states of a token of B (the first half of the groups) or C
      const int i = tid + S::HELP * j, at = i % (M::BC / 2) * 4, n = at % S::NP;
      const bool is_c = i >= M::BC / 2;
      tb[j] = t0 + at / S::NP;
      bc_stride[j] = is_c ? a.cs_t : a.bs_t;
      bc[j] = static_cast<const T*>(is_c ? a.C : a.B) + tb[j] * bc_stride[j] + g * (is_c ? a.cs_g : a.bs_g) + n;
      has_bc[j] = n < a.N;
    }
  }
  AIR_DEVICE void row(int which, const T* p, const void* any, bool in) {
    T* dst = sm.rows[ring][which][tid];
    if constexpr (VEC) copy_async<E * (int)sizeof(T)>(dst, in ? p : any, in);
    else copy_words<T, E>(dst, p, any, odd[which], in ? live : -8);
  }
  // E elements of a fetched row. Channels past the group's last one get whatever shares their words: nothing of theirs is kept.
  AIR_DEVICE void read(int slot, int which, float* f) const {
    if constexpr (VEC) load_v<T, E>(sm.rows[slot][which][tid], f);
    else read_words<T, E>(sm.rows[slot][which][tid], odd[which], f);
  }
  // The next stage's rows, complete for this helper after arrived() with kAhead - 1 stages fetched after it
  AIR_DEVICE void fetch() {
    const bool in = tf < t1 && live > 0;
    row(0, x, a.x, in);
    row(1, dt, a.dt, in);
    if (!FIRST && a.z) row(2, z, a.z, in);
    tf += S::TS;
    x += S::TS * a.xs;
    dt += S::TS * a.ds;
    z += S::TS * a.zs;
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = tid + S::HELP * j;
      if (i >= (FIRST ? M::BC / 2 : M::BC)) continue;
      const bool in_ = tb[j] < t1 && has_bc[j];
      if (vec_bc) copy_async<4 * (int)sizeof(T)>(sm.raw_bc[ring][i], in_ ? bc[j] : a.B, in_);
      else {
        const int n = i % (M::BC / 2) * 4 % S::NP;
#pragma unroll
        for (int e = 0; e < 4; ++e) sm.raw_bc[ring][i][e] = in_ && n + e < a.N ? bc[j][e] : from_f<T>(0.f);
      }
      tb[j] += S::TS;
      bc[j] += S::TS * bc_stride[j];
    }
    ring = (ring + 1) % kRing;
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  AIR_DEVICE void arrived() { asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory"); }
  // Stage k, `in`: this helper's token is one of the tile's. Tokens past the end change nothing: their step is zero.
  AIR_DEVICE void prepare(int k, bool in) {
    const int slot = k % kRing;
    float xv[E], dv[E];
    read(slot, 0, xv);
    read(slot, 1, dv);
#pragma unroll
    for (int i = 0; i < E && (S::HT * S::TS == S::HELP || tok < S::TS); i += 2) {
      float v = dv[i] + bias[i], w = dv[i + 1] + bias[i + 1];
      if (a.softplus) unpack2(softplus2(v, w), v, w);
      if (!in) v = w = 0.f;
      sm.step[k & 1][tok][step_slot<E>((c + i) / 2)] = make_float4(v, w, v * xv[i], w * xv[i + 1]);
    }
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int i = tid + S::HELP * j;
      if (i >= (FIRST ? M::BC / 2 : M::BC)) continue;
      float f[4];
      load_v<T, 4>(sm.raw_bc[slot][i], f);
      const int which = i / (M::BC / 2), at = i % (M::BC / 2) * 4;
      float2* p = reinterpret_cast<float2*>(&sm.bc[k & 1][at / S::NP][at % S::NP / 2]) + which;
      p[0] = make_float2(f[0], f[1]);
      p[2] = make_float2(f[2], f[3]);
    }
  }
  // The outputs of stage k, for the tokens of the mask
  AIR_DEVICE void finish(int k, unsigned mask) {
    T* o = out;
    out += S::TS * a.os;
    if (live <= 0 || !(mask >> tok & 1)) return;
    const int slot = k % kRing;
    float y[E], f[E], g[E];
    if (a.skip) read(slot, 0, f);
    if (a.z) read(slot, 2, g);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      f2 sum = 0ull;
#pragma unroll
      for (int q = 0; q < L; q += 2) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(&sm.y[k & 1][tok][y_slot<L, E>((c + i) / 2, q)]);
        sum = q ? add2(sum, add2(v.x, v.y)) : add2(v.x, v.y);
      }
      if (a.skip) sum = fma2(pack2(skip[i], skip[i + 1]), pack2(f[i], f[i + 1]), sum);
      if (a.z) sum = mul2(sum, silu2(pack2(g[i], g[i + 1])));
      unpack2(sum, y[i], y[i + 1]);
    }
    if constexpr (VEC) store_v<T, E>(o, y);
    else store_words<T, E>(o, y, live);
  }
};

// ---- scan warps: two states of two channels a lane, as pairs over the channels
template <typename T, int L, bool SELECT>
struct Scan {
  using S = Shape<L>;
  const ScanArgs& a;
  Smem<T, L>& sm;
  const int q, cp;                  // lane among the pair's L, pair in the block
  const int64_t d;                  // first channel
  const int left;                   // channels there are from it on
  const int slot, part;             // of the pair in `step`, of the lane in `y`
  const bool whole;
  f2 A[2], h[2];

  AIR_DEVICE Scan(const ScanArgs& a_, Smem<T, L>& s, int64_t d0, int left_)
      : a(a_), sm(s), q(threadIdx.x % L), cp(threadIdx.x / L), d(d0 + cp * 2), left(left_ - cp * 2), slot(step_slot<S::E>(cp)),
        part(y_slot<L, S::E>(cp, q)), whole(a_.N % 2 == 0 && reinterpret_cast<uintptr_t>(a_.state) % 8 == 0) {
    float v[2][2];
    rows(a.A, v, false);
#pragma unroll
    for (int i = 0; i < 2; ++i) A[i] = pack2(v[0][i] * kLog2e, v[1][i] * kLog2e);
    zero();
  }
  AIR_DEVICE void zero() { h[0] = h[1] = 0ull; }
  // v[channel][state] of [D][N] rows; `al`: the two states of a lane are one aligned access
  AIR_DEVICE void rows(const float* base, float (&v)[2][2], bool al) const {
#pragma unroll
    for (int s_ = 0; s_ < 2; ++s_) {
      const float* p = base + (d + s_) * a.N + q * 2;
      v[s_][0] = v[s_][1] = 0.f;
      if (s_ >= left) continue;
      if (al && q * 2 < a.N) load_v<float, 2>(p, v[s_]);
      else if (!al) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (q * 2 + i < a.N) v[s_][i] = p[i];
      }
    }
  }
  AIR_DEVICE void load(const float* base, bool al) {      // one sequence's rows (of the pool or scratch)
    float v[2][2];
    rows(base, v, al);
    h[0] = pack2(v[0][0], v[1][0]);
    h[1] = pack2(v[0][1], v[1][1]);
  }
  AIR_DEVICE void store(float* base, bool al) const {
    float v[2][2];
    unpack2(h[0], v[0][0], v[1][0]);
    unpack2(h[1], v[0][1], v[1][1]);
#pragma unroll
    for (int s_ = 0; s_ < 2; ++s_) {
      float* p = base + (d + s_) * a.N + q * 2;
      if (s_ >= left) continue;
      if (al && q * 2 < a.N) store_v<float, 2>(p, v[s_]);
      else if (!al) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (q * 2 + i < a.N) p[i] = v[s_][i];
      }
    }
  }
  AIR_DEVICE ulonglong2 step(int buf, int i) const { return *reinterpret_cast<const ulonglong2*>(&sm.step[buf][i][slot]); }
  // K tokens from i on, whose steps are in st: first all their decays (K independent chains a state), then the chains
  // through h. What the chains read, and the next tokens' steps, are loaded before. `sum`: of delta.
  template <bool OUT, int K>
  AIR_DEVICE void tokens(int buf, int i, ulonglong2* st, int next, f2& sum) {
    f2 u[K * 2], p[K * 2], e[K * 2], dx[K];
    float4 c[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      u[k * 2] = mul2(st[k].x, A[0]);
      u[k * 2 + 1] = mul2(st[k].x, A[1]);
      dx[k] = st[k].y;
      if (!OUT) sum = add2(sum, st[k].x);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) c[k] = sm.bc[buf][i + k][q];             // B, B', C, C'
    if (next >= 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) st[k] = step(buf, next + k);
    }
    decays<K * 2>(u, p, e);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      h[0] = decayed2<SELECT>(u[k * 2], p[k * 2], e[k * 2], h[0], dx[k], dup2(c[k].x));
      h[1] = decayed2<SELECT>(u[k * 2 + 1], p[k * 2 + 1], e[k * 2 + 1], h[1], dx[k], dup2(c[k].y));
      if (OUT) *reinterpret_cast<f2*>(&sm.y[buf][i + k][part]) = fma2(dup2(c[k].w), h[1], mul2(dup2(c[k].z), h[0]));
    }
  }
  template <bool OUT>
  AIR_DEVICE void stage(int buf, f2& sum) {
    ulonglong2 st[kGroup];
#pragma unroll
    for (int k = 0; k < kGroup; ++k) st[k] = step(buf, k);
#pragma unroll
    for (int i = 0; i < S::TS; i += kGroup) tokens<OUT, kGroup>(buf, i, st, i + kGroup < S::TS ? i + kGroup : -1, sum);
  }
  template <bool OUT>
  AIR_DEVICE void token(int buf, int i, f2& sum) {
    ulonglong2 st = step(buf, i);
    tokens<OUT, 1>(buf, i, &st, -1, sum);
  }
};

// 2^u h in two steps: with positive rates (or negative steps) 2^u may pass f32 while the product does not, and nothing grows
// to nothing.
AIR_DEVICE float grown(float u, float h) {
  const float half = exp2f(0.5f * u);
  return h == 0.f ? 0.f : h * half * half;
}

AIR_DEVICE bool starts_from(const SeqArgs& a, int n, int64_t& slot) {
  const SeqRange s = seq_range(a, n, false);
  slot = s.slot;
  return s.init;
}

template <typename T, int L, bool FIRST, bool VEC, bool SELECT>
__global__ void __launch_bounds__(Shape<L>::THREADS, Shape<L>::BLOCKS) scan_tiles_kernel(const __grid_constant__ ScanArgs a, const __grid_constant__ TileArgs ta, bool vec_bc) {
  using S = Shape<L>;
  extern __shared__ __align__(16) uint8_t raw_smem[];
  Smem<T, L>& sm = *reinterpret_cast<Smem<T, L>*>(raw_smem);
  const int blocks = ta.blocks_g * a.G;
  const int tile = blockIdx.x / blocks, blk = blockIdx.x % blocks;
  const int per_group = a.D / a.G, grp = blk / ta.blocks_g, first_ch = blk % ta.blocks_g * S::CH;
  const int left = per_group - first_ch;                     // channels of the group from here on
  const int64_t d0 = (int64_t)grp * per_group + first_ch;
  int t0 = tile * ta.tile;
  const int t1 = (int)min((int64_t)a.seq.T, (int64_t)t0 + ta.tile);
  Segment seg;
  if (FIRST) {
    seg = segment_at(a.seq, t1 - 1);
    if (seg.n < 0 || seg.hi <= t1) return;                   // nothing goes on in the next tile
    t0 = max(t0, seg.lo);
  } else {
    seg = segment_at(a.seq, t0);
  }
  const bool idle = !FIRST && seg.n < 0 && seg.hi >= t1;      // no token of the tile is in a sequence
  const int stages = idle ? 0 : (t1 - t0 + S::TS - 1) / S::TS;
  const int64_t row = (int64_t)a.D * a.N;

  if (threadIdx.x >= S::SCAN) {
    Helper<T, L, FIRST, VEC> w(a, sm, d0, grp, left, vec_bc, t0, t1);
    auto next = [&](int k) {                                 // stage k's buffers
      if (k > 0) w.fetch();
      w.arrived();
      w.prepare(k, t0 + k * S::TS + w.tok < t1);
      give<S::THREADS>(prepared(k));
    };
    if (stages > 0) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) w.fetch();
      next(0);
      if (stages > 1) next(1);
    }
    if (!FIRST && a.seq.S > 0) {
      // offsets and rows that are not sound are reported once, empty sequences without a state start one of zeros
      for (int n = tile * S::HELP + w.tid; n < a.seq.N; n += ta.tiles * S::HELP) {
        const SeqRange s = seq_range(a.seq, n, blk == 0);
        if (a.seq.cu && s.slot >= 0 && s.t0 == s.t1 && !s.init)
          for (int64_t i = d0 * a.N; i < (d0 + min(left, S::CH)) * a.N; ++i) a.state[s.slot * row + i] = 0.f;
      }
    } else if (!FIRST && blk == 0) {
      for (int n = tile * S::HELP + w.tid; n < a.seq.N; n += ta.tiles * S::HELP) seq_range(a.seq, n);
    }
    for (int k = 0; k < stages; ++k) {
      const int t = t0 + k * S::TS;
      unsigned mask = ~0u;
      if (!FIRST && (seg.n < 0 || t < seg.lo || t + S::TS > seg.hi)) {
        mask = tokens_inside<1>(a.seq, t);
        seg = segment_at(a.seq, min(t + S::TS, a.seq.T - 1));
      }
      take<S::THREADS>(scanned(k));
      if (!FIRST) w.finish(k, mask & (t + S::TS <= t1 ? ~0u : (1u << (t1 - t)) - 1));
      if (k + 2 < stages) next(k + 2);
    }
    return;
  }

  Scan<T, L, SELECT> w(a, sm, d0, left);
  const bool al = a.N % 2 == 0;                              // scratch is aligned
  auto enter = [&](int t) {                                  // the state before token t of seg
    w.zero();
    if (seg.n < 0) return;
    int64_t slot;
    if (seg.lo == t) {
      if (!starts_from(a.seq, seg.n, slot)) {
        if (FIRST) w.store(ta.init + tile * row, al);
        return;
      }
      // where the sequence ends in another tile, that tile's block may have replaced the pool's row already
      if (!FIRST && ta.tiles > 1 && seg.hi > t1) w.load(ta.init + tile * row, al);
      else w.load(a.state + slot * row, w.whole);
      if (FIRST) w.store(ta.init + tile * row, al);
    } else if (!FIRST && t == tile * ta.tile && tile > 0) {
      f2 acc[2] = {0ull, 0ull};
      float sum[2] = {0.f, 0.f};
      for (int j = tile - 1; j >= 0; --j) {
        w.load(ta.h + j * row, al);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float u, v;
          unpack2(mul2(w.A[i], pack2(sum[0], sum[1])), u, v);
          float a, b;
          unpack2(w.h[i], a, b);
          acc[i] = add2(pack2(grown(u, a), grown(v, b)), acc[i]);
        }
#pragma unroll
        for (int s_ = 0; s_ < 2; ++s_)
          if (s_ < w.left) sum[s_] += ta.sum[(int64_t)j * a.D + w.d + s_];
        if (j * ta.tile <= seg.lo) break;
      }
      w.h[0] = acc[0];
      w.h[1] = acc[1];
    }
  };
  auto leave = [&]() {
    int64_t slot;
    if (seg.n < 0) return;
    starts_from(a.seq, seg.n, slot);
    if (slot >= 0) w.store(a.state + slot * row, w.whole);
  };
  enter(t0);
  float total[2] = {0.f, 0.f}, low[2] = {0.f, 0.f};          // the sum of delta and what its roundings lost
  for (int k = 0; k < stages; ++k) {
    const int t = t0 + k * S::TS;
    take<S::THREADS>(prepared(k));
    f2 sum2 = 0ull;
    if (FIRST || t + S::TS <= seg.hi) {
      w.template stage<!FIRST>(k & 1, sum2);
    } else {
      for (int i = 0; i < S::TS && t + i < t1; ++i) {
        while (t + i >= seg.hi) {
          leave();
          seg = segment_at(a.seq, t + i);
          enter(t + i);
        }
        w.template token<!FIRST>(k & 1, i, sum2);
      }
    }
    float sum[2];
    unpack2(sum2, sum[0], sum[1]);
    if (FIRST) {
#pragma unroll
      for (int s_ = 0; s_ < 2; ++s_) {
        const float n = total[s_] + sum[s_], back = n - total[s_];
        low[s_] += (total[s_] - (n - back)) + (sum[s_] - back);
        total[s_] = n;
      }
    }
    give<S::THREADS>(scanned(k));
  }
  if (FIRST) {
    w.store(ta.h + tile * row, al);
#pragma unroll
    for (int s_ = 0; s_ < 2; ++s_)
      if (w.q == 0 && s_ < w.left) ta.sum[(int64_t)tile * a.D + w.d + s_] = total[s_] + low[s_];
  } else if (seg.hi <= t1) {
    leave();
  }
}

template <int L>
int channel_blocks(const ScanArgs& a) {
  const int per_group = a.D / a.G;
  return (per_group + Shape<L>::CH - 1) / Shape<L>::CH;
}

int lanes_of(int N) { return N <= 8 ? 4 : N <= 16 ? 8 : N <= 32 ? 16 : 32; }

template <typename T, int L, bool VEC>
const char* launch(const ScanArgs& a, const ScanPlan& p, float* ws, bool vec_bc, cudaStream_t st) {
  using S = Shape<L>;
  const int64_t row = (int64_t)a.D * a.N;
  TileArgs ta{p.tiles, p.tile, channel_blocks<L>(a), ws, ws + p.tiles * row, ws + 2 * p.tiles * row};
  const int64_t blocks = (int64_t)ta.blocks_g * a.G;
  if (blocks * p.tiles >= (1ll << 31)) return "selective_scan: too many channels and tokens for one call";
  constexpr int bytes = sizeof(Smem<T, L>);
  static unsigned long long done1 = 0, done2 = 0, done3 = 0;
  constexpr auto first = scan_tiles_kernel<T, L, true, VEC, false>;
  if (p.tiles > 1) {
    if (!set_max_smem_per_device(first, bytes, done1)) return "selective_scan: the device has too little shared memory";
    first<<<(unsigned)(blocks * (p.tiles - 1)), S::THREADS, bytes, st>>>(a, ta, vec_bc);
  }
  // The form of the decay's sum (choose_decay). Eight scan warps on an SM hide its chain, so the shorter form pays: 8192 x
  // 8192 takes 657 us with it and 681 without, 8000 x 2048 with 64 states 590 and 608; with one block an SM 16384 x 4096 takes 840 us
  // with it and 809 without, 8000 x 2048 with 24 states 413 and 389. Up to 8 states it never paid (4000 x 4096: 186 and 184).
  constexpr bool always = L == 32, never = L == 4;
  constexpr auto shorter = scan_tiles_kernel<T, L, false, VEC, !never>, other = scan_tiles_kernel<T, L, false, VEC, always>;
  const bool pays = always || (!never && p.pairs);
  if (!set_max_smem_per_device(pays ? shorter : other, bytes, pays ? done2 : done3))
    return "selective_scan: the device has too little shared memory";
  (pays ? shorter : other)<<<(unsigned)(blocks * p.tiles), S::THREADS, bytes, st>>>(a, ta, vec_bc);
  return nullptr;
}

template <typename T, int L>
const char* launch(const ScanArgs& a, const ScanPlan& p, float* ws, cudaStream_t st) {
  auto ok = [](const void* q, int64_t stride, int bytes) {
    return reinterpret_cast<uintptr_t>(q) % bytes == 0 && stride * (int64_t)sizeof(T) % bytes == 0;
  };
  constexpr int part = Shape<L>::E * sizeof(T) > 16 ? 16 : Shape<L>::E * sizeof(T), four = 4 * sizeof(T);
  const bool rows = a.D / a.G % Shape<L>::E == 0 && ok(a.x, a.xs, part) && ok(a.dt, a.ds, part) && ok(a.out, a.os, part) &&
                    (!a.z || ok(a.z, a.zs, part));
  const bool bc = a.N % 4 == 0 && ok(a.B, a.bs_t, four) && ok(a.C, a.cs_t, four) && (a.G == 1 || (ok(a.B, a.bs_g, four) && ok(a.C, a.cs_g, four)));
  return rows ? launch<T, L, true>(a, p, ws, bc, st) : launch<T, L, false>(a, p, ws, bc, st);
}

}  // namespace

ScanPlan scan_plan(const ScanArgs& a, int sms) {
  const int L = lanes_of(a.N);
  const int64_t per_group = a.D / a.G, ch = L == 4 ? Shape<4>::CH : L == 8 ? Shape<8>::CH : L == 16 ? Shape<16>::CH : Shape<32>::CH;
  const int64_t blocks = (per_group + ch - 1) / ch * a.G;
  // Time of one token with c blocks on the busiest SM: two at once take 1.5 times as long as one (82 against 54 ns with 16
  // states); blocks of 256 + 256 threads have an SM to themselves and count as two. A cut adds a first pass of 0.65 of the
  // work over what crosses tiles: all of a long sequence, less of short ones.
  const bool pairs = L <= 16;
  auto speed = [&](int64_t n) {
    const int64_t c = (n + sms - 1) / sms;
    return pairs ? c / 2 * 1.5 + c % 2 : c * 1.5;
  };
  ScanPlan best{1, a.seq.T, false, 0};
  double cost = a.seq.T * speed(blocks);
  for (int64_t n = 2; n <= 64 && a.seq.T / n >= 64; ++n) {
    const int64_t tile = ((a.seq.T + n - 1) / n + 15) / 16 * 16;
    const int64_t tiles = (a.seq.T + tile - 1) / tile;
    if (tiles < 2) break;
    const double crossing = std::min(1.0, (double)tiles / std::max(1, a.seq.N));
    const double c = tile * speed(blocks * tiles) + 0.65 * crossing * tile * speed(blocks * (tiles - 1)) + 48.0 + tiles;
    if (c < cost) {
      cost = c;
      best = {(int)tiles, (int)tile, false, (int64_t)tiles * a.D * (2 * a.N + 1)};
    }
  }
  best.pairs = blocks * best.tiles > sms;
  return best;
}

// A sequence's start and end cost a walk through a tile 1.2 us (offsets, then the state, one after the other), so calls of
// short sequences go sequence by sequence: 4000 tokens of 4096 channels in sequences of 4 take 643 us here and 663 there,
// in sequences of 8 425 and 596, of 16 312 and 567; 64 sequences of one token 60 and 18. The lengths are on the device: a call
// whose mean is below the limit pays for a long sequence among short ones (4000 tokens with 1000 sequences of one:
// 816 and 5750 us).
bool scan_tiles_worth(const ScanArgs& a) { return a.N <= 64 && a.seq.T >= 6ll * a.seq.N; }

const char* launch_scan_tiles(const ScanArgs& a, const ScanPlan& p, float* ws, bool f32, cudaStream_t st) {
#define AIR_SCAN_L(n) \
  if (lanes_of(a.N) == n) return f32 ? launch<float, n>(a, p, ws, st) : launch<__nv_bfloat16, n>(a, p, ws, st);
  AIR_SCAN_L(4)
  AIR_SCAN_L(8)
  AIR_SCAN_L(16)
  AIR_SCAN_L(32)
#undef AIR_SCAN_L
  return "selective_scan: too many states";
}

}  // namespace air
