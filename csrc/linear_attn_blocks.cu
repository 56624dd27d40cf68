// Linear attention with one decay per head, prompts in blocks of 128 tokens on the tensor cores
// (tcgen05, operands by TMA, accumulators in TMEM).
//
// Within a block, with G_i = g_1 + ... + g_i and the incoming state S (transposed: [dk, dv]):
//   o_i = scale * ( exp(G_i) q_i S  +  sum_{j <= i} exp(G_i - G_j) (q_i k_j) v_j )
//   S'  = exp(G_128) S + sum_j exp(G_128 - G_j) k_j^T v_j
// which is four matrix products a block and head: Q K^T, Q S, P V and W V, with P the masked, decayed
// scores and W the transposed, decayed keys. A CTA walks the blocks of one head one after the other
// with S in registers (f32), so q, k, v are read and o is written once: 4 x 32 KB a block at
// dk = dv = 128.
//
// Roundings: P and the copy of S that Q S reads are bf16 (the outputs are bf16 too; the other operands
// are exact). S itself stays f32: the keys times their f32 decay factors are split into three bf16
// parts that add up to all 24 bits, each block's update is accumulated on its own and added to S in
// registers, because adding it to a long-lived accumulator inside the tensor core would round the
// whole state 24 times a block.
//
// Split over the length: the (sequence, head, block) triples form one list that is cut into one range
// per SM. A sequence longer than two ranges is cut inside; a first kernel computes the state that each
// cut-off piece adds (K and V only), a second one chains these states along the list, and the main
// kernel starts each range from its incoming state. All sums have a fixed order.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <string.h>
#include "common.cuh"
#include "linear_attn.h"
#include "sm100.cuh"

namespace air {

namespace {

using namespace sm100;

constexpr int C = 128;             // tokens per block
constexpr int kMinCut = 4;         // blocks: shorter ranges are not worth a cut
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFloor = -104.f;   // exp(-104) is 0 in f32: one token's decay needs no more

// ---------------------------------------------------------------- the list of blocks and its cuts
struct Pos { int n, h, c; };       // sequence, head, block

AIR_DEVICE int seq_begin(const LinAttnArgs& a, int n) { return a.cu ? a.cu[n] : 0; }
AIR_DEVICE int seq_len(const LinAttnArgs& a, int n) {
  if (!a.cu) return a.T;
  const int t0 = a.cu[n], t1 = a.cu[n + 1];
  if (t0 < 0 || t1 < t0 || t1 > a.T) {
    set_error(a.err, kErrBounds);
    return 0;
  }
  return t1 - t0;
}
AIR_DEVICE int seq_blocks(const LinAttnArgs& a, int n) { return (seq_len(a, n) + C - 1) / C; }
AIR_DEVICE int64_t seq_slot(const LinAttnArgs& a, int n) {
  if (!a.state) return -1;
  const int64_t s = a.slots ? (int64_t)a.slots[n] : (int64_t)n;
  if (s >= a.S) set_error(a.err, kErrBounds);
  return s < 0 || s >= a.S ? -1 : s;
}
AIR_DEVICE bool seq_init(const LinAttnArgs& a, int n) {
  return a.has_state ? a.has_state[n] != 0 : a.has_state_all != 0;
}

struct Range {
  Pos begin, end;                  // end: one past the last block, as the position of the next one
  int blocks;                      // blocks of the range
  int cut_begin, cut_end;          // the range starts / ends inside an item
  int tail;                        // blocks of the last piece when cut_end
};

// The position of list index p (warp-wide), its item's length and the index within the item.
AIR_DEVICE Pos locate(const LinAttnArgs& a, int64_t p, int64_t total, int& len) {
  const int lane = threadIdx.x & 31;
  Pos r{a.N, 0, 0};
  len = 0;
  if (p >= total) return r;
  int64_t base = 0;
  for (int n0 = 0; n0 < a.N; n0 += 32) {
    const int nb = n0 + lane < a.N ? seq_blocks(a, n0 + lane) : 0;
    int64_t inc = (int64_t)nb * a.H;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const int64_t all = __shfl_sync(0xffffffffu, inc, 31);
    if (p < base + all) {
      const unsigned past = __ballot_sync(0xffffffffu, base + inc > p);
      const int l = __ffs(past) - 1;
      const int64_t before = l ? __shfl_sync(0xffffffffu, inc, l ? l - 1 : 0) : 0;
      len = __shfl_sync(0xffffffffu, nb, l);
      const int64_t rel = p - base - before;
      r.n = n0 + l;
      r.h = (int)(rel / len);
      r.c = (int)(rel % len);
      return r;
    }
    base += all;
  }
  return r;
}

// The first position at or after list index p where a range may start: p itself inside an item that
// is cut, else the nearer end of the item (warp-wide). Index and position.
AIR_DEVICE Pos snap(const LinAttnArgs& a, int64_t p, int64_t total, int longest, int64_t& at) {
  int len;
  at = p < total ? p : total;
  Pos r = locate(a, p, total, len);
  if (r.c == 0 || r.n >= a.N || len > longest) return r;
  at += 2 * r.c < len ? -r.c : len - r.c;
  return locate(a, at, total, len);
}

AIR_DEVICE Range make_range(const LinAttnArgs& a, int r, int R) {
  const int lane = threadIdx.x & 31;
  int64_t total = 0;
  int most = 0;
  for (int n = lane; n < a.N; n += 32) {
    const int nb = seq_blocks(a, n);
    total += nb;
    most = max(most, nb);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  most = __reduce_max_sync(0xffffffffu, most);
  total *= a.H;
  int64_t per = (total + R - 1) / R;
  const int longest = (int)(2 * (per > kMinCut ? per : kMinCut));
  if (most > longest && per < kMinCut) per = kMinCut;
  Range g;
  int64_t i0, i1;
  g.begin = snap(a, r * per, total, longest, i0);
  g.end = snap(a, (r + 1) * per, total, longest, i1);
  g.blocks = (int)(i1 - i0);
  g.cut_begin = g.blocks > 0 && g.begin.c > 0;
  g.cut_end = g.blocks > 0 && g.end.n < a.N && g.end.c > 0;
  g.tail = g.cut_end ? min(g.blocks, g.end.c) : 0;
  return g;
}

// Walks blocks of the list in order.
struct Walk {
  const LinAttnArgs& a;
  Pos p;
  int nb, t0, len;
  AIR_DEVICE Walk(const LinAttnArgs& args, const Pos& begin) : a(args), p(begin) { load(); }
  AIR_DEVICE void load() {
    if (p.n < a.N) {
      t0 = seq_begin(a, p.n);
      len = seq_len(a, p.n);
      nb = (len + C - 1) / C;
    }
  }
  AIR_DEVICE int token() const { return t0 + p.c * C; }
  AIR_DEVICE int count() const { return min(C, len - p.c * C); }
  AIR_DEVICE bool last() const { return p.c + 1 == nb; }
  AIR_DEVICE void next() {
    if (++p.c < nb) return;
    p.c = 0;
    if (++p.h < a.H) return;
    p.h = 0;
    do { ++p.n; } while (p.n < a.N && seq_len(a, p.n) == 0);
    load();
  }
};

// ---------------------------------------------------------------- descriptors
// N-contiguous (MN-major) operand in the 128-byte swizzle layout: rows of K are 128 B (64 bf16 of N),
// 8-row atoms 1024 B apart along K (SBO), the next 64 columns of N one panel further (LBO).
AIR_DEVICE uint64_t mn_desc(const void* p, uint32_t panel_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_u32(p) & 0x3FFFF) >> 4);
  d |= (uint64_t)(panel_bytes >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
constexpr uint32_t kBMn = 1u << 16;      // B is N-contiguous

AIR_DEVICE void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
AIR_DEVICE void tma_load_3d(void* dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(dst)), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
AIR_DEVICE uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
AIR_DEVICE float lo_f(uint32_t u) { return __uint_as_float(u << 16); }
AIR_DEVICE float hi_f(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// ---------------------------------------------------------------- shared memory
template <int DK, int DV>
struct Smem {
  static constexpr int kKTile = C * DK * 2, kVTile = C * DV * 2, kSTile = DK * DV * 2;
  static constexpr int kK = 0, kV = 2 * kKTile, kQ = kV + 2 * kVTile, kS = kQ + kKTile, kBars = kS + kSTile;
};
struct alignas(16) Block {         // one block's decays, all from sums within 32 tokens
  float gl[C];                     // log2 of exp(g_1 + ... + g_i) over the token's own 32
  float e[C];                      // exp(g_{j+1} + ... ) up to the end of the token's 32
  float w[C];                      // exp(g_{j+1} + ... + g_128); 0 past the sequence's end
  float t2[4];                     // log2 of the 32s' total decays
  float f;                         // the block's total decay: exp(total), or expm1(total) when slow
  int slow;
};
struct Bars {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], gfull[2], gempty[2];
  uint64_t qfull, qempty;
  uint64_t sc_done, qs_done, o_done, u_done, p_ready, o_scaled, o_free, s_ready, kt_ready[2], kt_free[2], u_free;
  uint32_t tmem;
  int abort;
  Range range;
  Block blk[2];
};

constexpr int kThreads = 512;      // 4 service warps, 4 output warps, 8 state warps
// TMEM columns
constexpr uint32_t kSC = 0, kO = 128, kU = 256;
// the three parts of the transposed keys; buffer 0 shares the upper half of the scores' columns
// (free once P is written), buffer 1 exists in the state-only kernel
__device__ constexpr uint32_t kKT[2][3] = {{384, 448, 64}, {0, 128, 192}};

// STATE: the state-only pass over each range's cut-off last piece.
template <int DK, int DV, bool STATE>
__global__ void __launch_bounds__(kThreads, 1)
linear_blocks_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ LinAttnArgs a,
                     float* __restrict__ ws_state, int4* __restrict__ ws_meta) {
  using M = Smem<DK, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* b = reinterpret_cast<Bars*>(smem + M::kBars);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kKt = STATE ? 2 : 1;     // buffers of the transposed keys

  if (warp == 2) {
    const Range g = make_range(a, blockIdx.x, gridDim.x);
    if (lane == 0) b->range = g;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b->kfull[i], 1);
      mbar_init(&b->kempty[i], 8);
      mbar_init(&b->vfull[i], 1);
      mbar_init(&b->vempty[i], 1);
      mbar_init(&b->gfull[i], 1);
      mbar_init(&b->gempty[i], STATE ? 8 : 12);
      mbar_init(&b->kt_ready[i], 8);
      mbar_init(&b->kt_free[i], 1);
    }
    mbar_init(&b->qfull, 1);
    mbar_init(&b->qempty, 1);
    mbar_init(&b->sc_done, 1);
    mbar_init(&b->qs_done, 1);
    mbar_init(&b->o_done, 1);
    mbar_init(&b->u_done, 1);
    mbar_init(&b->p_ready, 4);
    mbar_init(&b->o_scaled, 4);
    mbar_init(&b->o_free, 4);
    mbar_init(&b->s_ready, 8);
    mbar_init(&b->u_free, 8);
    b->abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&b->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b->tmem;
  const Range rg = b->range;
  Pos begin = rg.begin;
  int nblk = rg.blocks;
  if constexpr (STATE) {
    nblk = rg.tail;
    begin = Pos{rg.end.n, rg.end.h, rg.end.c - rg.tail};
    if (threadIdx.x == 0) ws_meta[blockIdx.x * 2].x = rg.cut_end;
  }
  // a block has an incoming state unless it opens a fresh sequence
  auto incoming = [&](const Walk& w, int i) {
    if constexpr (STATE) return i > 0;
    return w.p.c > 0 || (seq_init(a, w.p.n) && seq_slot(a, w.p.n) >= 0);
  };
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) {    // one thread
    if (ok && !mbar_wait(bar, parity & 1, &b->abort)) {
      ok = false;
      set_error(a.err, kErrTimeout);
      b->abort = 1;
    }
    return ok;
  };
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {   // all lanes give up together
    wait(bar, parity);
    return ok = __all_sync(0xffffffffu, ok);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      Walk w(a, begin);
      int issued = 0;
      for (int i = 0; i < nblk; ++i, w.next()) {
        const int s = i & 1, u = i >> 1;
        const int z = w.token();
        if (i >= 2 && !wait(&b->kempty[s], u - 1)) break;
        mbar_expect_tx(&b->kfull[s], M::kKTile);
#pragma unroll
        for (int p = 0; p < DK / 64; ++p)
          tma_load_3d(smem + M::kK + s * M::kKTile + p * C * 128, &tm_k, &b->kfull[s], 64 * p, w.p.h / a.k_div, z);
        if constexpr (!STATE) {
          if (i >= 1 && !wait(&b->qempty, i - 1)) {
            mbar_wait(&b->kfull[s], u & 1, nullptr, 50ull * 1000 * 1000);
            break;
          }
          mbar_expect_tx(&b->qfull, M::kKTile);
#pragma unroll
          for (int p = 0; p < DK / 64; ++p)
            tma_load_3d(smem + M::kQ + p * C * 128, &tm_q, &b->qfull, 64 * p, w.p.h / a.q_div, z);
        }
        if (i >= 2 && !wait(&b->vempty[s], u - 1)) {
          mbar_wait(&b->kfull[s], u & 1, nullptr, 50ull * 1000 * 1000);
          if (!STATE) mbar_wait(&b->qfull, i & 1, nullptr, 50ull * 1000 * 1000);
          break;
        }
        mbar_expect_tx(&b->vfull[s], M::kVTile);
#pragma unroll
        for (int p = 0; p < DV / 64; ++p)
          tma_load_3d(smem + M::kV + s * M::kVTile + p * C * 128, &tm_v, &b->vfull[s], 64 * p, w.p.h / a.v_div, z);
        issued = i + 1;
      }
      // never leave the CTA with copies in flight into its shared memory
      for (int i = max(0, issued - 2); i < issued; ++i) {
        mbar_wait(&b->kfull[i & 1], (i >> 1) & 1, nullptr, 50ull * 1000 * 1000);
        mbar_wait(&b->vfull[i & 1], (i >> 1) & 1, nullptr, 50ull * 1000 * 1000);
        if (!STATE && i == issued - 1) mbar_wait(&b->qfull, i & 1, nullptr, 50ull * 1000 * 1000);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      constexpr uint32_t id_qk = idesc_bf16_f32(128, C);
      constexpr uint32_t id_mn = idesc_bf16_f32(128, DV) | kBMn;
      Walk w(a, begin);
      int n_in = 0;                      // blocks with an incoming state so far
      for (int i = 0; i < nblk; ++i, w.next()) {
        const int s = i & 1, u = i >> 1;
        const uint8_t* sk = smem + M::kK + s * M::kKTile;
        const uint8_t* sv = smem + M::kV + s * M::kVTile;
        if constexpr (!STATE) {
          const bool in = incoming(w, i);
          // scores = Q K^T (their columns also hold the third key part of the block before)
          if (!wait(&b->kfull[s], u) || !wait(&b->qfull, i)) break;
          if (i >= 1 && !wait(&b->u_done, i - 1)) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < DK / 16; ++ks) {
            const int off = (ks / 4) * C * 128;
            mma_bf16(tmem + kSC, sw128_desc(smem + M::kQ + off) + 2 * (ks & 3), sw128_desc(sk + off) + 2 * (ks & 3),
                     id_qk, ks > 0);
          }
          mma_commit(&b->sc_done);
          if (in) {
            // O = Q S
            if (!wait(&b->s_ready, n_in)) break;
            if (i >= 1 && !wait(&b->o_free, i - 1)) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < DK / 16; ++ks) {
              const int off = (ks / 4) * C * 128;
              mma_bf16(tmem + kO, sw128_desc(smem + M::kQ + off) + 2 * (ks & 3),
                       mn_desc(smem + M::kS + ks * 2048, DK * 128), id_mn, ks > 0);
            }
            mma_commit(&b->qs_done);
          }
          mma_commit(&b->qempty);
          // O (+)= P V
          if (!wait(&b->p_ready, i) || !wait(&b->vfull[s], u)) break;
          if (in ? !wait(&b->o_scaled, n_in) : (i >= 1 && !wait(&b->o_free, i - 1))) break;
          if (in) ++n_in;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < C / 16; ++ks)
            mma_bf16_ts(tmem + kO, tmem + kSC + 8 * ks, mn_desc(sv + ks * 2048, C * 128), id_mn, in || ks > 0);
          mma_commit(&b->o_done);
        } else {
          if (!wait(&b->vfull[s], u)) break;
        }
        // U = W V, the smallest parts first
        const int kb = i % kKt;
        if (!wait(&b->kt_ready[kb], i / kKt)) break;
        if (STATE && i >= 1 && !wait(&b->u_free, i - 1)) break;
        tc_fence_after();
#pragma unroll
        for (int part = 2; part >= 0; --part)
#pragma unroll
          for (int ks = 0; ks < C / 16; ++ks)
            mma_bf16_ts(tmem + kU, tmem + kKT[kb][part] + 8 * ks, mn_desc(sv + ks * 2048, C * 128), id_mn,
                        part < 2 || ks > 0);
        mma_commit(&b->u_done);
        mma_commit(&b->vempty[s]);
        if (STATE) mma_commit(&b->kt_free[kb]);
      }
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------- decays
    // lane l: tokens 4l .. 4l + 3; eight lanes make one of the four 32s
    Walk w(a, begin);
    float total_piece = 0.f;
    for (int i = 0; i < nblk; ++i, w.next()) {
      const int s = i & 1;
      if (i >= 2 && !wait_warp(&b->gempty[s], (i >> 1) - 1)) break;
      const int t0 = w.token(), nt = w.count();
      float g[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * lane + e;
        const float x = j < nt ? a.decay[(int64_t)(t0 + j) * a.decay_t + w.p.h] : 0.f;
        g[e] = x < kFloor ? kFloor : x;
      }
      float pre[4], suf[4];              // inclusive sums up to, exclusive sums after each token, in the 32
      pre[0] = g[0]; pre[1] = pre[0] + g[1]; pre[2] = pre[1] + g[2]; pre[3] = pre[2] + g[3];
      suf[3] = 0.f; suf[2] = g[3]; suf[1] = suf[2] + g[2]; suf[0] = suf[1] + g[1];
      float up = pre[3], down = suf[0] + g[0];
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        const float x = __shfl_up_sync(0xffffffffu, up, o, 8), y = __shfl_down_sync(0xffffffffu, down, o, 8);
        if ((lane & 7) >= o) up += x;
        if ((lane & 7) + o < 8) down += y;
      }
      float after = __shfl_down_sync(0xffffffffu, down, 1, 8);
      if ((lane & 7) == 7) after = 0.f;
      float bef = __shfl_up_sync(0xffffffffu, up, 1, 8);
      if ((lane & 7) == 0) bef = 0.f;
      const float t[4] = {__shfl_sync(0xffffffffu, up, 7), __shfl_sync(0xffffffffu, up, 15),
                          __shfl_sync(0xffffffffu, up, 23), __shfl_sync(0xffffffffu, up, 31)};
      float later = 0.f;                 // the 32s after this one
#pragma unroll
      for (int q = 3; q > 0; --q)
        if (lane / 8 < q) later += t[q];
      Block& k = b->blk[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = 4 * lane + e;
        k.gl[j] = (bef + pre[e]) * kLog2e;
        k.e[j] = expf(suf[e] + after);
        k.w[j] = j < nt ? expf(suf[e] + after + later) : 0.f;
      }
      const float total = (t[3] + t[2]) + (t[1] + t[0]);
      if (lane < 4) k.t2[lane] = (lane == 0 ? t[0] : lane == 1 ? t[1] : lane == 2 ? t[2] : t[3]) * kLog2e;
      if (lane == 0) {
        k.slow = total > -0.5f;
        k.f = k.slow ? expm1f(total) : expf(total);
        total_piece += total;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->gfull[s]);
    }
    if (STATE && lane == 0 && nblk > 0) {
      // the piece's own decay, and whether it opens its sequence
      ws_meta[blockIdx.x * 2].y = __float_as_int(total_piece);
      ws_meta[blockIdx.x * 2].z = begin.c == 0;
      ws_meta[blockIdx.x * 2].w = begin.n;
      ws_meta[blockIdx.x * 2 + 1].x = begin.h;
    }
  } else if (warp >= 4 && warp < 8) {
    // ---------------------------------------------------------------- scores -> P, O -> out
    if constexpr (!STATE) {
      const int q = warp & 3, row = 32 * q + lane;
      const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
      Walk w(a, begin);
      int n_in = 0;
      for (int i = 0; i < nblk; ++i, w.next()) {
        const int s = i & 1, u = i >> 1;
        const bool in = incoming(w, i);
        const int nt = w.count();
        if (!wait_warp(&b->gfull[s], u)) break;
        const Block& k = b->blk[s];
        const float gl = k.gl[row];
        float fb[4];                     // row factor of each earlier 32, and of the incoming state (index q)
        {
          float x = gl;
#pragma unroll
          for (int c = 3; c >= 0; --c) {
            fb[c] = 0.f;
            if (c < q) {
              fb[c] = exp2f(x) * a.scale;
              x += k.t2[c];
            }
          }
          if (!wait_warp(&b->sc_done, i)) break;
          tc_fence_after();
          const float rs = exp2f(x) * a.scale;      // exp(G_i): the incoming state's factor
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
            if (c <= q) {
              float v[32];
              tmem_ld32(trow + kSC + 32 * c, v);
              if (c < q) {
                const float4* e4 = reinterpret_cast<const float4*>(&k.e[32 * c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 e = e4[j];
                  pk[2 * j] = pack_bf16(v[4 * j] * fb[c] * e.x, v[4 * j + 1] * fb[c] * e.y);
                  pk[2 * j + 1] = pack_bf16(v[4 * j + 2] * fb[c] * e.z, v[4 * j + 3] * fb[c] * e.w);
                }
              } else {
                const float4* g4 = reinterpret_cast<const float4*>(&k.gl[32 * c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float4 g = g4[j];
                  const float p0 = 4 * j <= lane ? v[4 * j] * a.scale * exp2f(gl - g.x) : 0.f;
                  const float p1 = 4 * j + 1 <= lane ? v[4 * j + 1] * a.scale * exp2f(gl - g.y) : 0.f;
                  const float p2 = 4 * j + 2 <= lane ? v[4 * j + 2] * a.scale * exp2f(gl - g.z) : 0.f;
                  const float p3 = 4 * j + 3 <= lane ? v[4 * j + 3] * a.scale * exp2f(gl - g.w) : 0.f;
                  pk[2 * j] = pack_bf16(p0, p1);
                  pk[2 * j + 1] = pack_bf16(p2, p3);
                }
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j) pk[j] = 0u;
            }
            tmem_st16(trow + kSC + 16 * c, pk);
          }
          tmem_wait_st();
          if (nt < C) {
            // rows of V past the sequence's end: 0 x whatever they hold must stay 0
            if (!wait_warp(&b->vfull[s], u)) break;
            if (row >= nt) {
#pragma unroll
              for (int p = 0; p < DV / 64; ++p)
#pragma unroll
                for (int c = 0; c < 8; ++c)
                  *reinterpret_cast<uint4*>(smem + M::kV + s * M::kVTile + p * C * 128 + row * 128 + 16 * c) =
                      make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&b->gempty[s]);
            mbar_arrive(&b->p_ready);
          }
          if (in) {
            if (!wait_warp(&b->qs_done, n_in)) break;
            ++n_in;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DV / 32; ++c) {
              float v[32];
              tmem_ld32(trow + kO + 32 * c, v);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                uint32_t r[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) r[j] = __float_as_uint(v[16 * h + j] * rs);
                tmem_st16(trow + kO + 32 * c + 16 * h, r);
              }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->o_scaled);
          }
        }
        if (!wait_warp(&b->o_done, i)) break;
        tc_fence_after();
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (int64_t)(w.token() + row) * a.os_t + (int64_t)w.p.h * a.os_h;
#pragma unroll
        for (int c = 0; c < DV / 32; ++c) {
          float v[32];
          tmem_ld32(trow + kO + 32 * c, v);
          if (c == DV / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->o_free);
          }
          if (row < nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(out + 32 * c + 8 * j) =
                  make_uint4(pack_bf16(v[8 * j], v[8 * j + 1]), pack_bf16(v[8 * j + 2], v[8 * j + 3]),
                             pack_bf16(v[8 * j + 4], v[8 * j + 5]), pack_bf16(v[8 * j + 6], v[8 * j + 7]));
          }
        }
      }
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- transposed keys, state
    // warps 8..11 and 12..15 share the lanes (state columns k); the first four take the first half of
    // the tokens of W and of the state's dv columns, the others the second half
    const int q = warp & 3, half = (warp - 8) >> 2, k0 = 32 * q + lane;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
    constexpr int HV = DV / 2;
    const bool live = k0 < DK;
    float S[HV];
#pragma unroll
    for (int j = 0; j < HV; ++j) S[j] = 0.f;
    Walk w(a, begin);
    for (int i = 0; i < nblk; ++i, w.next()) {
      const int s = i & 1, u = i >> 1;
      const int nt = w.count();
      if constexpr (!STATE) {
        const bool in = incoming(w, i);
        if (w.p.c == 0 || i == 0) {
          // a new piece: its incoming state is the range's (cut), the pool's, or zero. Of a sequence that
          // is cut the chain kernel copied the pool's: the range that ends it may write that row first
          const float* src = nullptr;
          if (w.p.c > 0) src = ws_state + (size_t)(blockIdx.x - 1) * DV * DK;
          else if (in && rg.cut_end && w.p.n == rg.end.n && w.p.h == rg.end.h)
            src = ws_state + (size_t)(gridDim.x + blockIdx.x) * DV * DK;
          else if (in) src = a.state + ((size_t)seq_slot(a, w.p.n) * a.H + w.p.h) * DV * DK;
#pragma unroll
          for (int j = 0; j < HV; ++j) S[j] = src && live ? src[(size_t)(half * HV + j) * DK + k0] : 0.f;
        }
        if (in) {
          // bf16 copy for Q S (the products that read the one before are complete: u_done)
          if (live) {
#pragma unroll
            for (int c = 0; c < HV / 8; ++c) {
              const int v0 = half * HV + 8 * c;
              uint8_t* dst = smem + M::kS + (v0 / 64) * DK * 128 + k0 * 128 + ((((v0 % 64) / 8) ^ (k0 & 7)) << 4);
              *reinterpret_cast<uint4*>(dst) =
                  make_uint4(pack_bf16(S[8 * c], S[8 * c + 1]), pack_bf16(S[8 * c + 2], S[8 * c + 3]),
                             pack_bf16(S[8 * c + 4], S[8 * c + 5]), pack_bf16(S[8 * c + 6], S[8 * c + 7]));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b->s_ready);
        }
      }
      const int kb = i % kKt;
      if (!wait_warp(&b->kfull[s], u) || !wait_warp(&b->gfull[s], u)) break;
      if constexpr (STATE) {
        if (i >= kKt && !wait_warp(&b->kt_free[kb], i / kKt - 1)) break;
      } else {
        if (!wait_warp(&b->p_ready, i)) break;       // the scores' columns are free
      }
      tc_fence_after();
      const Block& k = b->blk[s];
      const float bf = k.f;
      const bool slow = k.slow;
      {
        const uint8_t* col = smem + M::kK + s * M::kKTile + (k0 / 64) * C * 128 + (k0 & 7) * 2;
        const int ch = (k0 % 64) / 8;
#pragma unroll
        for (int c = 0; c < 2; ++c) {            // 32 tokens: 16 columns of each part
          const int j0 = 64 * half + 32 * c;
          uint32_t part[3][16];
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            const float4 wj = *reinterpret_cast<const float4*>(&k.w[j0 + j]);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tok = j0 + j + e;
              const uint16_t raw = live && tok < nt ? *reinterpret_cast<const uint16_t*>(col + tok * 128 + ((ch ^ (tok & 7)) << 4)) : 0;
              x[e] = __uint_as_float((uint32_t)raw << 16) * (e == 0 ? wj.x : e == 1 ? wj.y : e == 2 ? wj.z : wj.w);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x0 = x[2 * e], x1 = x[2 * e + 1];
              const int o = j / 2 + e;
              part[0][o] = pack_bf16(x0, x1);
              x0 -= lo_f(part[0][o]);
              x1 -= hi_f(part[0][o]);
              part[1][o] = pack_bf16(x0, x1);
              part[2][o] = pack_bf16(x0 - lo_f(part[1][o]), x1 - hi_f(part[1][o]));
            }
          }
#pragma unroll
          for (int p = 0; p < 3; ++p) tmem_st16(trow + kKT[kb][p] + 32 * half + 16 * c, part[p]);
        }
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&b->kt_ready[kb]);
        mbar_arrive(&b->kempty[s]);
        mbar_arrive(&b->gempty[s]);
      }
      if (!wait_warp(&b->u_done, i)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < HV / 32; ++c) {
        float v[32];
        tmem_ld32(trow + kU + half * HV + 32 * c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float& x = S[32 * c + j];
          x = slow ? x + fmaf(x, bf, v[j]) : fmaf(x, bf, v[j]);
        }
      }
      tc_fence_before();
      if constexpr (STATE) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->u_free);
        if (i + 1 == nblk && live) {
          float* dst = ws_state + (size_t)blockIdx.x * DV * DK;
#pragma unroll
          for (int j = 0; j < HV; ++j) dst[(size_t)(half * HV + j) * DK + k0] = S[j];
        }
      } else if (w.last() && live) {
        const int64_t slot = seq_slot(a, w.p.n);
        if (slot >= 0) {
          float* dst = a.state + ((size_t)slot * a.H + w.p.h) * DV * DK;
#pragma unroll
          for (int j = 0; j < HV; ++j) dst[(size_t)(half * HV + j) * DK + k0] = S[j];
        }
      }
    }
  } else if (!STATE) {
    // warp 3: empty sequences keep their state, or zeros when they are fresh
    for (int n = blockIdx.x; n < a.N; n += gridDim.x) {
      if (seq_len(a, n) > 0 || seq_init(a, n)) continue;
      const int64_t slot = seq_slot(a, n);
      if (slot < 0) continue;
      float4* dst = reinterpret_cast<float4*>(a.state + (size_t)slot * a.H * DV * DK);
      for (int64_t x = lane; x < (int64_t)a.H * DV * DK / 4; x += 32) dst[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  __syncwarp();
  if (warp == 1 && lane == 0) {
    // products in flight still read shared memory and TMEM
    mma_commit(&b->kt_free[1]);
    mbar_wait(&b->kt_free[1], STATE ? (nblk / 2) & 1 : 0, nullptr, 50ull * 1000 * 1000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Chains the cut-off pieces: row r of ws_state becomes the incoming state of range r + 1,
//   S_r = U_r + exp(D_r) S_{r-1}, where a piece that opens its sequence takes the pool's state (or 0).
// and row R + r a copy of the pool's state of the sequence that opens in range r and is cut at its end.
// Grid (R, elements / 1024): the CTAs of a row that opens a sequence walk the rows that continue it.
__global__ void __launch_bounds__(256) linear_chain_kernel(const LinAttnArgs a, float* __restrict__ ws_state,
                                                          const int4* __restrict__ ws_meta) {
  int4 m = ws_meta[blockIdx.x * 2];
  if (!m.x || !m.z) return;
  const int n = m.w, h = ws_meta[blockIdx.x * 2 + 1].x;
  const size_t per = (size_t)a.dk * a.dv, x = (size_t)blockIdx.y * 1024 + threadIdx.x * 4;
  if (x >= per) return;
  const int64_t slot = seq_slot(a, n);
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (slot >= 0 && seq_init(a, n)) {
    s = *reinterpret_cast<const float4*>(a.state + ((size_t)slot * a.H + h) * per + x);
    *reinterpret_cast<float4*>(ws_state + (size_t)(gridDim.x + blockIdx.x) * per + x) = s;
  }
  for (int r = blockIdx.x;;) {
    float4* row = reinterpret_cast<float4*>(ws_state + (size_t)r * per + x);
    const float4 v = *row;
    const float d = __int_as_float(m.y);
    const bool slow = d > -0.5f;
    const float f = slow ? expm1f(d) : expf(d);
    s.x = slow ? s.x + fmaf(s.x, f, v.x) : fmaf(s.x, f, v.x);
    s.y = slow ? s.y + fmaf(s.y, f, v.y) : fmaf(s.y, f, v.y);
    s.z = slow ? s.z + fmaf(s.z, f, v.z) : fmaf(s.z, f, v.z);
    s.w = slow ? s.w + fmaf(s.w, f, v.w) : fmaf(s.w, f, v.w);
    *row = s;
    if (++r >= gridDim.x) break;
    m = ws_meta[r * 2];
    if (!m.x || m.z) break;              // the next range ends its sequence, or its last piece opens another
  }
}

// ---------------------------------------------------------------- host side
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// [T, heads, d] rows in boxes of 128 tokens x one head x 64 columns
bool encode_rows(CUtensorMap* m, const void* p, int d, int heads, int T, int64_t st_h, int64_t st_t) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)T};
  // the stride of a dimension of one element is never used; it only has to be valid
  cuuint64_t strides[2] = {heads > 1 ? (cuuint64_t)st_h * 2 : (cuuint64_t)d * 2, T > 1 ? (cuuint64_t)st_t * 2 : (cuuint64_t)d * 2};
  cuuint32_t box[3] = {64, 1, C};
  cuuint32_t es[3] = {1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool needs_cut(const LinAttnArgs& a, int sms) {
  // an item of ceil(len / 128) blocks is cut when it is longer than two ranges of total / sms blocks,
  // and the total is at least H items of that length
  return a.H * 2 < sms && (a.T + C - 1) / C > 2 * kMinCut;
}

template <int DK, int DV>
const char* launch_dims(const LinAttnArgs& a, float* ws, int sms, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  if (!encode_rows(&tq, a.q, DK, a.H / a.q_div, a.T, a.qs_h, a.qs_t) ||
      !encode_rows(&tk, a.k, DK, a.H / a.k_div, a.T, a.ks_h, a.ks_t) ||
      !encode_rows(&tv, a.v, DV, a.H / a.v_div, a.T, a.vs_h, a.vs_t))
    return "linear_attention: cuTensorMapEncodeTiled failed";
  constexpr int kSmem = Smem<DK, DV>::kBars + (int)sizeof(Bars) + 1024;
  static unsigned long long done_main = 0, done_state = 0;
  if (!set_max_smem_per_device(linear_blocks_kernel<DK, DV, false>, kSmem, done_main) ||
      !set_max_smem_per_device(linear_blocks_kernel<DK, DV, true>, kSmem, done_state))
    return "linear_attention: shared memory limit";
  int4* meta = nullptr;
  if (needs_cut(a, sms)) {
    if (!ws) return "linear_attention: workspace";
    meta = reinterpret_cast<int4*>(ws + (size_t)2 * sms * DK * DV);
    linear_blocks_kernel<DK, DV, true><<<sms, kThreads, kSmem, st>>>(tq, tk, tv, a, ws, meta);
    linear_chain_kernel<<<dim3(sms, (DK * DV + 1023) / 1024), 256, 0, st>>>(a, ws, meta);
  }
  linear_blocks_kernel<DK, DV, false><<<sms, kThreads, kSmem, st>>>(tq, tk, tv, a, ws, meta);
  return nullptr;
}

}  // namespace

bool linear_blocks_supported(const LinAttnArgs& a, bool f32) {
  auto ok = [](const void* p, int64_t sh, int64_t st, int heads, int T) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (heads == 1 || (sh % 8 == 0 && sh > 0)) &&
           (T == 1 || (st % 8 == 0 && st > 0)) && sh < (1ll << 38) && st < (1ll << 38);
  };
  return !f32 && (a.dk == 64 || a.dk == 128) && (a.dv == 64 || a.dv == 128) && a.T > 0 &&
         ok(a.q, a.qs_h, a.qs_t, a.H / a.q_div, a.T) && ok(a.k, a.ks_h, a.ks_t, a.H / a.k_div, a.T) &&
         ok(a.v, a.vs_h, a.vs_t, a.H / a.v_div, a.T) && ok(a.out, a.os_h, a.os_t, a.H, a.T) &&
         reinterpret_cast<uintptr_t>(a.state) % 16 == 0;
}

int64_t linear_blocks_workspace(const LinAttnArgs& a, int sms) {
  return needs_cut(a, sms) ? (int64_t)sms * (2 * a.dk * a.dv + 8) : 0;
}

const char* launch_linear_blocks(const LinAttnArgs& a, float* ws, int sms, cudaStream_t st) {
  if (a.dk == 128 && a.dv == 128) return launch_dims<128, 128>(a, ws, sms, st);
  if (a.dk == 128 && a.dv == 64) return launch_dims<128, 64>(a, ws, sms, st);
  if (a.dk == 64 && a.dv == 128) return launch_dims<64, 128>(a, ws, sms, st);
  if (a.dk == 64 && a.dv == 64) return launch_dims<64, 64>(a, ws, sms, st);
  return "linear_attention: head size";
}

}  // namespace air
