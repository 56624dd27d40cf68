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
// are exact). S itself stays f32: the keys times their f32 decay factors are split into four bf16
// parts that add up to all 24 bits, each block's update is accumulated on its own and added to S in
// registers, because adding it to a long-lived accumulator inside the tensor core would round the
// whole state 32 times a block.
//
// A CTA has 20 warps, each with one task, that pass blocks on through mbarriers (every wait is bounded): copies;
// decays (sums of log decays within 32 tokens; a difference of sums is taken for two tokens of the same 32 only); the
// two groups of products, Q K^T / Q S / P V and W V, issued by one thread each; scores -> P and O -> output; keys -> W;
// the state. NaN and infinities in V show in W V: there the state's warps turn them into zeros before P V, where 0
// times them would reach earlier tokens' outputs, and the output's warps write NaN to their columns from their
// token on. W goes through a ring of 16 tokens at a time, so that its production and W V overlap, and W V of a block
// overlaps Q K^T and P. The tasks' code is kept short (rolled loops, waits as a call): when it did not fit the
// instruction cache the same work took four times as long.
//
// Split over the length: the (sequence, head, block) triples form one list. Where a sequence is longer than
// two SMs' shares of it, the list is cut into one stretch per SM: a first kernel computes the state that each
// cut-off piece adds (K and V only), a second one chains these states along the list, and the main kernel
// starts each stretch from its incoming state. Otherwise whole sequences are dealt out, the longest first.
// All sums have a fixed order.
//
// Measured (B200): 148 heads of 128, 2048 tokens each, one head per SM: 74.5 us, 7300 clocks a block (SM cycles over 16
// blocks, set-up included). The tensor pipe is active 49 % of them, tensor memory 53 %, HBM 46 %, L1 and shared
// memory 38 %: no unit is near its limit. What bounds it is the chain of a block's steps: Q K^T of the next block
// starts behind P V of this one, because P lies over the scores and Q has one tile. One prompt of 16384 tokens, 32
// heads: 186 us (71, 9.5 and 127 for each of the three kernels alone; their ends overlap) of an 83 us floor; 13 ragged
// prompts of 8111 tokens together: 102 to 108 us; 77 tokens, 16 heads of 64: 9.2 us.
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
// Tokens of sequence n, -1 where its offsets are out of range: it is skipped like an empty one, and keeps its state.
AIR_DEVICE int seq_len(const LinAttnArgs& a, int n) {
  if (!a.cu) return a.T;
  const int t0 = a.cu[n], t1 = a.cu[n + 1];
  if (t0 < 0 || t1 < t0 || t1 > a.T) {
    set_error(a.err, kErrBounds);
    return -1;
  }
  return t1 - t0;
}
AIR_DEVICE int seq_blocks(const LinAttnArgs& a, int n) { return (seq_len(a, n) + C - 1) / C; }
AIR_DEVICE int64_t seq_slot(const LinAttnArgs& a, int n) {
  if (!a.state) return -1;
  const int64_t s = a.slots ? (int64_t)a.slots[n] : (int64_t)n;
  if (s < -1 || s >= a.S) set_error(a.err, kErrBounds);
  return s < 0 || s >= a.S ? -1 : s;
}
AIR_DEVICE bool seq_init(const LinAttnArgs& a, int n) {
  return a.has_state ? a.has_state[n] != 0 : a.has_state_all != 0;
}

constexpr int kSort = 32;          // so many sequences are put in order of their length
struct Range {
  Pos begin, end;                  // end: one past the last block, as the position of the next one
  int blocks;                      // blocks of the range
  int whole;                       // whole items, dealt out in turns, instead of a stretch of the list
  int cut_end, tail;               // the stretch ends inside an item; blocks of that last piece
};
// The sequence of item t, and the item that CTA r of R gets in turn k: forth and back over the CTAs.
AIR_DEVICE int item_seq(const LinAttnArgs& a, const int* order, int t) { return a.N <= kSort ? order[t / a.H] : t / a.H; }
AIR_DEVICE int item_of(int k, int r, int R) { return k * R + (k & 1 ? R - 1 - r : r); }

// The first position at or after list index p where a stretch may start: p itself inside an item that is
// cut, else the nearer end of the item (warp-wide). Returns its index. nb, inc: blocks of sequence `lane`
// and their running sum.
AIR_DEVICE int snap(const LinAttnArgs& a, int p, int total, int longest, int nb, int inc, Pos& pos) {
  const int lane = threadIdx.x & 31;
  pos = Pos{a.N, 0, 0};
  if (p >= total) return total;
  int base = 0, len = 0;
  for (int n0 = 0;;) {
    const int all = __shfl_sync(0xffffffffu, inc, 31) * a.H;
    if (p < base + all) {
      const int l = __ffs(__ballot_sync(0xffffffffu, base + inc * a.H > p)) - 1;
      len = __shfl_sync(0xffffffffu, nb, l);
      const int rel = p - base - (__shfl_sync(0xffffffffu, inc, l) - len) * a.H;
      pos = Pos{n0 + l, rel / len, rel % len};
      break;
    }
    base += all;
    n0 += 32;
    nb = n0 + lane < a.N ? seq_blocks(a, n0 + lane) : 0;
    inc = nb;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
  }
  if (pos.c == 0 || len > longest) return p;
  const int c = pos.c;
  pos.c = 0;
  if (2 * c < len) return p - c;
  if (++pos.h == a.H) {
    pos.h = 0;
    do { ++pos.n; } while (pos.n < a.N && seq_len(a, pos.n) <= 0);
  }
  return p + len - c;
}

// What CTA r of R works on (warp-wide; order: shared memory for kSort entries).
__device__ __noinline__ Range make_range(const LinAttnArgs& a, int r, int R, int* order) {
  const int lane = threadIdx.x & 31;
  const int nb = lane < a.N ? seq_blocks(a, lane) : 0;
  // Disjoint sequences have at most T / C + N blocks, which times H stays below 2^30. Offsets that go back and
  // forth can name any number: such a call is reported and does nothing.
  const int limit = a.T / C + a.N;
  int total = nb, most = nb;
  for (int n = lane + 32; n < a.N; n += 32) {
    const int x = seq_blocks(a, n);
    total = min(total + x, limit + 1);
    most = max(most, x);
  }
  const int64_t sum = (int64_t)__reduce_add_sync(0xffffffffu, total >> 16) * 65536 + __reduce_add_sync(0xffffffffu, total & 0xFFFF);
  most = __reduce_max_sync(0xffffffffu, most);
  Range g{};
  if (sum > limit) {
    if (lane == 0) set_error(a.err, kErrBounds);
    return g;
  }
  total = (int)sum * a.H;
  int per = (total + R - 1) / R;
  const int longest = 2 * max(per, kMinCut);
  if (most <= longest) {
    // no item is worth a cut: the longest first, so that the turns even out
    g.whole = 1;
    if (a.N <= kSort) {
      int rank = 0;
      for (int m = 0; m < a.N; ++m) {
        const int x = __shfl_sync(0xffffffffu, nb, m);
        rank += x > nb || (x == nb && m < lane);
      }
      if (lane < a.N) order[rank] = lane;
      __syncwarp();
    }
    int blocks = 0;
    for (int k = lane; k * (int64_t)R < (int64_t)a.N * a.H; k += 32) {
      const int t = item_of(k, r, R);
      if (t < a.N * a.H) blocks += seq_blocks(a, item_seq(a, order, t));
    }
    g.blocks = __reduce_add_sync(0xffffffffu, blocks);
    return g;
  }
  per = max(per, kMinCut);
  int inc = nb;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  const int64_t p0 = (int64_t)r * per, p1 = p0 + per;
  const int i0 = snap(a, (int)min(p0, (int64_t)total), total, longest, nb, inc, g.begin);
  const int i1 = snap(a, (int)min(p1, (int64_t)total), total, longest, nb, inc, g.end);
  g.blocks = i1 - i0;
  g.cut_end = g.blocks > 0 && g.end.n < a.N && g.end.c > 0;
  g.tail = g.cut_end ? min(g.blocks, g.end.c) : 0;
  return g;
}

// Walks the blocks of a range in order.
struct Walk {
  const LinAttnArgs& a;
  const int* order;
  Pos p;
  int nb, t0, len, turn, whole;
  AIR_DEVICE Walk(const LinAttnArgs& args, const int* ord, const Pos& begin, int dealt)
      : a(args), order(ord), p(begin), nb(0), turn(-1), whole(dealt) {
    if (whole) deal();
    else load();
  }
  AIR_DEVICE void load() {
    nb = 0;
    if (p.n >= a.N) return;
    t0 = seq_begin(a, p.n);
    len = seq_len(a, p.n);
    nb = (len + C - 1) / C;
  }
  AIR_DEVICE void deal() {
    for (p.c = 0;;) {
      const int t = item_of(++turn, blockIdx.x, gridDim.x);
      if (turn * (int64_t)gridDim.x >= (int64_t)a.N * a.H) return;
      if (t >= a.N * a.H) continue;
      p.n = item_seq(a, order, t);
      p.h = t % a.H;
      load();
      if (nb > 0) return;
    }
  }
  AIR_DEVICE int token() const { return t0 + p.c * C; }
  AIR_DEVICE int count() const { return min(C, len - p.c * C); }
  AIR_DEVICE bool last() const { return p.c + 1 == nb; }
  AIR_DEVICE void next() {
    if (++p.c < nb) return;
    if (whole) return deal();
    p.c = 0;
    if (++p.h < a.H) return;
    p.h = 0;
    do { ++p.n; } while (p.n < a.N && seq_len(a, p.n) <= 0);
    load();
  }
};

// ---------------------------------------------------------------- descriptors
// Both operands use the 128-byte swizzle layout (8 rows of 128 B an atom, atoms 1024 B apart); the
// descriptors' high words are equal: stride 1024, version 1, SWIZZLE_128B.
constexpr uint32_t kDescHi = (1024 >> 4) | (1u << 14) | (2u << 29);
// K-contiguous operand, low word.
AIR_DEVICE uint32_t k_desc(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
// N-contiguous (MN-major) operand: rows of K hold 64 bf16 of N, the next 64 columns of N are one panel
// further (the leading byte offset).
AIR_DEVICE uint32_t mn_desc(uint32_t addr, uint32_t panel_bytes) { return ((addr & 0x3FFFF) >> 4) | (panel_bytes >> 4) << 16; }
constexpr uint32_t kBMn = 1u << 16;      // instruction descriptor: B is N-contiguous

AIR_DEVICE void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi) : "memory");
}
AIR_DEVICE void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "mov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(acc), "n"(kDescHi) : "memory");
}

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
AIR_DEVICE void tma_load_3d(uint32_t dst, const void* tmap, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
AIR_DEVICE void tma_store_3d(const void* tmap, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
               ::"l"(tmap), "r"(smem_u32(src)), "r"(x), "r"(y), "r"(z) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until the stores of this thread have read shared memory (READ) or are complete.
template <bool READ> AIR_DEVICE void tma_store_wait() {
  if constexpr (READ) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  else asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}
AIR_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Bounded wait: gives up after about a quarter of a second, or when another role of the CTA has, and
// leaves word of it in *abort_flag. The loop is a call, so that the many waits stay small: the code of
// all roles together has to stay in the instruction cache.
__device__ __noinline__ void bar_wait_slow(uint64_t* bar, uint32_t parity, int* abort_flag) {
  const long long t0 = clock64();
#pragma unroll 1
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return;
    if (*(volatile int*)abort_flag != 0) return;
    if (clock64() - t0 > (1ll << 29)) {
      *(volatile int*)abort_flag = 1;
      return;
    }
  }
}
// After an abort a wait returns without what it waited for. Whoever then goes on to global memory (a copy, an
// output, a state's row) looks first whether it did, and leaves; what a role does until then stays inside the
// CTA's own memory.
AIR_DEVICE void bar_wait(uint64_t* bar, uint32_t parity, int* abort_flag) {
  if (!mbar_try_wait(bar, parity & 1)) bar_wait_slow(bar, parity & 1, abort_flag);
}
// For copies in flight at the end: waits on whatever happened, for a shorter time.
__device__ __noinline__ void bar_drain(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity & 1) && clock64() - t0 < (1ll << 27)) {}
}
// Two f32 operations in one instruction.
AIR_DEVICE uint64_t f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
AIR_DEVICE void unf2(uint64_t r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
AIR_DEVICE uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AIR_DEVICE uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
AIR_DEVICE uint32_t bf2_mul(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
AIR_DEVICE uint32_t bf2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
AIR_DEVICE uint32_t bf2_neg(uint32_t a) {
  uint32_t r;
  asm("neg.bf16x2 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
// 16 lanes x 32 columns from matrix fragments: for every 4 columns 4 j + t % 4, thread t writes lane t / 4
// (r[2 j]) and 8 + t / 4 (r[2 j + 1]).
AIR_DEVICE void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Four transposed 8 x 8 tiles of 16-bit numbers: thread t gets rows 2 (t % 4), + 1 of column t / 4 of each.
AIR_DEVICE void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
AIR_DEVICE void sts128(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
AIR_DEVICE uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// ---------------------------------------------------------------- shared memory
template <int DK, int DV>
struct Smem {
  static constexpr int kKTile = C * DK * 2, kVTile = C * DV * 2, kSTile = DK * DV * 2;
  static constexpr int kK = 0, kV = 2 * kKTile, kQ = kV + 2 * kVTile, kS = kQ + kKTile, kBars = kS + kSTile;
};
constexpr int kRing = 4;           // blocks whose decays and descriptions are in shared memory
struct alignas(16) Block {
  // decays, all from sums within 32 tokens
  float gl[C];                     // log2 of exp(g_1 + ... + g_i) over the token's own 32
  float e[C];                      // exp(g_{j+1} + ... ) up to the end of the token's 32
  uint32_t w[3][C / 2];            // exp(g_{j+1} + ... + g_128) as three bf16 parts, two tokens a word
  float t2[4];                     // log2 of the 32s' total decays
  // S <- exp(total) S + U as one S + (f S + U): f = expm1(total), one = 1 where the decay is slow, so
  // that a slow head does not drift by a factor that is rounded the same way every block
  float f, one;
  int tok, nt;                     // first token, tokens
  int h, hq, hk, hv;               // head, and the ones it reads
  int in;                          // the block has an incoming state
  int first;                       // first block of a piece: S comes from src (null: zeros)
  const float* src;
  float* dst;                      // where S goes after the block (null: nowhere)
};
struct Bars {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], dfull[kRing], gfull[kRing], gempty[kRing];
  uint64_t qfull, qempty;
  uint64_t sc_done, qs_done, o_done, o_scaled, o_free, s_ready, drain[2];
  // pairs: the waiting side may be two phases behind (for o_staged: copies that wait for a late description)
  uint64_t p_ready[2], u_done[2], u_free[2], o_staged[2], v_clean[2];
  uint64_t kt_ready[4], kt_free[4];
  uint32_t tmem;
  int abort;
  alignas(8) uint8_t odd[2][8];    // V's tile had NaN or infinities: 4 times 32 rows of the left, of the right columns
  uint8_t first[2][4][128];        // then: the first row of each column that had (C: none)
  Range range;
  int order[kSort];
  Block blk[kRing];
};

// 20 warps: 4 of service (products of the output, copies, decays, products of the state), 4 of output, 4 of
// keys, 8 of state.
constexpr int kThreads = 640;
AIR_DEVICE bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// TMEM columns. P takes the lower half of the scores' columns as they are read. The decayed keys go
// through a ring of four times 16 tokens (four parts of 8 columns).
constexpr uint32_t kSC = 0, kP = 0, kKT = 128, kO = 256, kU = 384;
// The state-only kernel has neither scores nor O and takes two regions for U in turn.
template <bool STATE> AIR_DEVICE uint32_t u_cols(int i) { return STATE && (i & 1) ? kO : kU; }

// Turns NaN and infinities in rows [x0, x1) and columns [c0, c0 + n) of V's tile into zeros (warp-wide); the first row
// of each column that had one goes to first (C: none). Eight columns a lane.
__device__ __noinline__ void clear_odd(uint8_t* tile, int x0, int x1, int c0, int n, uint8_t* first) {
  const int lane = threadIdx.x & 31, chunk = c0 / 8 + lane;
  if (lane < n / 8) {
    first += 8 * chunk;
    for (int e = 0; e < 8; ++e) first[e] = C;
#pragma unroll 1
    for (int x = x0; x < x1; ++x) {
      uint16_t* v = reinterpret_cast<uint16_t*>(tile + (chunk >> 3) * C * 128 + x * 128 + (((chunk ^ x) & 7) << 4));
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        if ((v[e] & 0x7F80u) != 0x7F80u) continue;
        v[e] = 0;
        if (first[e] == C) first[e] = (uint8_t)x;
      }
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// STATE: the state-only pass over each range's cut-off last piece.
template <int DK, int DV, bool STATE>
__global__ void __launch_bounds__(kThreads, 1)
linear_blocks_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                     const __grid_constant__ LinAttnArgs a,
                     float* __restrict__ ws_state, int4* __restrict__ ws_meta) {
  using M = Smem<DK, DV>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023u);   // an offset, so that accesses stay shared-space
  Bars* b = reinterpret_cast<Bars*>(smem + M::kBars);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  if (warp == 2) {
    const Range g = make_range(a, blockIdx.x, gridDim.x, b->order);
    if (lane == 0) b->range = g;
  }
  if (warp == 3 && lane == 0) {
    prefetch_tmap(&tm_k);
    prefetch_tmap(&tm_v);
    if (!STATE) prefetch_tmap(&tm_q);
    if (!STATE) prefetch_tmap(&tm_o);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&b->kfull[i], 1);
      mbar_init(&b->kempty[i], 8);
      mbar_init(&b->vfull[i], 1);
      mbar_init(&b->vempty[i], 1);
      mbar_init(&b->drain[i], 1);
      mbar_init(&b->p_ready[i], 4);
      mbar_init(&b->u_done[i], 1);
      mbar_init(&b->u_free[i], 8);
      mbar_init(&b->o_staged[i], 4);
      mbar_init(&b->v_clean[i], 8);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&b->kt_ready[i], 4);
      mbar_init(&b->kt_free[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&b->dfull[i], 1);
      mbar_init(&b->gfull[i], 1);
      mbar_init(&b->gempty[i], STATE ? 18 : 19);
    }
    mbar_init(&b->qfull, 1);
    mbar_init(&b->qempty, 4);
    mbar_init(&b->sc_done, 1);
    mbar_init(&b->qs_done, 1);
    mbar_init(&b->o_done, 1);
    mbar_init(&b->o_scaled, 4);
    mbar_init(&b->o_free, 4);
    mbar_init(&b->s_ready, 8);
    b->abort = 0;
    fence_mbar_init();
  }
  if constexpr (STATE) {
    // most ranges of most calls have nothing to do here
    __syncthreads();
    if (b->range.tail == 0) {
      if (threadIdx.x == 0) ws_meta[blockIdx.x * 2].x = 0;
      return;                              // counts as the trigger of the next kernel
    }
  }
  if (warp == 1) tmem_alloc(&b->tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // the chained states come from the kernel before, which may still run; so may the copies of the pool
  if (ws_state) pdl_wait();
  pdl_trigger();
  const uint32_t tmem = __shfl_sync(0xffffffffu, b->tmem, 0);
  const int nblk = __shfl_sync(0xffffffffu, STATE ? b->range.tail : b->range.blocks, 0);
  auto wait = [&](uint64_t* bar, int parity) { bar_wait(bar, parity, &b->abort); };
  constexpr uint32_t id_mn = idesc_bf16_f32(128, DV) | kBMn;
  auto aborted = [&] { return *(volatile int*)&b->abort != 0; };
  auto warp_aborted = [&] { return __any_sync(0xffffffffu, aborted()) != 0; };   // one answer for the whole warp

  if (warp < 4) {
    if (warp == 1) {
      // -------------------------------------------------------------- copies
      if (lane == 0) {
        const uint32_t sm = smem_u32(smem);
        int k_issued = 0, v_issued = 0, q_issued = 0;
        int h0 = 0, tok0 = 0, rows0 = 0, h1 = 0, tok1 = 0, rows1 = 0;    // the two blocks before
        // the output of a block out of V's tile, of which it took the place
        auto out = [&](int i, int h, int tok, int rows) {
          wait(&b->o_staged[i & 1], i >> 1);
          if (aborted()) return;
#pragma unroll 1
          for (int x = 0; x < rows; x += 32)
#pragma unroll
            for (int c = 0; c < DV / 64; ++c)
              tma_store_3d(&tm_o, smem + M::kV + (i & 1) * M::kVTile + c * C * 128 + x * 128, 64 * c, h, tok + x);
          tma_store_wait<true>();
        };
#pragma unroll 1
        for (int i = 0; i < nblk; ++i) {
          const int s = i & 1, u = i >> 1, r = i % kRing;
          wait(&b->dfull[r], i / kRing);
          const int z = b->blk[r].tok, h = b->blk[r].h, nt = b->blk[r].nt, hq = b->blk[r].hq, hk = b->blk[r].hk, hv = b->blk[r].hv;
          mbar_arrive(&b->gempty[r]);
          if (i >= 2) wait(&b->kempty[s], u - 1);
          if (aborted()) break;
          mbar_expect_tx(&b->kfull[s], M::kKTile);
#pragma unroll
          for (int p = 0; p < DK / 64; ++p)
            tma_load_3d(sm + M::kK + s * M::kKTile + p * C * 128, &tm_k, &b->kfull[s], 64 * p, hk, z);
          ++k_issued;
          if (i >= 2) {
            if constexpr (STATE) wait(&b->vempty[s], u - 1);
            else out(i - 2, h0, tok0, rows0);
          }
          if (aborted()) break;
          mbar_expect_tx(&b->vfull[s], M::kVTile);
#pragma unroll
          for (int p = 0; p < DV / 64; ++p)
            tma_load_3d(sm + M::kV + s * M::kVTile + p * C * 128, &tm_v, &b->vfull[s], 64 * p, hv, z);
          ++v_issued;
          if constexpr (!STATE) {
            if (i >= 1) wait(&b->qempty, i - 1);
            if (aborted()) break;
            mbar_expect_tx(&b->qfull, M::kKTile);
#pragma unroll
            for (int p = 0; p < DK / 64; ++p) tma_load_3d(sm + M::kQ + p * C * 128, &tm_q, &b->qfull, 64 * p, hq, z);
            ++q_issued;
          }
          h0 = h1, tok0 = tok1, rows0 = rows1;
          h1 = h, tok1 = z, rows1 = nt & ~31;
        }
        // never leave the CTA with copies in flight into its shared memory
        for (int i = max(0, k_issued - 2); i < k_issued; ++i) bar_drain(&b->kfull[i & 1], i >> 1);
        for (int i = max(0, v_issued - 2); i < v_issued; ++i) bar_drain(&b->vfull[i & 1], i >> 1);
        if (q_issued) bar_drain(&b->qfull, q_issued - 1);
        if (!STATE && !aborted()) {
          if (nblk > 1) out(nblk - 2, h0, tok0, rows0);
          if (nblk > 0) out(nblk - 1, h1, tok1, rows1);
        }
        tma_store_wait<false>();
      }
      __syncwarp();
      if constexpr (!STATE) {
        // empty sequences keep their state, or zeros when they are fresh
        for (int n = blockIdx.x; n < a.N; n += gridDim.x) {
          if (seq_len(a, n) != 0 || seq_init(a, n)) continue;
          const int64_t slot = seq_slot(a, n);
          if (slot < 0) continue;
          float4* dst = reinterpret_cast<float4*>(a.state + (size_t)slot * a.H * DV * DK);
          for (int64_t x = lane; x < (int64_t)a.H * DV * DK / 4; x += 32) dst[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
    } else if (warp == 0) {
      // -------------------------------------------------------------- products of the output
      // The whole warp walks and waits, so that operands stay in uniform registers; one lane issues. Q K^T
      // of the next block goes out behind P V, so that its P is there when its Q S can start.
      if constexpr (!STATE) {
        constexpr uint32_t id_qk = idesc_bf16_f32(128, C);
        int n_in = 0;                      // blocks with an incoming state so far
        const uint32_t sm = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
        const uint32_t dq = k_desc(sm + M::kQ), ds = mn_desc(sm + M::kS, DK * 128);
#pragma unroll 1
        for (int i = -1; i < nblk; ++i) {
          if (i >= 0) {
            const int s = i & 1, r = i % kRing;
            const uint32_t dvs = mn_desc(sm + M::kV + s * M::kVTile, C * 128);
            wait(&b->gfull[r], i / kRing);
            const int in = __shfl_sync(0xffffffffu, b->blk[r].in, 0);
            const int steps = __shfl_sync(0xffffffffu, (b->blk[r].nt + 15) / 16, 0);
            if (warp_aborted()) break;
            if (lane == 0) mbar_arrive(&b->gempty[r]);
            if (in) {
              // O = Q S
              wait(&b->s_ready, n_in);
              if (i >= 1) wait(&b->o_free, i - 1);
              tc_fence_after();
              if (elect()) {
#pragma unroll
                for (int ks = 0; ks < DK / 16; ++ks)
                  mma_ss(tmem + kO, dq + (ks / 4) * (C * 128 >> 4) + 2 * (ks & 3), ds + ks * (2048 >> 4), id_mn, ks > 0);
                mma_commit(&b->qs_done);
              }
              __syncwarp();
            }
            // O (+)= P V
            wait(&b->vfull[s], i >> 1);
            wait(&b->v_clean[s], i >> 1);
            wait(&b->p_ready[s], i >> 1);
            if (in) wait(&b->o_scaled, n_in);
            else if (i >= 1) wait(&b->o_free, i - 1);
            n_in += in;
            tc_fence_after();
            if (elect()) {
#pragma unroll 1
              for (int ks = 0; ks < steps; ++ks)
                mma_ts(tmem + kO, tmem + kP + 8 * ks, dvs + ks * (2048 >> 4), id_mn, in || ks > 0);
              mma_commit(&b->o_done);
            }
            __syncwarp();
          }
          if (i + 1 < nblk) {
            // scores = Q K^T
            const uint32_t dks = k_desc(sm + M::kK + ((i + 1) & 1) * M::kKTile);
            wait(&b->kfull[(i + 1) & 1], (i + 1) >> 1);
            wait(&b->qfull, i + 1);
            tc_fence_after();
            if (elect()) {
#pragma unroll
              for (int ks = 0; ks < DK / 16; ++ks) {
                const int off = (ks / 4) * (C * 128 >> 4) + 2 * (ks & 3);
                mma_ss(tmem + kSC, dq + off, dks + off, id_qk, ks > 0);
              }
              mma_commit(&b->sc_done);
            }
            __syncwarp();
          }
        }
        // products in flight still read shared memory and TMEM
        if (elect()) mma_commit(&b->drain[0]);
        __syncwarp();
        bar_drain(&b->drain[0], 0);
      }
    } else if (warp == 3) {
      // -------------------------------------------------------------- products of the state
      int n = 0;                           // 16s of tokens so far
      const uint32_t sm = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
#pragma unroll 1
      for (int i = 0; i < nblk; ++i) {
        const int s = i & 1, r = i % kRing;
        const uint32_t dvs = mn_desc(sm + M::kV + s * M::kVTile, C * 128);
        wait(&b->dfull[r], i / kRing);
        const int nt = __shfl_sync(0xffffffffu, b->blk[r].nt, 0), units = (nt + 15) / 16;
        if (warp_aborted()) break;
        if (lane == 0) mbar_arrive(&b->gempty[r]);
        wait(&b->vfull[s], i >> 1);
        if (!STATE && nt < C) wait(&b->p_ready[s], i >> 1);       // V's rows past the end are zeroed by then
        if (const int f = i - (STATE ? 2 : 1); f >= 0) wait(&b->u_free[f & 1], f >> 1);
        // U = W V, 16 tokens at a time, the smallest parts first
#pragma unroll 1
        for (int c = 0; c < units; ++c, ++n) {
          wait(&b->kt_ready[n & 3], n >> 2);
          tc_fence_after();
          if (elect()) {
            const uint32_t ta = tmem + kKT + 32 * (n & 3), td = tmem + u_cols<STATE>(i);
#pragma unroll
            for (int part = 3; part >= 0; --part)
              mma_ts(td, ta + 8 * part, dvs + c * (2048 >> 4), id_mn, part < 3 || c > 0);
            mma_commit(&b->kt_free[n & 3]);
            if (c + 1 == units) {
              mma_commit(&b->u_done[s]);
              if (STATE) mma_commit(&b->vempty[s]);     // else V's tile goes on to hold the output
            }
          }
          __syncwarp();
        }
      }
      if (elect()) mma_commit(&b->drain[1]);
      __syncwarp();
      bar_drain(&b->drain[1], 0);
    } else if (warp == 2) {
      // -------------------------------------------------------------- decays and descriptions
      // lane l: tokens 4l .. 4l + 3; eight lanes make one of the four 32s
      const Range rg = b->range;
      Walk w(a, b->order, STATE ? Pos{rg.end.n, rg.end.h, rg.end.c - rg.tail} : rg.begin, rg.whole);
      if (STATE && lane == 0) {
        ws_meta[blockIdx.x * 2] = make_int4(rg.cut_end, 0, w.p.c == 0, w.p.n);
        ws_meta[blockIdx.x * 2 + 1].x = w.p.h;
      }
      float total_piece = 0.f;
      for (int i = 0; i < nblk; ++i) {
        const int r = i % kRing, t0 = w.token(), nt = w.count();
        if (i >= kRing) wait(&b->gempty[r], i / kRing - 1);
        if (warp_aborted()) break;
        Block& k = b->blk[r];
        if (lane == 0) {                   // what the copies need does not wait for the rest
          k.tok = t0;
          k.nt = nt;
          k.h = w.p.h;
          k.hq = w.p.h / a.q_div;
          k.hk = w.p.h / a.k_div;
          k.hv = w.p.h / a.v_div;
          mbar_arrive(&b->dfull[r]);
        }
        float g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * lane + e;
          g[e] = j < nt ? a.decay[(int64_t)(t0 + j) * a.decay_t + w.p.h] : 0.f;
        }
        const int64_t slot = STATE ? -1 : seq_slot(a, w.p.n);
        float* row = slot < 0 ? nullptr : a.state + ((size_t)slot * a.H + w.p.h) * DV * DK;
        const bool resumes = !STATE && w.p.c == 0 && row && seq_init(a, w.p.n);
        if (resumes)                       // the state that a sequence starts from, on its way into L2
          for (int x = lane * 128; x < DV * DK * 4; x += 32 * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(row) + x));
        if (lane == 0) {
          k.first = i == 0 || w.p.c == 0;
          k.src = nullptr;
          k.dst = nullptr;
          if constexpr (STATE) {
            if (i + 1 == nblk) k.dst = ws_state + (size_t)blockIdx.x * DV * DK;
          } else {
            k.in = w.p.c > 0 || resumes;
            // The incoming state: the pool's; of a sequence that is cut the chain kernel's copy of it, because
            // the range that ends the sequence may write the pool's row first; inside a cut, the chain's.
            if (resumes)
              k.src = rg.cut_end && w.p.n == rg.end.n && w.p.h == rg.end.h
                          ? ws_state + (size_t)(gridDim.x + blockIdx.x) * DV * DK : row;
            else if (i == 0 && w.p.c > 0)
              k.src = ws_state + (size_t)(blockIdx.x - 1) * DV * DK;
            if (w.last()) k.dst = row;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = g[e] < kFloor ? kFloor : g[e];
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
        float after = __shfl_down_sync(0xffffffffu, down, 1, 8), bef = __shfl_up_sync(0xffffffffu, up, 1, 8);
        if ((lane & 7) == 7) after = 0.f;
        if ((lane & 7) == 0) bef = 0.f;
        const float t[4] = {__shfl_sync(0xffffffffu, up, 7), __shfl_sync(0xffffffffu, up, 15),
                            __shfl_sync(0xffffffffu, up, 23), __shfl_sync(0xffffffffu, up, 31)};
        float later = 0.f;                 // the 32s after this one
#pragma unroll
        for (int q = 3; q > 0; --q)
          if (lane / 8 < q) later += t[q];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = 4 * lane + e;
          k.gl[j] = (bef + pre[e]) * kLog2e;
          k.e[j] = ex2((suf[e] + after) * kLog2e);
          float w = j < nt ? expf(suf[e] + after + later) : 0.f;
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const __nv_bfloat16 h = f2bf(w);
            reinterpret_cast<__nv_bfloat16*>(k.w[p])[j] = h;
            w -= bf2f(h);
          }
        }
        const float total = (t[3] + t[2]) + (t[1] + t[0]);
        if (lane < 4) k.t2[lane] = (lane == 0 ? t[0] : lane == 1 ? t[1] : lane == 2 ? t[2] : t[3]) * kLog2e;
        if (lane == 0) {
          const bool slow = total > -0.5f;
          k.f = slow ? expm1f(total) : expf(total);
          k.one = slow ? 1.f : 0.f;
          total_piece += total;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->gfull[r]);
        w.next();
      }
      if (STATE && lane == 0) ws_meta[blockIdx.x * 2].y = __float_as_int(total_piece);   // the piece's own decay
    }
  } else if (warp < 8 && !STATE) {
    // ---------------------------------------------------------------- scores -> P, O -> out
    if constexpr (!STATE) {
      const int q = warp & 3, row = 32 * q + lane;
      const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
      int n_in = 0;
      int nt = 0, in = 0, h = 0, tok = 0;
      float gl = 0.f, rs = 0.f;            // log2 of the decay from the row's 32's and the block's begin to the row
      auto fetch = [&](int i) {
        wait(&b->gfull[i % kRing], i / kRing);
        const Block& k = b->blk[i % kRing];
        const float4 t = *reinterpret_cast<const float4*>(k.t2);
        nt = k.nt;
        in = k.in;
        h = k.h;
        tok = k.tok;
        gl = k.gl[row];
        rs = gl + (q > 2 ? t.z : 0.f) + (q > 1 ? t.y : 0.f) + (q > 0 ? t.x : 0.f);
      };
      if (nblk > 0) fetch(0);
#pragma unroll 1
      for (int i = 0; i < nblk; ++i) {
        const int s = i & 1, u = i >> 1, r = i % kRing;
        if (warp_aborted()) break;
        const Block& k = b->blk[r];
        wait(&b->sc_done, i);
        if (lane == 0) {
          mbar_arrive(&b->kempty[s]);      // Q K^T is done with K, and with Q unless Q S is to come
          if (!in) mbar_arrive(&b->qempty);
        }
        tc_fence_after();
        // rolled loops: the roles' code has to stay in the instruction cache together
#pragma unroll 1
        for (int c = 0; c < q; ++c) {
          uint32_t pk[16];
          float v[32];
          tmem_ld32(trow + kSC + 32 * c, v);
          // the decay from the end of 32 c to the row, of its own terms: taken off rs it would keep the rounding
          // of whatever the earlier 32s decay by
          const float f = ex2(gl + (c < 1 && q > 1 ? k.t2[1] : 0.f) + (c < 2 && q > 2 ? k.t2[2] : 0.f)) * a.scale;
          const uint64_t ff = f2(f, f);
          const float4* e4 = reinterpret_cast<const float4*>(&k.e[32 * c]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 e = e4[j];
            float p0, p1, p2, p3;
            unf2(mul2(f2(v[4 * j], v[4 * j + 1]), mul2(ff, f2(e.x, e.y))), p0, p1);
            unf2(mul2(f2(v[4 * j + 2], v[4 * j + 3]), mul2(ff, f2(e.z, e.w))), p2, p3);
            pk[2 * j] = pack_bf16(p0, p1);
            pk[2 * j + 1] = pack_bf16(p2, p3);
          }
          tmem_st16(trow + kP + 16 * c, pk);
        }
        {
          uint32_t pk[16];
          float v[32];
          tmem_ld32(trow + kSC + 32 * q, v);
          const float4* g4 = reinterpret_cast<const float4*>(&k.gl[32 * q]);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 g = g4[j];
            float p0 = v[4 * j] * a.scale * ex2(gl - g.x), p1 = v[4 * j + 1] * a.scale * ex2(gl - g.y);
            float p2 = v[4 * j + 2] * a.scale * ex2(gl - g.z), p3 = v[4 * j + 3] * a.scale * ex2(gl - g.w);
            p0 = 4 * j <= lane ? p0 : 0.f;
            p1 = 4 * j + 1 <= lane ? p1 : 0.f;
            p2 = 4 * j + 2 <= lane ? p2 : 0.f;
            p3 = 4 * j + 3 <= lane ? p3 : 0.f;
            pk[2 * j] = pack_bf16(p0, p1);
            pk[2 * j + 1] = pack_bf16(p2, p3);
          }
          tmem_st16(trow + kP + 16 * q, pk);
#pragma unroll
          for (int j = 0; j < 16; ++j) pk[j] = 0u;
#pragma unroll 1
          for (int c = q + 1; c < 4; ++c) tmem_st16(trow + kP + 16 * c, pk);
        }
        tmem_wait_st();
        if (nt < C) {
          // rows of V past the sequence's end: 0 x whatever they hold must stay 0
          wait(&b->vfull[s], u);
          if (row >= nt && row < (nt + 15) / 16 * 16) {
#pragma unroll 1
            for (int c = 0; c < DV / 8; ++c)
              *reinterpret_cast<uint4*>(smem + M::kV + s * M::kVTile + (c / 8) * C * 128 + row * 128 + 16 * (c % 8)) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&b->p_ready[s]);
          mbar_arrive(&b->gempty[r]);
        }
        if (in) {
          wait(&b->qs_done, n_in);
          if (lane == 0) mbar_arrive(&b->qempty);
          ++n_in;
          tc_fence_after();
          const float f = ex2(rs) * a.scale;
          const uint64_t ff = f2(f, f);
#pragma unroll 1
          for (int c = 0; c < DV / 32; ++c) {
            float v[32];
            tmem_ld32(trow + kO + 32 * c, v);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t o[16];
#pragma unroll
              for (int j = 0; j < 16; j += 2) {
                float o0, o1;
                unf2(mul2(f2(v[16 * h + j], v[16 * h + j + 1]), ff), o0, o1);
                o[j] = __float_as_uint(o0);
                o[j + 1] = __float_as_uint(o1);
              }
              tmem_st16(trow + kO + 32 * c + 16 * h, o);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&b->o_scaled);
        }
        // the next block's facts, before this one's output is waited for
        const int o_nt = nt;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (int64_t)(tok + row) * a.os_t + (int64_t)h * a.os_h;
        if (i + 1 < nblk) fetch(i + 1);
        wait(&b->o_done, i);
        wait(&b->u_done[s], u);            // the state's products are done with V, too
        wait(&b->v_clean[s], u);
        if (warp_aborted()) break;
        tc_fence_after();
        // 32 full rows leave through the tile of V, which the products have finished with, as copies of
        // 64 columns (a thread's own row is 256 bytes in global memory: 32 lines a store); the rows of a
        // partial 32 one by one
        const bool full = 32 * q + 32 <= o_nt;
        uint8_t* stage = smem + M::kV + s * M::kVTile + row * 128;
        const uint32_t st32 = smem_u32(stage);
#pragma unroll 1
        for (int c = 0; c < DV / 32; ++c) {
          float v[32];
          tmem_ld32(trow + kO + 32 * c, v);
          if (c == DV / 32 - 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->o_free);
          }
          uint32_t o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) o[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
          if (full) {
            const uint32_t at = st32 + (c >> 1) * C * 128;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              sts128(at + (((4 * (c & 1) + j) ^ (lane & 7)) << 4), o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          } else if (row < o_nt) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(out + 32 * c + 8 * j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        }
        if (*reinterpret_cast<const uint64_t*>(b->odd[s]) != 0u) {
#pragma unroll 1
          for (int x = 0; x < 4 * DV; ++x) {
            const int part = x / DV, c = x % DV;
            if (!b->odd[s][4 * (c / (DV / 2)) + part] || row < b->first[s][part][c] || row >= o_nt) continue;
            if (full) *reinterpret_cast<uint16_t*>(stage + (c >> 6) * C * 128 + ((((c & 63) >> 3) ^ (lane & 7)) << 4) + 2 * (c & 7)) = 0x7FFF;
            else reinterpret_cast<uint16_t*>(out)[c] = 0x7FFF;
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->o_staged[s]);
      }
    }
  } else if (warp < 12) {
    // ---------------------------------------------------------------- transposed, decayed keys
    // A warp has 32 columns k of the keys, 16 tokens at a time and two to a word: transposed loads give
    // a thread columns t / 4, + 8, + 16, + 24 and tokens 2 (t % 4), + 1, + 8, + 9. The products k w of
    // bf16 numbers come in four parts that add up to all their bits: k w1 is its rounding plus an exact
    // rest (16 bits), k w2 the same with k w3.
    const int q = warp & 3;
    const bool live = 32 * q < DK;               // dk = 64: the upper lanes are zeros
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16) + kKT;
    const uint32_t col0 = smem_u32(smem) + M::kK + (live ? q / 2 : 0) * C * 128 + (lane & 7) * 128 +
                          (((4 * (q & 1) + (lane >> 3)) ^ (lane & 7)) << 4);
    // In the state-only kernel (full blocks) the output warps share the work: every second 16 tokens.
    constexpr int kStep = STATE ? 2 : 1;
    const int mine = STATE && warp < 8;
    int n = 0;                                   // 16s of tokens in the blocks before
#pragma unroll 1
    for (int i = 0; i < nblk; ++i) {
      const int s = i & 1, r = i % kRing;
      wait(&b->gfull[r], i / kRing);
      wait(&b->kfull[s], i >> 1);
      if (warp_aborted()) break;
      const Block& k = b->blk[r];
      const int nt = k.nt, units = (nt + 15) / 16;
      const int from = live ? nt : 0;            // tokens from here on count as zeros, whatever they hold
      const uint32_t col = col0 + s * M::kKTile;
      uint32_t x[2][4];
      ldsm_t(col + mine * 2048, x[0]);
      ldsm_t(col + mine * 2048 + 1024, x[1]);
#pragma unroll 1
      for (int c = mine; c < units; c += kStep) {
        if (16 * c + 16 > from) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int j = 16 * c + 8 * h + 2 * (lane & 3);
            const uint32_t keep = (j < from ? 0xFFFFu : 0u) | (j + 1 < from ? 0xFFFF0000u : 0u);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[h][e] &= keep;
          }
        }
        uint32_t p[2][16];                       // lanes 0..15 and 16..31: [part][8 tokens][8 columns]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = 8 * c + 4 * h + (lane & 3);
          const uint32_t w1 = k.w[0][j], w2 = k.w[1][j], w3 = k.w[2][j];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t* o = &p[e / 2][2 * h + e % 2];
            o[0] = bf2_mul(x[h][e], w1);
            o[4] = bf2_fma(x[h][e], w1, bf2_neg(o[0]));
            o[8] = bf2_mul(x[h][e], w2);
            o[12] = bf2_fma(x[h][e], w3, bf2_fma(x[h][e], w2, bf2_neg(o[8])));
          }
        }
        if (c + kStep < units) {
          ldsm_t(col + (c + kStep) * 2048, x[0]);
          ldsm_t(col + (c + kStep) * 2048 + 1024, x[1]);
        }
        const int kt = (n + c) & 3;
        if (n + c >= 4) wait(&b->kt_free[kt], (n + c) / 4 - 1);
        tc_fence_after();
        tmem_st_frag(trow + 32 * kt, p[0]);
        tmem_st_frag(trow + 32 * kt + (16u << 16), p[1]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->kt_ready[kt]);
      }
      n += units;
      if (lane == 0) {
        mbar_arrive(&b->kempty[s]);
        mbar_arrive(&b->gempty[r]);
      }
    }
  } else {
    // ---------------------------------------------------------------- state
    // a thread has row k of the state (transposed) and half of its dv columns, in registers
    const int q = warp & 3, half = (warp - 12) >> 2, k0 = 32 * q + lane;
    const uint32_t trow = tmem + ((uint32_t)(32 * q) << 16);
    constexpr int HV = DV / 2;
    const bool live = k0 < DK;
    const uint32_t srow = smem_u32(smem) + M::kS + k0 * 128 + (half * HV / 64) * DK * 128;
    float S[HV];
    int n_in = 0;                                // blocks with an incoming state so far
#pragma unroll
    for (int j = 0; j < HV; ++j) S[j] = 0.f;
#pragma unroll 1
    for (int i = -1; i < nblk; ++i) {
      if (warp_aborted()) break;
      if (i >= 0) {
        // S after the block: the products' update, and the state's row at the end of a piece
        wait(&b->gfull[i % kRing], i / kRing);
        const Block& k = b->blk[i % kRing];
        const uint64_t ff = f2(k.f, k.f), one = f2(k.one, k.one);
        float* dst = k.dst;
        const int nt = k.nt;
        wait(&b->u_done[i & 1], i >> 1);
        if (warp_aborted()) break;
        tc_fence_after();
        uint64_t z = 0;                          // 0 x the update: not 0 where it has NaN or infinities
#pragma unroll
        for (int c = 0; c < HV / 16; ++c) {
          float v[16];
          tmem_ld16(trow + u_cols<STATE>(i) + half * HV + 16 * c, v);
#pragma unroll
          for (int j = 0; j < 16; j += 2) {
            const uint64_t x = f2(S[16 * c + j], S[16 * c + j + 1]);
            if (!STATE) z = fma2(f2(v[j], v[j + 1]), 0, z);
            unf2(fma2(x, one, fma2(x, ff, f2(v[j], v[j + 1]))), S[16 * c + j], S[16 * c + j + 1]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&b->u_free[i & 1]);
          mbar_arrive(&b->gempty[i % kRing]);
        }
        if constexpr (!STATE) {
          // a column of the update is finite where V's column is: else this warp's 32 tokens of V are gone through
          const bool odd = __any_sync(0xffffffffu, z != 0);
          if (odd) clear_odd(smem + M::kV + (i & 1) * M::kVTile, 32 * q, min(32 * q + 32, nt), half * HV, HV, b->first[i & 1][q]);
          if (lane == 0) {
            b->odd[i & 1][warp - 12] = odd;
            mbar_arrive(&b->v_clean[i & 1]);
          }
        }
        if (dst && live) {
          float* d = dst + half * HV * DK + k0;
#pragma unroll
          for (int j = 0; j < HV; ++j) d[j * DK] = S[j];
        }
      }
      if (STATE || i + 1 >= nblk) continue;
      wait(&b->gfull[(i + 1) % kRing], (i + 1) / kRing);
      if (warp_aborted()) break;
      const Block& k = b->blk[(i + 1) % kRing];
      if (k.first) {
        const float* src = k.src;
        const float* d = src + half * HV * DK + k0;
#pragma unroll
        for (int j = 0; j < HV; ++j) S[j] = src && live ? d[j * DK] : 0.f;
      }
      if (k.in) {
        // bf16 copy for Q S, once the products that read the one before are complete
        if (n_in > 0) wait(&b->qs_done, n_in - 1);
        ++n_in;
        if (live) {
#pragma unroll
          for (int c = 0; c < HV / 8; ++c)
            sts128(srow + ((((half * HV % 64) / 8 + c) ^ (k0 & 7)) << 4), pack_bf16(S[8 * c], S[8 * c + 1]),
                   pack_bf16(S[8 * c + 2], S[8 * c + 3]), pack_bf16(S[8 * c + 4], S[8 * c + 5]), pack_bf16(S[8 * c + 6], S[8 * c + 7]));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->s_ready);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && aborted()) {
    set_error(a.err, kErrTimeout);
    if (STATE) ws_meta[blockIdx.x * 2].y = 0x7FC00000;   // NaN: what is chained onto this piece is none
  }
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
  pdl_wait();
  pdl_trigger();
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

// [T, heads, d] rows in boxes of some tokens x one head x 64 columns
bool encode_rows(CUtensorMap* m, const void* p, int d, int heads, int T, int64_t st_h, int64_t st_t, int rows = C) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)T};
  // the stride of a dimension of one element is never used; it only has to be valid
  cuuint64_t strides[2] = {heads > 1 ? (cuuint64_t)st_h * 2 : (cuuint64_t)d * 2, T > 1 ? (cuuint64_t)st_t * 2 : (cuuint64_t)d * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)rows};
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
  CUtensorMap tq, tk, tv, to;
  if (!encode_rows(&tq, a.q, DK, a.H / a.q_div, a.T, a.qs_h, a.qs_t) ||
      !encode_rows(&tk, a.k, DK, a.H / a.k_div, a.T, a.ks_h, a.ks_t) ||
      !encode_rows(&tv, a.v, DV, a.H / a.v_div, a.T, a.vs_h, a.vs_t) ||
      !encode_rows(&to, a.out, DV, a.H, a.T, a.os_h, a.os_t, 32))
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
    linear_blocks_kernel<DK, DV, true><<<sms, kThreads, kSmem, st>>>(tq, tk, tv, to, a, ws, meta);
  }
  // The other two start while their predecessor ends (programmatic dependent launch): they set up, and wait for
  // it to be complete before they read what it wrote.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = meta ? 1 : 0;
  cudaError_t e = cudaSuccess;
  if (meta) {
    cfg.gridDim = dim3(sms, (DK * DV + 1023) / 1024);
    cfg.blockDim = dim3(256);
    e = cudaLaunchKernelEx(&cfg, linear_chain_kernel, a, ws, (const int4*)meta);
  }
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, linear_blocks_kernel<DK, DV, false>, tq, tk, tv, to, a, ws, meta);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

// Few tokens: the block kernel needs about 11 us for its first block whatever that holds, the token-by-token
// one 2.5 us + 0.55 us a token (32 heads of 128, one sequence: 9.5 against 11.7 us at 12 tokens, 11.8 against
// 11.7 at 16). Sequences of a token or two each: 16 x 32 heads 12.1 against 33 us at one token, 15.9 against 33
// at two; 128 x 32 heads 108 against 152 and 154 against 153 (the states' traffic bounds both). Lengths are on the
// device, so empty sequences count: one prompt of 1000 tokens in 700 slots goes token by token.
bool linear_blocks_worth(const LinAttnArgs& a) { return a.T > 12 && 2 * (int64_t)a.T > 3 * (int64_t)a.N; }

bool linear_blocks_supported(const LinAttnArgs& a, bool f32) {
  auto ok = [](const void* p, int64_t sh, int64_t st, int heads, int T) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (heads == 1 || (sh % 8 == 0 && sh > 0)) &&
           (T == 1 || (st % 8 == 0 && st > 0)) && sh < (1ll << 38) && st < (1ll << 38);
  };
  // A CTA may step over all empty sequences between two blocks, one by one or 148th of the items by turns: up to 2^20 of
  // them (some 100 clocks each) or 2^17 turns (250) stay far inside the 2^29 clocks after which waits give up.
  const bool short_walk = (int64_t)a.N * (a.H > 16 ? a.H : 16) <= (1ll << 24);
  return !f32 && short_walk && ((int64_t)a.T / C + a.N) * a.H < (1ll << 30) && (a.dk == 64 || a.dk == 128) && (a.dv == 64 || a.dv == 128) && a.T > 0 &&
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
