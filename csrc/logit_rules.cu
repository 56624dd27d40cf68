// What a request asks of its logits before sampling, in one pass over the vocabulary:
//   x -> x / rho^c (x > 0) or x * rho^c          repetition penalty, c = the token's count so far
//     -> x - c * frequency - [c > 0] * presence
//     -> x + bias[token]                          (a short list of tokens per row)
//     -> -inf where the grammar's allow bit is 0
// Memory-bound: 4 or 2 + 1 bytes read and 4 written per entry. A CTA walks a stretch of one row with the next
// tile's loads in flight, so that the row's own values (which row of counts, the penalties' powers, the bias
// list) are fetched once a stretch and their latency is not paid per tile. A masked entry is selected away, so
// whatever its logit holds (NaN, infinities) does not get through.
#include "common.cuh"
#include "logit_rules.h"

namespace air {

namespace {

constexpr int kThreads = 128, kPer = 4, kGroups = 1, kTile = kThreads * kPer * kGroups;
constexpr int kTable = 32;         // counts below this take rho^c from a table

struct Entries {
  float x[kGroups][kPer];
  uint32_t c[kGroups];             // four counts
  uint32_t m[kGroups];             // four allow bits
};

// Four entries per thread and tile. VEC: four neighbouring ones in one access (rows and pointers aligned for it,
// V a multiple of 4), so that a warp reads and writes whole lines; otherwise entries t, t + 128, ... one by one.
// 192 x 128256 bf16 (175 MB): 38 us with 512-entry tiles and eight of them a stretch, 42 with 2048-entry tiles,
// 43 with one tile a CTA, 41 with 16 a stretch.
template <bool VEC, bool BF16>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const LogitRulesArgs a, int tiles) {
  __shared__ float pw[kTable];
  __shared__ int ids[kThreads];
  __shared__ float vals[kThreads];
  __shared__ int wn[kThreads / 32];
  const int row = blockIdx.y, t = threadIdx.x;
  const int first = blockIdx.x * tiles * kTile, last = min(a.V, first + tiles * kTile);
  auto place = [&](int g, int j) { return kThreads * kPer * g + (VEC ? kPer * t + j : t + kThreads * j); };
  const float* lf = static_cast<const float*>(a.logits) + (size_t)row * a.ld_in;
  const __nv_bfloat16* lb = static_cast<const __nv_bfloat16*>(a.logits) + (size_t)row * a.ld_in;
  const uint32_t* mk = a.mask ? a.mask + (size_t)row * ((a.V + 31) / 32) : nullptr;
  int64_t crow = -1;
  if (a.counts) {
    crow = a.count_row ? a.count_row[row] : row;
    if (crow < -1 || crow >= a.S) {
      set_error(a.err, kErrBounds);
      crow = -1;
    }
  }
  const uint8_t* cnt = crow >= 0 ? a.counts + (size_t)crow * a.V : nullptr;
  auto load = [&](int i0, Entries& n) {
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      n.c[g] = 0;
      n.m[g] = 0xFu;
      if constexpr (VEC) {
        const int i = i0 + place(g, 0);
        if (i >= last) continue;
        if constexpr (BF16) {
          const uint2 u = __ldcs(reinterpret_cast<const uint2*>(lb + i));
          n.x[g][0] = __uint_as_float(u.x);      // two bf16 a word until they are used
          n.x[g][1] = __uint_as_float(u.y);
        } else {
          const float4 f = __ldcs(reinterpret_cast<const float4*>(lf + i));
          n.x[g][0] = f.x; n.x[g][1] = f.y; n.x[g][2] = f.z; n.x[g][3] = f.w;
        }
        if (cnt) n.c[g] = __ldcs(reinterpret_cast<const uint32_t*>(cnt + i));
        if (mk) n.m[g] = mk[i >> 5] >> (i & 31);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const int i = i0 + place(g, j);
          n.x[g][j] = i < last ? (BF16 ? bf2f(lb[i]) : lf[i]) : 0.f;
          if (cnt && i < last) n.c[g] |= (uint32_t)cnt[i] << (8 * j);
          if (mk && i < last && !((mk[i >> 5] >> (i & 31)) & 1u)) n.m[g] &= ~(1u << j);
        }
      }
    }
  };
  Entries next;
  load(first, next);
  const float rho = cnt && a.repetition ? a.repetition[row] : 1.f;
  const float fr = cnt && a.frequency ? a.frequency[row] : 0.f, pr = cnt && a.presence ? a.presence[row] : 0.f;
  if (t < kTable && rho != 1.f) pw[t] = powf(rho, (float)t);
  int b0 = 0, b1 = 0;
  if (a.bias_ptr) {
    b0 = a.bias_ptr[row];
    b1 = a.bias_ptr[row + 1];
    if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
      set_error(a.err, kErrBounds);
      b0 = b1 = 0;
    }
  }
  // The list's 128 entries from b on: those of [i0, i1), gathered in list order. All threads call it.
  auto gather = [&](int b, int i0, int i1) {
    const int id = b + t < b1 ? a.bias_ids[b + t] : i0 - 1, lane = t & 31, wid = t >> 5;
    if (b + t < b1 && (id < 0 || id >= a.V)) set_error(a.err, kErrBounds);
    const bool in = id >= i0 && id < i1;
    const unsigned hit = __ballot_sync(0xffffffffu, in);
    __syncthreads();                         // the entries before are used
    if (lane == 0) wn[wid] = __popc(hit);
    __syncthreads();
    int at = __popc(hit & ((1u << lane) - 1)), total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < wid) at += wn[w];
      total += wn[w];
    }
    if (in) {
      ids[at] = id;
      vals[at] = a.bias_vals[b + t];
    }
    __syncthreads();
    return total;
  };
  const bool longer = b1 - b0 > kThreads;    // a list that does not fit is gathered tile by tile
  int nb = 0;
  if (longer || b0 == b1) __syncthreads();
  else nb = gather(b0, first, last);
  for (int i0 = first; i0 < last; i0 += kTile) {
    Entries e = next;
    if (i0 + kTile < last) load(i0 + kTile, next);
    float x[kGroups][kPer];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      if constexpr (VEC && BF16) {
        const uint32_t u0 = __float_as_uint(e.x[g][0]), u1 = __float_as_uint(e.x[g][1]);
        x[g][0] = __uint_as_float(u0 << 16); x[g][1] = __uint_as_float(u0 & 0xFFFF0000u);
        x[g][2] = __uint_as_float(u1 << 16); x[g][3] = __uint_as_float(u1 & 0xFFFF0000u);
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) x[g][j] = e.x[g][j];
      }
      if (e.c[g] == 0) continue;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const uint32_t k = (e.c[g] >> (8 * j)) & 0xFFu;
        if (k == 0) continue;
        float& v = x[g][j];
        if (rho != 1.f && v != 0.f) {        // 0 stays 0 even where rho^c overflows
          // a quotient: 1 / rho^c is rounded once more, and overflows where rho^c is below 2^-128
          const float f = k < kTable ? pw[k] : powf(rho, (float)k);
          v = v < 0.f ? v * f : v / f;
        }
        v = v - fr * (float)k - pr;
      }
    }
    // the thread that holds an entry adds its biases one after the other (repeated tokens add up)
    for (int b = b0; b < b1; b += kThreads) {
      if (longer) nb = gather(b, i0, min(last, i0 + kTile));
      for (int n = 0; n < nb; ++n) {
        const int at = ids[n] - i0;
        if (at < 0 || at >= kTile) continue;
        const int o = at % (kThreads * kPer), gs = at / (kThreads * kPer);
        if ((VEC ? o / kPer : o % kThreads) != t) continue;
        const int js = VEC ? o % kPer : o / kThreads;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int j = 0; j < kPer; ++j)
            if (g == gs && j == js) x[g][j] += vals[n];
      }
    }
    float* out = a.out + (size_t)row * a.ld_out + i0;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (!((e.m[g] >> j) & 1u)) x[g][j] = -INFINITY;
      if constexpr (VEC) {
        if (i0 + place(g, 0) < last)
          __stcs(reinterpret_cast<float4*>(out + place(g, 0)), make_float4(x[g][0], x[g][1], x[g][2], x[g][3]));
      } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (i0 + place(g, j) < last) out[place(g, j)] = x[g][j];
      }
    }
  }
}

}  // namespace

void launch_logit_rules(const LogitRulesArgs& a, cudaStream_t st) {
  if (a.B <= 0 || a.V <= 0) return;
  auto mult = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  const bool vec = a.V % 4 == 0 && a.ld_in % 4 == 0 && a.ld_out % 4 == 0 && mult(a.logits, 16) && mult(a.out, 16) &&
                   mult(a.counts, 4);
  // stretches of up to eight tiles, fewer while that leaves less than two CTAs for each of 148 SMs
  const int64_t all = (a.V + kTile - 1) / kTile;
  const int tiles = (int)max((int64_t)1, min((int64_t)8, all * a.B / (2 * 148)));
  const dim3 grid((unsigned)((all + tiles - 1) / tiles), a.B);
  if (vec) {
    if (a.bf16) logit_rules_kernel<true, true><<<grid, kThreads, 0, st>>>(a, tiles);
    else logit_rules_kernel<true, false><<<grid, kThreads, 0, st>>>(a, tiles);
  } else {
    if (a.bf16) logit_rules_kernel<false, true><<<grid, kThreads, 0, st>>>(a, tiles);
    else logit_rules_kernel<false, false><<<grid, kThreads, 0, st>>>(a, tiles);
  }
}

}  // namespace air
