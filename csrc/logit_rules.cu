// What a request asks of its logits before sampling, in one pass over the vocabulary:
//   x -> x / rho^c (x > 0) or x * rho^c          repetition penalty, c = the token's count so far
//     -> x - c * frequency - [c > 0] * presence
//     -> x + bias[token]                          (a short list of tokens per row)
//     -> -inf where the grammar's allow bit is 0
// Memory-bound: a CTA takes 2048 entries of one row and every thread eight of them. A masked
// entry is selected away, so whatever its logit holds (NaN, infinities) does not get through.
#include "common.cuh"
#include "logit_rules.h"

namespace air {

namespace {

constexpr int kThreads = 256, kPer = 8, kTile = kThreads * kPer;

// VEC: eight neighbouring entries per thread in 16-byte accesses (rows and pointers aligned for
// it, V a multiple of 8); otherwise entries t, t + 256, ... of the tile one by one.
template <bool VEC, bool BF16>
__global__ void __launch_bounds__(kThreads) logit_rules_kernel(const LogitRulesArgs a) {
  const int row = blockIdx.y, i0 = blockIdx.x * kTile, t = threadIdx.x;
  const int i1 = min(a.V, i0 + kTile);
  auto index = [&](int j) { return VEC ? i0 + kPer * t + j : i0 + t + kThreads * j; };
  float x[kPer];
  uint8_t c[kPer];
  const float* lf = static_cast<const float*>(a.logits) + (size_t)row * a.ld_in;
  const __nv_bfloat16* lb = static_cast<const __nv_bfloat16*>(a.logits) + (size_t)row * a.ld_in;
  int64_t crow = -1;
  if (a.counts) {
    crow = a.count_row ? a.count_row[row] : row;
    if (crow >= a.S) {
      set_error(a.err, kErrBounds);
      crow = -1;
    }
  }
  const uint8_t* cnt = crow >= 0 ? a.counts + (size_t)crow * a.V : nullptr;
  if constexpr (VEC) {
    const int i = index(0);
    if (i < i1) {
      if constexpr (BF16) {
        bf16x8_to_f32(*reinterpret_cast<const uint4*>(lb + i), x);
      } else {
        const float4 lo = *reinterpret_cast<const float4*>(lf + i), hi = *reinterpret_cast<const float4*>(lf + i + 4);
        x[0] = lo.x; x[1] = lo.y; x[2] = lo.z; x[3] = lo.w;
        x[4] = hi.x; x[5] = hi.y; x[6] = hi.z; x[7] = hi.w;
      }
      const uint2 u = cnt ? *reinterpret_cast<const uint2*>(cnt + i) : make_uint2(0, 0);
#pragma unroll
      for (int j = 0; j < kPer; ++j) c[j] = (uint8_t)((j < 4 ? u.x : u.y) >> (8 * (j & 3)));
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = index(j);
      x[j] = i < i1 ? (BF16 ? bf2f(lb[i]) : lf[i]) : 0.f;
      c[j] = cnt && i < i1 ? cnt[i] : 0;
    }
  }
  if (cnt) {
    const float rho = a.repetition ? a.repetition[row] : 1.f;
    const float fr = a.frequency ? a.frequency[row] : 0.f, pr = a.presence ? a.presence[row] : 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (VEC && index(0) >= i1) break;
      if (c[j] == 0) continue;
      const float n = (float)c[j];
      if (rho != 1.f && x[j] != 0.f) {     // 0 stays 0 even where rho^c overflows
        const float f = powf(rho, n);
        x[j] = x[j] > 0.f ? x[j] / f : x[j] * f;
      }
      x[j] = x[j] - fr * n - pr;
    }
  }
  if (a.bias_ptr) {
    // the row's list, 256 entries at a time: those of this tile are gathered in list order, and
    // the thread that holds an entry adds them one after the other (repeated tokens add up)
    __shared__ int ids[kThreads];
    __shared__ float vals[kThreads];
    __shared__ int wn[kThreads / 32];
    int b0 = a.bias_ptr[row], b1 = a.bias_ptr[row + 1];
    if (b0 < 0 || b1 < b0 || b1 > a.n_bias) {
      set_error(a.err, kErrBounds);
      b0 = b1 = 0;
    }
    const int lane = t & 31, wid = t >> 5;
    for (int b = b0; b < b1; b += kThreads) {
      const int id = b + t < b1 ? a.bias_ids[b + t] : -1;
      if (b + t < b1 && (id < 0 || id >= a.V)) set_error(a.err, kErrBounds);
      const bool in = id >= i0 && id < i1;
      const unsigned m = __ballot_sync(0xffffffffu, in);
      if (lane == 0) wn[wid] = __popc(m);
      __syncthreads();
      int at = 0, total = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < wid) at += wn[w];
        total += wn[w];
      }
      if (in) {
        at += __popc(m & ((1u << lane) - 1));
        ids[at] = id - i0;
        vals[at] = a.bias_vals[b + t];
      }
      __syncthreads();
      for (int e = 0; e < total; ++e) {
        const int o = ids[e];
        if ((VEC ? o / kPer : o % kThreads) != t) continue;
        const int js = VEC ? o % kPer : o / kThreads;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (j == js) x[j] += vals[e];
      }
      __syncthreads();
    }
  }
  if (a.mask) {
    const uint32_t* mk = a.mask + (size_t)row * ((a.V + 31) / 32);
    if constexpr (VEC) {
      if (index(0) < i1) {
        const uint32_t m = mk[index(0) >> 5] >> (index(0) & 31);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (!((m >> j) & 1u)) x[j] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = index(j);
        if (i < i1 && !((mk[i >> 5] >> (i & 31)) & 1u)) x[j] = -INFINITY;
      }
    }
  }
  float* out = a.out + (size_t)row * a.ld_out;
  if constexpr (VEC) {
    const int i = index(0);
    if (i < i1) {
      *reinterpret_cast<float4*>(out + i) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(out + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (index(j) < i1) out[index(j)] = x[j];
  }
}

}  // namespace

void launch_logit_rules(const LogitRulesArgs& a, cudaStream_t st) {
  if (a.B <= 0 || a.V <= 0) return;
  auto mult = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  const bool vec = a.V % 8 == 0 && a.ld_in % 8 == 0 && a.ld_out % 4 == 0 && mult(a.logits, 16) && mult(a.out, 16) &&
                   mult(a.counts, 8);
  const dim3 grid((a.V + kTile - 1) / kTile, a.B);
  if (vec) {
    if (a.bf16) logit_rules_kernel<true, true><<<grid, kThreads, 0, st>>>(a);
    else logit_rules_kernel<true, false><<<grid, kThreads, 0, st>>>(a);
  } else {
    if (a.bf16) logit_rules_kernel<false, true><<<grid, kThreads, 0, st>>>(a);
    else logit_rules_kernel<false, false><<<grid, kThreads, 0, st>>>(a);
  }
}

}  // namespace air
