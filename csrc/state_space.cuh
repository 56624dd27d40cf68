// Device helpers of the state-space operators.
#pragma once
#include "common.cuh"
#include "state_space.h"

namespace air {

template <typename T>
AIR_DEVICE float to_f(T v) {
  if constexpr (sizeof(T) == 2) return bf2f(v);
  else return v;
}
template <typename T>
AIR_DEVICE T from_f(float v) {
  if constexpr (sizeof(T) == 2) return f2bf(v);
  else return v;
}

constexpr float kLog2e = 1.44269504f;

// ---- paired f32 arithmetic
using f2 = unsigned long long;       // two floats, the operand of the paired instructions
AIR_DEVICE f2 pack2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
AIR_DEVICE f2 dup2(float a) { return pack2(a, a); }
AIR_DEVICE void unpack2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
AIR_DEVICE f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
AIR_DEVICE f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AIR_DEVICE f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
AIR_DEVICE float exp2_fast(float u) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u));
  return e;
}

// V consecutive elements as f32: one 16- or 8-byte access, or single elements (V = 1).
template <typename T, int V>
AIR_DEVICE void load_v(const T* p, float* f) {
  if constexpr (V == 1) f[0] = to_f(*p);
  else if constexpr (sizeof(T) == 2 && V % 8 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 8) bf16x8_to_f32(*reinterpret_cast<const uint4*>(p + i), f + i);
  }
  else if constexpr (sizeof(T) == 2 && V == 4) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    f[0] = lo.x; f[1] = lo.y; f[2] = hi.x; f[3] = hi.y;
  } else if constexpr (sizeof(T) == 2 && V == 2) {
    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
    f[0] = lo.x; f[1] = lo.y;
  } else if constexpr (V == 2) {
    const float2 lo = *reinterpret_cast<const float2*>(p);
    f[0] = lo.x; f[1] = lo.y;
  } else {
    static_assert(sizeof(T) == 4 && V % 4 == 0, "");
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 u = *reinterpret_cast<const float4*>(p + i);
      f[i] = u.x; f[i + 1] = u.y; f[i + 2] = u.z; f[i + 3] = u.w;
    }
  }
}
template <typename T, int V>
AIR_DEVICE void store_v(T* p, const float* f) {
  if constexpr (V == 1) *p = from_f<T>(f[0]);
  else if constexpr (sizeof(T) == 2 && V == 8) *reinterpret_cast<uint4*>(p) = f32_to_bf16x8(f);
  else if constexpr (sizeof(T) == 2 && V == 4) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(f[0], f[1]), hi = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  } else if constexpr (sizeof(T) == 2 && V == 2) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(f[0], f[1]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
  } else {
    static_assert(sizeof(T) == 4 && V % 4 == 0, "");
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  }
}

// B bytes from global to shared memory (4, 8 or a multiple of 16), zeros instead where `in` is false.
template <int B>
AIR_DEVICE void copy_async(void* dst, const void* src, bool in) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  if constexpr (B >= 16) {
#pragma unroll
    for (int i = 0; i < B; i += 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                   ::"r"(d + i), "l"(static_cast<const char*>(src) + i), "r"(in ? 16 : 0) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(d), "l"(src), "n"(B), "r"(in ? B : 0) : "memory");
  }
}

// ---- E elements (2 or 4) of a row that starts anywhere, as the 4-byte words that hold them. bf16 at an odd place takes a
// word more, of which half belongs to a neighbour: read, never written. `odd`: the first element's half of its word.
template <typename T>
AIR_DEVICE int odd_half(const T* p) { return sizeof(T) == 4 ? 0 : reinterpret_cast<uintptr_t>(p) >> 1 & 1; }
// Asynchronously to dst (E + 2 elements of bf16, E of f32), for the first `live` elements; `any` is readable, zeros where
// there is nothing to read.
template <typename T, int E>
AIR_DEVICE void copy_words(T* dst, const T* p, const void* any, int odd, int live) {
  constexpr int per = 4 / sizeof(T);
#pragma unroll
  for (int j = 0; j < E / per + per - 1; ++j) {
    const bool some = j * per - odd < live;
    copy_async<4>(dst + j * per, some ? static_cast<const void*>(p - odd + j * per) : any, some);
  }
}
// What copy_words put at p (aligned to 2 E elements of bf16, E of f32). Past `live` it may be a neighbour's.
template <typename T, int E>
AIR_DEVICE void read_words(const T* p, int odd, float* f) {
  if constexpr (sizeof(T) == 4) load_v<T, E>(p, f);
  else {
    uint32_t v[E / 2 + 1];
    if constexpr (E == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      v[0] = u.x; v[1] = u.y; v[2] = u.z;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      v[0] = u.x; v[1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      const uint32_t two = __funnelshift_r(v[i], v[i + 1], odd * 16);
      f[2 * i] = __uint_as_float(two << 16);
      f[2 * i + 1] = __uint_as_float(two & 0xffff0000u);
    }
  }
}
// The first `live` of E values to a row that starts anywhere, in words as far as they are its own.
template <typename T, int E>
AIR_DEVICE void store_words(T* o, const float* y, int live) {
  if (sizeof(T) == 2 && live == E) {
    if (!odd_half(o)) {
#pragma unroll
      for (int i = 0; i < E; i += 2) store_v<T, 2>(o + i, y + i);
    } else {
      o[0] = from_f<T>(y[0]);
#pragma unroll
      for (int i = 1; i + 1 < E; i += 2) store_v<T, 2>(o + i, y + i);
      o[E - 1] = from_f<T>(y[E - 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < live) o[i] = from_f<T>(y[i]);
  }
}

// 1 / (1 + exp(-x)) and x / (1 + exp(-x)). Subnormals count as zero in the exponential and the reciprocal: without that
// each of them costs three to four instructions more, for values below 2^-126.
AIR_DEVICE float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
AIR_DEVICE float sigmoid_f(float x) { return rcp_fast(1.f + exp2_fast(x * -kLog2e)); }
AIR_DEVICE float silu_f(float x) { return x * sigmoid_f(x); }
AIR_DEVICE f2 silu2(f2 x) {
  float a, b;
  unpack2(mul2(x, dup2(-kLog2e)), a, b);
  unpack2(add2(pack2(exp2_fast(a), exp2_fast(b)), dup2(1.f)), a, b);
  return mul2(x, pack2(rcp_fast(a), rcp_fast(b)));
}

// log(1 + exp(x)) = max(x, 0) + log(1 + u), u = exp(-|x|) in [0, 1]. The logarithm is u P(u) with P of degree 8 (equal
// ripple of the relative error, computed for this interval: 6.5e-8, 1.8e-7 with the roundings): small steps keep their
// relative accuracy, which the logarithm of the rounded sum 1 + u would lose, and it needs no special-function unit.
AIR_DEVICE float softplus_f(float x) {
  const float u = exp2_fast(fabsf(x) * -kLog2e);
  float p = fmaf(0.00523269409f, u, -0.0295052398f);
  p = fmaf(p, u, 0.0782259554f);
  p = fmaf(p, u, -0.136632457f);
  p = fmaf(p, u, 0.191060066f);
  p = fmaf(p, u, -0.24842982f);
  p = fmaf(p, u, 0.333190978f);
  p = fmaf(p, u, -0.499994934f);
  p = fmaf(p, u, 0.99999994f);
  return x != x ? x : fmaf(p, u, fmaxf(x, 0.f));
}

// A state's step: 2^u h + in, u = delta A log2(e). Beside slow decays, |u| <= log2(e) / 32, it is (2^u - 1) h + (h + in): so a
// slow decay keeps its rate, where 2^u itself, rounded to 24 bits, would change a rate of 2^-10 by 2^-14 of itself at every
// token. 2^u - 1 is a quadratic times u there (equal ripple of the relative error, computed for this interval: 3.2e-7, 4.2e-7
// with the roundings). Beyond it 2^u h is rounded at its own size, not at that of the h it forgets; the exponential is then
// off by at most 7.6e-6 of the rate.
constexpr float kNearDecay = 0.0450842196f, kDecay0 = 0.693147182f, kDecay1 = 0.24024117f, kDecay2 = 0.0555041097f;
AIR_DEVICE float decayed(float u, float h, float dx, float b) {
  const float p = fmaf(fmaf(kDecay2, u, kDecay1), u, kDecay0) * u;
  const bool slow = fabsf(u) <= kNearDecay;
  return fmaf(slow ? p : exp2_fast(u), h, fmaf(dx, b, slow ? h : 0.f));
}

struct SeqRange {
  int t0, t1;        // tokens [t0, t1)
  int64_t slot;      // state row, -1: none
  bool init;         // the state row holds the incoming state
};

// Sequence n of the batch. Bad offsets: no tokens, and its state stays. A state row out of range: none.
AIR_DEVICE SeqRange seq_range(const SeqArgs& a, int n, bool report = true) {
  SeqRange s;
  s.t0 = a.cu ? a.cu[n] : a.step ? n : 0;
  s.t1 = a.cu ? a.cu[n + 1] : a.step ? n + 1 : a.T;
  s.slot = a.slots ? (int64_t)a.slots[n] : a.S > 0 ? (int64_t)n : -1;
  if (s.t0 < 0 || s.t1 < s.t0 || s.t1 > a.T) {
    if (report) set_error(a.err, kErrBounds);
    s.t0 = s.t1 = 0;
    s.slot = -1;
  }
  if (s.slot < -1 || s.slot >= a.S) {
    if (report) set_error(a.err, kErrBounds);
    s.slot = -1;
  }
  s.init = s.slot >= 0 && (a.has_state ? a.has_state[n] != 0 : a.has_state_all != 0);
  return s;
}

// State row of single token n (SeqArgs with `step`), -1: none.
AIR_DEVICE int64_t state_row(const SeqArgs& a, int n, bool report) {
  const int64_t slot = a.slots ? (int64_t)a.slots[n] : (int64_t)n;
  if (slot >= 0 && slot < a.S) return slot;
  if (slot != -1 && report) set_error(a.err, kErrBounds);
  return -1;
}

// The sequence that holds token t among rising offsets, by the whole warp: the last n with cu[n] <= t, in steps that
// look at 32 offsets each. Whatever the offsets are, the result is in [0, N) and the caller checks its range.
AIR_DEVICE int seq_of_token(const int* cu, int N, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = N;                        // the sequence is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int i = lo + (lane + 1) * step;
    const unsigned up = __ballot_sync(0xffffffffu, i < hi && cu[i] <= t);
    const int run = __ffs(~up) - 1;          // lanes whose offset is not past t (32: ffs of 0 is 0)
    const int k = up == 0xffffffffu ? 32 : run;
    hi = min(hi, lo + (k + 1) * step);
    lo += k * step;
  }
  return lo;
}

// One bit for each of the 32 tokens from t0: whether its sequence is sound and holds its W - 1 predecessors. By the
// whole warp.
template <int W>
AIR_DEVICE unsigned tokens_inside(const SeqArgs& a, int t0) {
  const int t = t0 + (threadIdx.x & 31);
  bool in = false;
  if (a.cu) {
    for (int n = a.N ? seq_of_token(a.cu, a.N, t0) : 0; n < a.N; ++n) {
      const int lo = a.cu[n], hi = a.cu[n + 1];
      if (lo >= t0 + 32) break;
      if (lo >= 0 && hi <= a.T) in |= t - lo >= W - 1 && t < hi;
    }
  } else {
    in = t >= W - 1 && t < a.T;
  }
  return __ballot_sync(0xffffffffu, in);
}

}  // namespace air
