// Linear attention with one decay per head: the token-by-token kernel that takes every shape, and
// the single-token step of the decode batch.
//   S_t = exp(g_t) S_{t-1} + v_t k_t^T,   o_t = scale * S_t q_t
// The state stays f32 in registers and in memory; q, k and v are widened to f32 when they are
// loaded and the output is rounded once.
#include "common.cuh"
#include "linear_attn.h"

namespace air {

namespace {

template <typename T>
AIR_DEVICE float ld_f(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}
template <typename T>
AIR_DEVICE void st_f(T* p, float v) {
  if constexpr (sizeof(T) == 2) *p = f2bf(v);
  else *p = v;
}
// four consecutive elements, 4 * sizeof(T) aligned
template <typename T>
AIR_DEVICE float4 ld4_f(const T* p) {
  if constexpr (sizeof(T) == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
    const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    return make_float4(lo.x, lo.y, hi.x, hi.y);
  } else {
    return *reinterpret_cast<const float4*>(p);
  }
}

// S <- exp(g) S + u without the bias of a rounded factor: near 1 the decay is applied as
// S + expm1(g) S, so a slow head that multiplies by the same factor for thousands of tokens does not
// drift (exp(g) rounded to f32 is off by up to 2^-25 the same way every token).
struct Decay {
  float f;
  bool slow;
  AIR_DEVICE explicit Decay(float g) : slow(g > -0.5f) { f = slow ? expm1f(g) : expf(g); }
  AIR_DEVICE float operator()(float s, float u) const { return slow ? s + fmaf(s, f, u) : fmaf(s, f, u); }
};

struct SeqView {
  int t0, t1;        // tokens [t0, t1)
  int64_t slot;      // state row, -1: none
  bool init;         // the state row holds the incoming state
};

AIR_DEVICE SeqView seq_view(const LinAttnArgs& a, int n) {
  SeqView s;
  s.t0 = a.cu ? a.cu[n] : n;
  s.t1 = a.cu ? a.cu[n + 1] : a.whole ? a.T : n + 1;
  s.slot = a.state ? (a.slots ? (int64_t)a.slots[n] : (int64_t)n) : -1;
  if (s.t0 < 0 || s.t1 < s.t0 || s.t1 > a.T) {   // skipped: no tokens, and its state stays
    set_error(a.err, kErrBounds);
    s.t0 = s.t1 = 0;
    s.slot = -1;
  }
  if (s.slot < -1 || s.slot >= a.S) {
    set_error(a.err, kErrBounds);
    s.slot = -1;
  }
  s.init = s.slot >= 0 && (a.has_state ? a.has_state[n] != 0 : a.has_state_all != 0);
  return s;
}

// Grid (N * H, ceil(dv / 32)), four warps of eight state rows: lane l holds columns l + 32 j of its
// warp's rows for the whole sequence. Per token a row costs dk multiply-adds for the update and dk
// for the output, the row sums are five shuffles. Latency-bound (one token after the other), which
// the block form of the tensor-core kernel avoids; this one takes what that does not: f32 inputs,
// head sizes other than 64 and 128, rows that are not 16-byte aligned, and calls of a dozen tokens
// (0.55 us a token at 32 heads of 128).
template <typename T, int J>
__global__ void __launch_bounds__(128) linear_scan_kernel(const LinAttnArgs a) {
  constexpr int R = 8;
  const int n = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const int lane = threadIdx.x & 31;
  const int r0 = blockIdx.y * 32 + (threadIdx.x >> 5) * R;
  if (r0 >= a.dv) return;
  const SeqView sv = seq_view(a, n);
  float S[R][J];
  float* st = sv.slot >= 0 ? a.state + ((size_t)sv.slot * a.H + h) * a.dv * a.dk : nullptr;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = lane + 32 * j;
      S[r][j] = sv.init && r0 + r < a.dv && c < a.dk ? st[(size_t)(r0 + r) * a.dk + c] : 0.f;
    }
  const T* q = static_cast<const T*>(a.q) + (int64_t)(h / a.q_div) * a.qs_h;
  const T* k = static_cast<const T*>(a.k) + (int64_t)(h / a.k_div) * a.ks_h;
  const T* v = static_cast<const T*>(a.v) + (int64_t)(h / a.v_div) * a.vs_h;
  T* out = static_cast<T*>(a.out) + (int64_t)h * a.os_h;
  if (a.zero_pad && !st) {
    if (lane < R && r0 + lane < a.dv)
      for (int t = sv.t0; t < sv.t1; ++t) st_f(out + t * a.os_t + r0 + lane, 0.f);
    return;
  }
  float kn[J], qn[J], vn = 0.f, gn = 0.f;       // the next token's operands, loaded one token ahead
  auto fetch = [&](int t) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = lane + 32 * j;
      kn[j] = c < a.dk ? ld_f(k + t * a.ks_t + c) : 0.f;
      qn[j] = c < a.dk ? ld_f(q + t * a.qs_t + c) : 0.f;
    }
    vn = lane < R && r0 + lane < a.dv ? ld_f(v + t * a.vs_t + r0 + lane) : 0.f;
    gn = a.decay[t * a.decay_t + h];
  };
  if (sv.t0 < sv.t1) fetch(sv.t0);
  for (int t = sv.t0; t < sv.t1; ++t) {
    float kt[J], qt[J];
#pragma unroll
    for (int j = 0; j < J; ++j) { kt[j] = kn[j]; qt[j] = qn[j]; }
    const float vt = vn;
    const Decay dec(gn);
    if (t + 1 < sv.t1) fetch(t + 1);
    float o = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float vr = __shfl_sync(0xffffffffu, vt, r);
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        S[r][j] = dec(S[r][j], vr * kt[j]);
        d = fmaf(S[r][j], qt[j], d);
      }
      d = warp_sum(d);
      if (lane == r) o = d;
    }
    if (lane < R && r0 + lane < a.dv) st_f(out + t * a.os_t + r0 + lane, o * a.scale);
  }
  if (st) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = lane + 32 * j;
        if (r0 + r < a.dv && c < a.dk) st[(size_t)(r0 + r) * a.dk + c] = S[r][j];
      }
  }
}

// One token per sequence. A warp takes R = 8 state rows of one (sequence, head): all its loads are
// issued before the first use (R x 512 bytes of the state), the update and the product with q
// follow in registers, and the eight row sums share one butterfly (9 shuffles for 8 rows at
// dk = 128). Bound by the state's 2 x 4 dv dk bytes per head: 64 rows x 32 heads of 128 take 43.9 us of a
// 41.9 us floor (6.2 TB/s), 251 x 64 heads of 128 x 64 159 us; one row of 32 heads 3.0 us, launch latency.
template <typename T, int DK>
__global__ void __launch_bounds__(128) linear_step_kernel(const LinAttnArgs a) {
  constexpr int LPR = DK / 4;              // lanes per state row
  constexpr int RPI = 32 / LPR;            // rows per load of the warp
  constexpr int R = 8, I = R / RPI;        // rows and loads per warp
  const int lane = threadIdx.x & 31;
  const int tiles = a.dv / R;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.N * a.H * tiles) return;
  const int tile = (int)(item % tiles);
  const int64_t nh = item / tiles;
  const int n = (int)(nh / a.H), h = (int)(nh % a.H);
  const int r0 = tile * R, sub = lane / LPR, c = (lane % LPR) * 4;
  T* out = static_cast<T*>(a.out) + n * a.os_t + (int64_t)h * a.os_h + r0;
  const SeqView sv = seq_view(a, n);
  if (sv.slot < 0) {                       // a padding row of the batch
    if (lane < R) st_f(out + lane, 0.f);
    return;
  }
  float4* st = reinterpret_cast<float4*>(a.state + (((size_t)sv.slot * a.H + h) * a.dv + r0 + sub) * DK + c);
  float4 s[I];
#pragma unroll
  for (int i = 0; i < I; ++i) s[i] = st[i * RPI * LPR];
  const float4 kt = ld4_f(static_cast<const T*>(a.k) + n * a.ks_t + (int64_t)(h / a.k_div) * a.ks_h + c);
  const float4 qt = ld4_f(static_cast<const T*>(a.q) + n * a.qs_t + (int64_t)(h / a.q_div) * a.qs_h + c);
  const float vt = lane < R ? ld_f(static_cast<const T*>(a.v) + n * a.vs_t + (int64_t)(h / a.v_div) * a.vs_h + r0 + lane) : 0.f;
  const Decay dec(a.decay[n * a.decay_t + h]);
  float d[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const float vr = __shfl_sync(0xffffffffu, vt, i * RPI + sub);
    s[i].x = dec(s[i].x, vr * kt.x);
    s[i].y = dec(s[i].y, vr * kt.y);
    s[i].z = dec(s[i].z, vr * kt.z);
    s[i].w = dec(s[i].w, vr * kt.w);
    st[i * RPI * LPR] = s[i];
    d[i] = fmaf(s[i].x, qt.x, fmaf(s[i].y, qt.y, fmaf(s[i].z, qt.z, s[i].w * qt.w)));
  }
  // Row sums. Each halving step sends one half of the rows to the partner lane and keeps the other.
  int row = 0;                             // the load index whose sum this lane ends up with
  int off = LPR / 2;
#pragma unroll
  for (int m = I; m > 1; m >>= 1, off >>= 1) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < m / 2; ++i) {
      const float send = up ? d[i] : d[i + m / 2];
      const float keep = up ? d[i + m / 2] : d[i];
      d[i] = keep + __shfl_xor_sync(0xffffffffu, send, off);
    }
    if (up) row += m / 2;
  }
  float o = d[0];
#pragma unroll
  for (; off > 0; off >>= 1) o += __shfl_xor_sync(0xffffffffu, o, off);
  if ((lane % (LPR / I)) == 0) st_f(out + row * RPI + sub, o * a.scale);
}

}  // namespace

void launch_linear_scan(const LinAttnArgs& a, bool f32, cudaStream_t st) {
  const dim3 grid((unsigned)(a.N * a.H), (unsigned)((a.dv + 31) / 32));
#define AIR_SCAN(J)                                                              \
  (f32 ? linear_scan_kernel<float, J><<<grid, 128, 0, st>>>(a)                   \
       : linear_scan_kernel<__nv_bfloat16, J><<<grid, 128, 0, st>>>(a))
  if (a.dk <= 64) AIR_SCAN(2);
  else if (a.dk <= 128) AIR_SCAN(4);
  else AIR_SCAN(8);
#undef AIR_SCAN
}

bool linear_step_supported(const LinAttnArgs& a, bool f32) {
  const int64_t e = f32 ? 4 : 2;
  auto ok4 = [&](const void* p, int64_t s0, int64_t s1) {   // four elements at a time
    return reinterpret_cast<uintptr_t>(p) % (4 * e) == 0 && s0 % 4 == 0 && s1 % 4 == 0;
  };
  return (a.dk == 64 || a.dk == 128) && a.dv % 8 == 0 && a.state &&
         reinterpret_cast<uintptr_t>(a.state) % 16 == 0 && ok4(a.q, a.qs_t, a.qs_h) && ok4(a.k, a.ks_t, a.ks_h);
}

void launch_linear_step(const LinAttnArgs& a, bool f32, cudaStream_t st) {
  const int64_t warps = (int64_t)a.N * a.H * (a.dv / 8);
  const unsigned grid = (unsigned)((warps + 3) / 4);
  if (a.dk == 128) {
    if (f32) linear_step_kernel<float, 128><<<grid, 128, 0, st>>>(a);
    else linear_step_kernel<__nv_bfloat16, 128><<<grid, 128, 0, st>>>(a);
  } else {
    if (f32) linear_step_kernel<float, 64><<<grid, 128, 0, st>>>(a);
    else linear_step_kernel<__nv_bfloat16, 64><<<grid, 128, 0, st>>>(a);
  }
}

}  // namespace air
