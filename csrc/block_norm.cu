// The way from a block's output to the next block's input in one pass:
//   h = y;  h = h rsqrt(mean(h^2) + eps) (post + w_offset);  h = h act(gate);
//   r = resid + scale h;  out = r rsqrt(mean(r^2) + eps) (w + w_offset)
// each step but the sum optional. A block has a row in registers, so y, gate and the residual are read once, r and out
// written once and nothing else goes to memory. All steps are f32 on the unrounded values of the step before; out and (in
// bf16) the stored residual are rounded once. Memory-bound with many rows: 6007 x 4096 with bf16 y and gate, f32 residual
// and both norms takes 59 us (5.8 TB/s, floor 52.6), f32 y 69 (floor 67.6), 4094 columns 87 and 4095 135 (pairs and
// single elements); one row 2.9 us, the latency of the loads and one or two block reductions.
#include <algorithm>

#include "state_space.cuh"

namespace air {

namespace {

// Sum over the block with one barrier: `red` alternates between two places, so a sum may be written while the one before
// is still read.
template <int NT>
struct RowSum {
  float (*red)[NT / 32];
  int place = 0;
  AIR_DEVICE float operator()(float v) {
    v = warp_sum(v);
    if constexpr (NT > 32) {
      if ((threadIdx.x & 31) == 0) red[place][threadIdx.x >> 5] = v;
      __syncthreads();
      const int lane = threadIdx.x & 31;
      v = warp_sum(lane < NT / 32 ? red[place][lane] : 0.f);
      place ^= 1;
    }
    return v;
  }
  // 1 / rms of a row whose squares add up to `ss` over the block
  AIR_DEVICE float inv_rms(float ss, const BlockNormArgs& a) { return rsqrtf((*this)(ss) / (float)a.K + a.eps); }
};

// NT threads, J groups of E consecutive elements per thread, E NT elements apart.
template <typename TY, typename TR, int NT, int J, int E>
__global__ void __launch_bounds__(NT) block_norm_kernel(const BlockNormArgs a) {
  __shared__ float red[2][NT / 32];
  RowSum<NT> sum{red};
  const int64_t t = blockIdx.x;
  const TY* y = static_cast<const TY*>(a.y) + t * a.ldy;
  float h[J][E];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = E * (threadIdx.x + NT * j);
    if (i < a.K) load_v<TY, E>(y + i, h[j]);
    else {
#pragma unroll
      for (int e = 0; e < E; ++e) h[j][e] = 0.f;
    }
  }
  if (a.post) {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(h[j][e], h[j][e], ss);
    const float inv = sum.inv_rms(ss, a);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = E * (threadIdx.x + NT * j);
      if (i >= a.K) continue;
      float w[E];
      load_v<float, E>(a.post + i, w);
#pragma unroll
      for (int e = 0; e < E; ++e) h[j][e] *= inv * (w[e] + a.w_offset);
    }
  }
  if (a.gate) {
    const TY* gate = static_cast<const TY*>(a.gate) + t * a.ldg;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = E * (threadIdx.x + NT * j);
      if (i >= a.K) continue;
      float g[E];
      load_v<TY, E>(gate + i, g);
#pragma unroll
      for (int e = 0; e < E; ++e) h[j][e] *= a.act == 0 ? silu_f(g[e]) : a.act == 1 ? sigmoid_f(g[e]) : g[e];
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = E * (threadIdx.x + NT * j);
    if (i >= a.K) continue;
    float r[E], s[E];
    if (a.resid) load_v<TR, E>(static_cast<const TR*>(a.resid) + t * a.ldr + i, r);
    if (a.scale_row) load_v<float, E>(a.scale_row + i, s);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float f = a.scale_row ? s[e] : a.scale;
      h[j][e] = a.resid ? fmaf(f, h[j][e], r[e]) : f * h[j][e];
      ss = fmaf(h[j][e], h[j][e], ss);
    }
    if (a.resid_out) store_v<TR, E>(static_cast<TR*>(a.resid_out) + t * a.ldro + i, h[j]);
  }
  if (!a.out) return;
  const float inv = a.w ? sum.inv_rms(ss, a) : 1.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = E * (threadIdx.x + NT * j);
    if (i >= a.K) continue;
    float o[E];
    if (a.w) {
      load_v<float, E>(a.w + i, o);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = h[j][e] * inv * (o[e] + a.w_offset);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = h[j][e];
    }
    if (a.o_bf16) store_v<__nv_bfloat16, E>(static_cast<__nv_bfloat16*>(a.out) + t * a.ldo + i, o);
    else store_v<float, E>(static_cast<float*>(a.out) + t * a.ldo + i, o);
  }
}

// The same with many rows: a block takes every gridDim-th row and copies its next row's parts to shared memory while it
// works on one, each thread its own part, so nothing waits for other threads but the reductions.
template <typename TY, typename TR, int NT, int J>
__global__ void __launch_bounds__(NT) block_norm_rows_kernel(const BlockNormArgs a) {
  constexpr int E = 4;
  extern __shared__ __align__(16) uint8_t raw_smem[];
  __shared__ float red[2][NT / 32];
  RowSum<NT> sum{red};
  using Ys = TY[J][NT][E];
  using Rs = TR[J][NT][E];
  constexpr int stage = 2 * sizeof(Ys) + sizeof(Rs);
  auto ys = [&](int b, int which) -> Ys& { return *reinterpret_cast<Ys*>(raw_smem + b * stage + which * sizeof(Ys)); };
  auto rs = [&](int b) -> Rs& { return *reinterpret_cast<Rs*>(raw_smem + b * stage + 2 * sizeof(Ys)); };
  auto fetch = [&](int64_t t, int b) {
    if (t < a.T) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int i = E * (threadIdx.x + NT * j);
        if (i >= a.K) continue;
        copy_async<E * sizeof(TY)>(ys(b, 0)[j][threadIdx.x], static_cast<const TY*>(a.y) + t * a.ldy + i, true);
        if (a.gate) copy_async<E * sizeof(TY)>(ys(b, 1)[j][threadIdx.x], static_cast<const TY*>(a.gate) + t * a.ldg + i, true);
        if (a.resid) copy_async<E * sizeof(TR)>(rs(b)[j][threadIdx.x], static_cast<const TR*>(a.resid) + t * a.ldr + i, true);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(blockIdx.x, 0);
  int b = 0;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, b ^= 1) {
    fetch(t + gridDim.x, b ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    float h[J][E], w[J][E];
    auto load_weights = [&](const float* p, float (&f)[J][E]) {      // asked for before the reduction they wait for
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int i = E * (threadIdx.x + NT * j);
        if (i < a.K) load_v<float, E>(p + i, f[j]);
      }
    };
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (E * (threadIdx.x + NT * j) < a.K) load_v<TY, E>(ys(b, 0)[j][threadIdx.x], h[j]);
      else h[j][0] = h[j][1] = h[j][2] = h[j][3] = 0.f;
    }
    if (a.post) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) ss = fmaf(h[j][e], h[j][e], ss);
      load_weights(a.post, w);
      const float inv = sum.inv_rms(ss, a);
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) h[j][e] *= inv * (w[j][e] + a.w_offset);
    }
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = E * (threadIdx.x + NT * j);
      if (i >= a.K) continue;
      float g[E], r[E], s[E];
      if (a.gate) {
        load_v<TY, E>(ys(b, 1)[j][threadIdx.x], g);
#pragma unroll
        for (int e = 0; e < E; ++e) h[j][e] *= a.act == 0 ? silu_f(g[e]) : a.act == 1 ? sigmoid_f(g[e]) : g[e];
      }
      if (a.resid) load_v<TR, E>(rs(b)[j][threadIdx.x], r);
      if (a.scale_row) load_v<float, E>(a.scale_row + i, s);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = a.scale_row ? s[e] : a.scale;
        h[j][e] = a.resid ? fmaf(f, h[j][e], r[e]) : f * h[j][e];
        ss = fmaf(h[j][e], h[j][e], ss);
      }
      if (a.resid_out) store_v<TR, E>(static_cast<TR*>(a.resid_out) + t * a.ldro + i, h[j]);
    }
    if (!a.out) continue;
    if (a.w) load_weights(a.w, w);
    const float inv = a.w ? sum.inv_rms(ss, a) : 1.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int i = E * (threadIdx.x + NT * j);
      if (i >= a.K) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = a.w ? h[j][e] * inv * (w[j][e] + a.w_offset) : h[j][e];
      if (a.o_bf16) store_v<__nv_bfloat16, E>(static_cast<__nv_bfloat16*>(a.out) + t * a.ldo + i, o);
      else store_v<float, E>(static_cast<float*>(a.out) + t * a.ldo + i, o);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename TY, typename TR, int NT, int J>
bool launch_rows(const BlockNormArgs& a, cudaStream_t st) {
  constexpr int bytes = 2 * J * NT * 4 * (2 * sizeof(TY) + sizeof(TR));
  const int per_sm = std::min(std::min(32, 2048 / NT), 200 * 1024 / (bytes + 1024));
  if (a.T <= 148 * per_sm) return false;
  static unsigned long long done = 0;
  if (!set_max_smem_per_device(block_norm_rows_kernel<TY, TR, NT, J>, bytes, done)) return false;
  block_norm_rows_kernel<TY, TR, NT, J><<<148 * per_sm, NT, bytes, st>>>(a);
  return true;
}

template <typename TY, typename TR, int E>
void launch(const BlockNormArgs& a, cudaStream_t st) {
  // Many rows: at 6007 x 4096 (bf16, gate, both norms) 256 threads take 59 us, 512 70 and a row a block without the copies
  // ahead 71; at 3000 x 8192 (floor 52.5) 1024 threads 71, 512 76.
  if constexpr (E == 4) {
    if (a.K <= 512 ? launch_rows<TY, TR, 32, 4>(a, st) : a.K <= 1024 ? launch_rows<TY, TR, 64, 4>(a, st) :
        a.K <= 2048 ? launch_rows<TY, TR, 128, 4>(a, st) : a.K > 4096 ? a.K <= 8192 && launch_rows<TY, TR, 1024, 2>(a, st) :
        sizeof(TY) == 2 ? launch_rows<TY, TR, 256, 4>(a, st) : launch_rows<TY, TR, 512, 2>(a, st))
      return;
  }
#define AIR_BN(NT, ELEMS) block_norm_kernel<TY, TR, NT, ELEMS / E, E><<<a.T, NT, 0, st>>>(a)
  if (a.K <= 1024) AIR_BN(128, 8);
  else if (a.K <= 2048) AIR_BN(256, 8);
  else if (a.K <= 4096) AIR_BN(512, 8);
  else if (a.K <= 8192) AIR_BN(1024, 8);
  else if (a.K <= 16384) AIR_BN(1024, 16);
  else AIR_BN(1024, 32);
#undef AIR_BN
}

}  // namespace

const char* launch_block_norm(const BlockNormArgs& a, int vec, cudaStream_t st) {
  if (a.T <= 0) return nullptr;
  if (a.K < 1 || a.K > kBlockNormMaxK) return "block_norm: 1 to 32768 columns";
#define AIR_BN_E(TY, TR) (vec == 4 ? launch<TY, TR, 4>(a, st) : vec == 2 ? launch<TY, TR, 2>(a, st) : launch<TY, TR, 1>(a, st))
  if (a.y_bf16 && a.r_bf16) AIR_BN_E(__nv_bfloat16, __nv_bfloat16);
  else if (a.y_bf16) AIR_BN_E(__nv_bfloat16, float);
  else if (a.r_bf16) AIR_BN_E(float, __nv_bfloat16);
  else AIR_BN_E(float, float);
#undef AIR_BN_E
  return nullptr;
}

}  // namespace air
