// The way from a block's output to the next block's input in one pass:
//   h = y;  h = h rsqrt(mean(h^2) + eps) (post + w_offset);  h = h act(gate);
//   r = resid + scale h;  out = r rsqrt(mean(r^2) + eps) (w + w_offset)
// each step but the sum optional. One CTA per row with the row in registers, so y, gate and the residual are read once,
// r and out written once and nothing else goes to memory. All steps are f32 on the unrounded values of the step before;
// out and (in bf16) the stored residual are rounded once. Memory-bound with many rows, the latency of one or two block
// reductions with one.
#include "state_space.cuh"

namespace air {

namespace {

// One RMS norm of the row held in h: 1 / rms. Elements past K are zero.
AIR_DEVICE float inv_rms(float ss, float* red, const BlockNormArgs& a) { return rsqrtf(block_sum(ss, red) / (float)a.K + a.eps); }

// NT threads, J groups of E consecutive elements per thread, E NT elements apart.
template <typename TY, typename TR, int NT, int J, int E>
__global__ void __launch_bounds__(NT) block_norm_kernel(const BlockNormArgs a) {
  __shared__ float red[32];
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
    const float inv = inv_rms(ss, red, a);
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
  const float inv = a.w ? inv_rms(ss, red, a) : 1.f;
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

template <typename TY, typename TR, int E>
void launch(const BlockNormArgs& a, cudaStream_t st) {
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

const char* launch_block_norm(const BlockNormArgs& a, bool vec, cudaStream_t st) {
  if (a.T <= 0) return nullptr;
  if (a.K < 1 || a.K > kBlockNormMaxK) return "block_norm: 1 to 32768 columns";
#define AIR_BN_E(TY, TR) (vec ? launch<TY, TR, 4>(a, st) : launch<TY, TR, 1>(a, st))
  if (a.y_bf16 && a.r_bf16) AIR_BN_E(__nv_bfloat16, __nv_bfloat16);
  else if (a.y_bf16) AIR_BN_E(__nv_bfloat16, float);
  else if (a.r_bf16) AIR_BN_E(float, __nv_bfloat16);
  else AIR_BN_E(float, float);
#undef AIR_BN_E
  return nullptr;
}

}  // namespace air
