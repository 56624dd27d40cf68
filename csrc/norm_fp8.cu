// Residual addition + RMSNorm + E4M3 rows, the input of the W8A8 projections, in one pass:
//   r = x + y;  n = r * rsqrt(mean(r^2) + eps) * (w + w_offset);  s = max|n| / 448;  code = E4M3(n / s)
// One CTA per row with the row in registers, so x and y are read once and the norm's output never
// goes to memory: 4 + 2 bytes read and 4 + 1 written per element (bf16 addend). The sum of squares,
// the maximum and the norm stay f32; the codes are the only rounding (the separate norm and
// quantiser round the norm's output to bf16 between them).
#include <cuda_fp8.h>
#include "common.cuh"
#include "norm_fp8.h"

namespace air {

namespace {

// Block-wide maximum of the bit patterns of non-negative floats, which order like the values and
// put NaN on top: a row with a NaN gets a NaN scale.
AIR_DEVICE float block_max_abs(uint32_t v, uint32_t* red) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if (lane == 0) red[wid] = v;
  __syncthreads();
  return __uint_as_float(__reduce_max_sync(0xffffffffu, lane < nw ? red[lane] : 0u));
}

// NT threads, V groups of 8 consecutive elements per thread.
template <int NT, int V>
__global__ void __launch_bounds__(NT) add_rmsnorm_fp8_kernel(const AddNormF8Args a) {
  __shared__ float red[32];
  __shared__ uint32_t redu[32];
  const int t = blockIdx.x;
  const float* x = a.x + (size_t)t * a.ldx;
  float r[V][8];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 8 * (threadIdx.x + NT * j);
    if (i < a.K) {
      const float4 lo = *reinterpret_cast<const float4*>(x + i), hi = *reinterpret_cast<const float4*>(x + i + 4);
      r[j][0] = lo.x; r[j][1] = lo.y; r[j][2] = lo.z; r[j][3] = lo.w;
      r[j][4] = hi.x; r[j][5] = hi.y; r[j][6] = hi.z; r[j][7] = hi.w;
      if (a.y) {
        float f[8];
        if (a.y_bf16) {
          bf16x8_to_f32(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.y) + (size_t)t * a.ldy + i), f);
        } else {
          const float* y = static_cast<const float*>(a.y) + (size_t)t * a.ldy + i;
          const float4 yl = *reinterpret_cast<const float4*>(y), yh = *reinterpret_cast<const float4*>(y + 4);
          f[0] = yl.x; f[1] = yl.y; f[2] = yl.z; f[3] = yl.w;
          f[4] = yh.x; f[5] = yh.y; f[6] = yh.z; f[7] = yh.w;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) r[j][e] += f[e];
      }
      if (a.resid) {
        float* o = a.resid + (size_t)t * a.ldr + i;
        *reinterpret_cast<float4*>(o) = make_float4(r[j][0], r[j][1], r[j][2], r[j][3]);
        *reinterpret_cast<float4*>(o + 4) = make_float4(r[j][4], r[j][5], r[j][6], r[j][7]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[j][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(r[j][e], r[j][e], ss);
  }
  const float scale = rsqrtf(block_sum(ss, red) / (float)a.K + a.eps);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 8 * (threadIdx.x + NT * j);
    if (i < a.K) {
      const float4 lo = *reinterpret_cast<const float4*>(a.w + i), hi = *reinterpret_cast<const float4*>(a.w + i + 4);
      const float w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        r[j][e] = r[j][e] * scale * (w[e] + a.w_offset);
        top = max(top, __float_as_uint(fabsf(r[j][e])));
      }
      if (a.out_bf16)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out_bf16) + (size_t)t * a.ldo + i) = f32_to_bf16x8(r[j]);
    }
  }
  const float amax = block_max_abs(top, redu);
  // 448 / amax overflows below 1.4e-36: such a row takes the smallest normal scale
  const bool tiny = amax > 0.f && amax < 448.f * 1.17549435e-38f;
  const float inv = tiny ? 8.50705917e37f : amax > 0.f ? 448.f / amax : 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 8 * (threadIdx.x + NT * j);
    if (i >= a.K) continue;
    uint32_t c[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const __nv_fp8x2_storage_t lo =
          __nv_cvt_float2_to_fp8x2(make_float2(r[j][4 * p] * inv, r[j][4 * p + 1] * inv), __NV_SATFINITE, __NV_E4M3);
      const __nv_fp8x2_storage_t hi =
          __nv_cvt_float2_to_fp8x2(make_float2(r[j][4 * p + 2] * inv, r[j][4 * p + 3] * inv), __NV_SATFINITE, __NV_E4M3);
      c[p] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    *reinterpret_cast<uint2*>(a.xq + (size_t)t * a.K + i) = make_uint2(c[0], c[1]);
  }
  if (threadIdx.x == 0) a.xs[t] = tiny ? 1.17549435e-38f : amax / 448.f;
}

}  // namespace

const char* launch_add_rmsnorm_fp8(const AddNormF8Args& a, cudaStream_t st) {
  if (a.T <= 0) return nullptr;
  if (a.K % 8 || a.K < 8 || a.K > kAddNormMaxK) return "add_rmsnorm_fp8: K must be a multiple of 8 up to 32768";
#define AIR_ANQ(NT, V) add_rmsnorm_fp8_kernel<NT, V><<<a.T, NT, 0, st>>>(a)
  if (a.K <= 2048) AIR_ANQ(128, 2);
  else if (a.K <= 4096) AIR_ANQ(256, 2);
  else if (a.K <= 8192) AIR_ANQ(512, 2);
  else if (a.K <= 16384) AIR_ANQ(1024, 2);
  else AIR_ANQ(1024, 4);
#undef AIR_ANQ
  return nullptr;
}

}  // namespace air
