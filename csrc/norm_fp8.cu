// Residual addition + RMSNorm + E4M3 rows, the input of the W8A8 projections, in one pass:
//   r = x + y;  n = r * rsqrt(mean(r^2) + eps) * (w + w_offset);  s = max|n| / 448;  code = E4M3(n / s)
// One CTA per row with the row in registers, so x and y are read once and the norm's output never
// goes to memory: 4 + 2 bytes read and 4 + 1 written per element (bf16 addend). The sum of squares,
// the maximum and the norm stay f32; the codes are the only rounding (the separate norm and
// quantiser round the norm's output to bf16 between them). Memory-bound with many rows: 6007 x 4096 takes
// 42.6 us of a 41.9 us floor (6.4 TB/s); one row 2.5 us, latency of two block reductions.
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

// NT threads, V groups of 4 consecutive elements per thread, 4 NT elements apart (whole lines a load).
template <int NT, int V>
__global__ void __launch_bounds__(NT) add_rmsnorm_fp8_kernel(const AddNormF8Args a) {
  __shared__ float red[32];
  __shared__ uint32_t redu[32];
  const int t = blockIdx.x;
  const float* x = a.x + (size_t)t * a.ldx;
  float r[V][4];
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (threadIdx.x + NT * j);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < a.K) f = *reinterpret_cast<const float4*>(x + i);
    r[j][0] = f.x; r[j][1] = f.y; r[j][2] = f.z; r[j][3] = f.w;
  }
  if (a.y) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int i = 4 * (threadIdx.x + NT * j);
      if (i >= a.K) continue;
      if (a.y_bf16) {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(a.y) + (size_t)t * a.ldy + i);
        const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
        const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
        r[j][0] += lo.x; r[j][1] += lo.y; r[j][2] += hi.x; r[j][3] += hi.y;
      } else {
        const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(a.y) + (size_t)t * a.ldy + i);
        r[j][0] += f.x; r[j][1] += f.y; r[j][2] += f.z; r[j][3] += f.w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (threadIdx.x + NT * j);
    if (a.resid && i < a.K)
      *reinterpret_cast<float4*>(a.resid + (size_t)t * a.ldr + i) = make_float4(r[j][0], r[j][1], r[j][2], r[j][3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fmaf(r[j][e], r[j][e], ss);
  }
  const float scale = rsqrtf(block_sum(ss, red) / (float)a.K + a.eps);
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (threadIdx.x + NT * j);
    if (i >= a.K) continue;
    const float4 f = *reinterpret_cast<const float4*>(a.w + i);
    const float w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      r[j][e] = r[j][e] * scale * (w[e] + a.w_offset);
      top = max(top, __float_as_uint(fabsf(r[j][e])));
    }
    if (a.out_bf16) {
      const __nv_bfloat162 lo = __floats2bfloat162_rn(r[j][0], r[j][1]), hi = __floats2bfloat162_rn(r[j][2], r[j][3]);
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out_bf16) + (size_t)t * a.ldo + i) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
  }
  const float amax = block_max_abs(top, redu);
  // 448 / amax overflows below 1.4e-36: such a row takes the smallest normal scale
  const bool tiny = amax > 0.f && amax < 448.f * 1.17549435e-38f;
  const float inv = tiny ? 8.50705917e37f : amax > 0.f ? 448.f / amax : 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = 4 * (threadIdx.x + NT * j);
    if (i >= a.K) continue;
    const __nv_fp8x2_storage_t lo = __nv_cvt_float2_to_fp8x2(make_float2(r[j][0] * inv, r[j][1] * inv), __NV_SATFINITE, __NV_E4M3);
    const __nv_fp8x2_storage_t hi = __nv_cvt_float2_to_fp8x2(make_float2(r[j][2] * inv, r[j][3] * inv), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint32_t*>(a.xq + (size_t)t * a.K + i) = (uint32_t)lo | ((uint32_t)hi << 16);
  }
  if (threadIdx.x == 0) a.xs[t] = tiny ? 1.17549435e-38f : amax / 448.f;
}

}  // namespace

const char* launch_add_rmsnorm_fp8(const AddNormF8Args& a, cudaStream_t st) {
  if (a.T <= 0) return nullptr;
  if (a.K % 8 || a.K < 8 || a.K > kAddNormMaxK) return "add_rmsnorm_fp8: K must be a multiple of 8 up to 32768";
  // Eight elements a thread up to 8192 (at 6007 x 4096: 42.6 us with 512 threads x 8, 50 with 256 x 16, 61 with
  // 128 x 32); beyond it the row needs more of the block's 1024 threads. Rows of at most 512 leave half or more of
  // 128 threads idle: once the rows are more than one wave of such blocks (16 an SM), blocks of 32 or 64 threads
  // take 13.6 against 19.6 us at 20000 x 256, 18.7 against 22.7 at 20000 x 512 and 3.8 against 4.2 at 3200 x 256;
  // with fewer rows the larger block is done sooner (400 x 256: 2.2 against 2.4 us).
  const bool waves = a.T > 148 * 16;
#define AIR_ANQ(NT, V) add_rmsnorm_fp8_kernel<NT, V><<<a.T, NT, 0, st>>>(a)
  if (waves && a.K <= 256) AIR_ANQ(32, 2);
  else if (waves && a.K <= 512) AIR_ANQ(64, 2);
  else if (a.K <= 1024) AIR_ANQ(128, 2);
  else if (a.K <= 2048) AIR_ANQ(256, 2);
  else if (a.K <= 4096) AIR_ANQ(512, 2);
  else if (a.K <= 8192) AIR_ANQ(1024, 2);
  else if (a.K <= 16384) AIR_ANQ(1024, 4);
  else AIR_ANQ(1024, 8);
#undef AIR_ANQ
  return nullptr;
}

}  // namespace air
