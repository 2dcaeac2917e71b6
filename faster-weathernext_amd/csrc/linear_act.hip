// Matrix products with bias, activation and residual in their epilogue, and their gradients (gfx950):
//
//   z = x w^T + b,  out = act(z) + residual;   dz = g act'(z),  gx = dz w,  gw = dz^T x,  gb = sum of dz
//
// One kernel for the three products: c[i, j] = sum over k of a(i, k) b(j, k) for operands of any strides.
#include "linear_act.h"

#include "fwn_attn.h"

namespace fwn {
namespace {

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }

__device__ __forceinline__ float load_one(const void* p, int64_t i, int type) {
  if (type == kOpF32) return ((const float*)p)[i];
  if (type == kOpBf16) return as_float((uint32_t)((const uint16_t*)p)[i] << 16);
  return __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)p)[i], 0);
}

__device__ __forceinline__ void store_one(void* p, int64_t i, int type, float v) {
  if (type == kOpF32)
    ((float*)p)[i] = v;
  else
    ((uint16_t*)p)[i] = __builtin_bit_cast(uint16_t, (__bf16)v);
}

__device__ __forceinline__ float activate(float z, int kind) {
  constexpr float c = 0.7978845608028654f;
  switch (kind) {
    case FWN_ACT_RELU: return z > 0.f || z != z ? z : 0.f;
    case FWN_ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.7071067811865476f));
    case FWN_ACT_GELU_TANH: return 0.5f * z * (1.f + tanhf(c * (z + 0.044715f * z * z * z)));
    case FWN_ACT_SILU: return z / (1.f + expf(-z));
    default: return z;
  }
}

__device__ __forceinline__ float slope(float z, int kind) {
  constexpr float c = 0.7978845608028654f;
  switch (kind) {
    case FWN_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case FWN_ACT_GELU:
      return 0.5f * (1.f + erff(z * 0.7071067811865476f)) + z * expf(-0.5f * z * z) * 0.3989422804014327f;
    case FWN_ACT_GELU_TANH: {
      const float t = tanhf(c * (z + 0.044715f * z * z * z));
      return 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * c * (1.f + 3.f * 0.044715f * z * z);
    }
    case FWN_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    default: return 1.f;
  }
}

constexpr int TILE = 64, STEP = 16;

// 64 x 64 outputs by 256 threads, 4 x 4 a thread, 16 k at a time through LDS.
__global__ void __launch_bounds__(256) product_kernel(ProductArgs a) {
  __shared__ float sa[STEP][TILE + 1], sb[STEP][TILE + 1];
  const int64_t tiles = (a.n + TILE - 1) / TILE;
  const int64_t i0 = (int64_t)blockIdx.x / tiles * TILE, j0 = (int64_t)blockIdx.x % tiles * TILE;
  const int ti = (int)threadIdx.x / 16, tj = (int)threadIdx.x % 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < a.k; k0 += STEP) {
    for (int e = threadIdx.x; e < TILE * STEP; e += 256) {
      const int r = e / STEP, k = e % STEP;
      const bool in = k0 + k < a.k;
      sa[k][r] = in && i0 + r < a.m ? load_one(a.a, (i0 + r) * a.a_row + (k0 + k) * a.a_k, a.op) : 0.f;
      sb[k][r] = in && j0 + r < a.n ? load_one(a.b, (j0 + r) * a.b_row + (k0 + k) * a.b_k, a.op) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < STEP; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ti + 16 * i], sb[k][tj + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t row = i0 + ti + 16 * i, col = j0 + tj + 16 * j;
      if (row >= a.m || col >= a.n) continue;
      float z = acc[i][j];
      if (a.a_scale) z *= a.a_scale[row] * a.b_scale[col];
      if (a.bias) z += load_one(a.bias, col, a.dtype);
      if (a.pre) store_one(a.pre, row * a.n + col, a.dtype, z);
      z = activate(z, a.activation);
      if (a.residual) z += load_one(a.residual, row * a.r_row + col, a.dtype);
      store_one(a.out, row * a.n + col, a.dtype, z);
    }
}

__global__ void __launch_bounds__(64) slope_kernel(SlopeArgs a) {
  const int c = (int)blockIdx.x * 64 + (int)threadIdx.x;
  if (c >= a.outs) return;
  float sum = 0.f;
  for (int64_t r = 0; r < a.rows; ++r) {
    const int64_t at = r * a.outs + c;
    float dz = load_one(a.g, at, a.dtype);
    if (a.activation) dz *= slope(load_one(a.pre, at, a.dtype), a.activation);
    sum += dz;
    if (a.dz) store_one(a.dz, at, a.dtype, dz);
  }
  if (a.gb) store_one(a.gb, c, a.dtype, sum);
}

}  // namespace

hipError_t launch_product(const ProductArgs& a, hipStream_t stream) {
  const int64_t blocks = ((a.m + TILE - 1) / TILE) * ((a.n + TILE - 1) / TILE);
  hipLaunchKernelGGL(product_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(slope_kernel, dim3((unsigned)(a.outs + 63) / 64), dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace fwn
