// Passes around the products of the linear layers (gfx950): operands laid out for them, dz = g act'(z) with its
// column sums, and the sums of partial rows.
#include "linear_act_device.h"

namespace fwn {
namespace {

constexpr int64_t kMostBlocks = 1 << 20;  // of the layout's launch; more are looped over

// Rows padded with zeros to 16 bytes, 16 bytes a thread.
template <typename T>
__global__ void __launch_bounds__(256) layout_kernel(LayoutArgs a) {
  constexpr int PER = 16 / sizeof(T);  // columns a thread
  const int64_t across = (a.cols + PER - 1) / PER, total = a.rows * across;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / across, at = id - row * across, col = at * PER;
    const T* p = (const T*)a.src + row * a.stride + col;
    uint32_t d[4] = {};
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (col + k < a.cols) d[k * (int)sizeof(T) / 4] |= (uint32_t)p[k] << 8 * (k * (int)sizeof(T) % 4);
    *(u32x4*)(a.dst + row * a.dst_stride + at * 16) = u32x4{d[0], d[1], d[2], d[3]};
  }
}

// dz = g act'(pre). bf16: dz is the products' operand and so rounded to it, which costs the gradients as much again as their
// own rounding (1,024 x 256 -> 1,024 with gelu_tanh: gx 2.34e-3 off, 1.65e-3 with dz left in float32); pre, kept in bf16 to
// be half the bytes, adds little (2.39e-3). The sums are of dz before it is rounded.
// 256 columns by `chunk` rows a workgroup, eight columns of every eighth row a thread: side by side where rows are whole
// aligned eights (VEC), else 32 apart, so that a wave's accesses lie side by side. F32: the dtype is float32.
template <int KIND, bool VEC, bool F32>
__global__ void __launch_bounds__(256) slope_kernel(SlopeArgs a) {
  __shared__ float red[8][256];
  const int across = (a.outs + 255) / 256, block = (int)blockIdx.x / across;
  const int lane = (int)threadIdx.x & 31, own = (int)threadIdx.x >> 5, c0 = ((int)blockIdx.x - block * across) * 256;
  const auto column = [&](int k) { return c0 + (VEC ? 8 * lane + k : lane + 32 * k); };
  const int64_t r0 = (int64_t)block * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  const int padded = (a.outs + 7) / 8 * 8;
  float sum[8] = {};
  if (!VEC || column(0) < a.outs) {
#pragma unroll 2
    for (int64_t r = r0 + own; r < r1; r += 8) {
      const int64_t at = r * a.outs;
      float dz[8], z[8];
      if constexpr (VEC) {
        load8(a.g, at + column(0), a.dtype, dz);
        if (KIND != FWN_ACT_NONE) load8(a.pre, at + column(0), a.dtype, z);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool in = column(k) < a.outs;
          dz[k] = in ? load_one(a.g, at + column(k), a.dtype) : 0.f;
          z[k] = in && KIND != FWN_ACT_NONE ? load_one(a.pre, at + column(k), a.dtype) : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (KIND != FWN_ACT_NONE) dz[k] *= slope<KIND, F32>(z[k]);
        sum[k] += dz[k];
      }
      if (a.dz) {
        char* const row = a.dz + r * a.dz_stride;
        if constexpr (VEC) {
          store8(row, column(0), a.dtype, dz);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (column(k) < padded) store_one(row, column(k), a.dtype, dz[k]);
        }
      }
    }
  }
  if (!a.part && !a.gb) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[own][column(k) - c0] = sum[k];
  __syncthreads();
  const int c = (int)threadIdx.x;
  if (c0 + c >= a.outs) return;
  float s = red[0][c];
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][c];
  if (a.gb)
    store_one(a.gb, c0 + c, a.dtype, s);
  else
    a.part[(int64_t)block * a.outs + c0 + c] = s;
}

constexpr int kSumCols = 16, kGroups = 64;  // columns of a workgroup, and shares of the rows that it adds in parallel

// Few columns a workgroup, so that a hundred rows of a thousand columns still fill a good part of the chip (1,024
// rows: of 768 columns 4.8 us with 64 columns a workgroup, of 8,192 24).
__global__ void __launch_bounds__(kSumCols * kGroups) column_sums_kernel(const float* part, int64_t count, int64_t n,
                                                                         void* out, int dtype) {
  __shared__ float red[kGroups][kSumCols];
  const int lane = (int)threadIdx.x % kSumCols, grp = (int)threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lane;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int64_t b = grp; b < count; b += kGroups) s += part[b * n + c];
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp < 8) {
#pragma unroll
    for (int k = 8; k < kGroups; k += 8) s += red[grp + k][lane];
  }
  __syncthreads();
  if (grp < 8) red[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || c >= n) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][lane];
  store_one(out, c, dtype, s);
}

}  // namespace

hipError_t launch_layout(const LayoutArgs& a, hipStream_t stream) {
  const int64_t per = a.op == kOpE4m3 ? 16 : a.op == kOpBf16 ? 8 : 4, threads = a.rows * ((a.cols + per - 1) / per);
  if (threads == 0) return hipSuccess;
  const int64_t blocks = (threads + 255) / 256;
  const dim3 grid((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)), block(256);
  if (a.op == kOpE4m3)
    hipLaunchKernelGGL(layout_kernel<uint8_t>, grid, block, 0, stream, a);
  else if (a.op == kOpBf16)
    hipLaunchKernelGGL(layout_kernel<uint16_t>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(layout_kernel<uint32_t>, grid, block, 0, stream, a);
  return hipGetLastError();
}

template <bool VEC, bool F32>
static hipError_t launch_slope_as(const SlopeArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)((a.outs + 255) / 256) * (unsigned)a.blocks), block(256);
  switch (a.activation) {
    case FWN_ACT_RELU: hipLaunchKernelGGL((slope_kernel<FWN_ACT_RELU, VEC, F32>), grid, block, 0, stream, a); break;
    case FWN_ACT_GELU: hipLaunchKernelGGL((slope_kernel<FWN_ACT_GELU, VEC, F32>), grid, block, 0, stream, a); break;
    case FWN_ACT_GELU_TANH: hipLaunchKernelGGL((slope_kernel<FWN_ACT_GELU_TANH, VEC, F32>), grid, block, 0, stream, a); break;
    case FWN_ACT_SILU: hipLaunchKernelGGL((slope_kernel<FWN_ACT_SILU, VEC, F32>), grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL((slope_kernel<FWN_ACT_NONE, VEC, F32>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream) {
  const bool vec = a.outs % 8 == 0 && (((uintptr_t)a.g | (uintptr_t)a.pre) & 15) == 0;
  if (a.dtype == FWN_F32) return vec ? launch_slope_as<true, true>(a, stream) : launch_slope_as<false, true>(a, stream);
  return vec ? launch_slope_as<true, false>(a, stream) : launch_slope_as<false, false>(a, stream);
}

hipError_t launch_column_sums(const float* part, int64_t count, int64_t n, void* out, int dtype, hipStream_t stream) {
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((n + kSumCols - 1) / kSumCols)),
                     dim3(kSumCols * kGroups), 0, stream, part, count, n,
                     out, dtype);
  return hipGetLastError();
}

}  // namespace fwn
