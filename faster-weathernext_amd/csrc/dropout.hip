// Dropout of rows with the residual's addition (gfx950): out = rnd(kept x 2^16 / (2^16 - T) + residual), its backward pass the same
// over the gradient. Nothing about what is kept is stored: see dropout_device.h.
//
// Bound by HBM, a streaming pass of one 16-byte vector of each tensor a thread and step, two steps at a time: 40,962 x 768 bf16 with a
// residual 34 us (5.6 TB/s), without 26; 10,242 x 1,283 float32 21 (5.0). The generator takes about half of that time beside it.
#include "dropout_device.h"

#include "fwn_attn.h"

namespace fwn {
namespace {

constexpr int kSteps = 2;  // vectors of a thread on their way at once

// Vectors of E channels, `across` a row; a thread takes every `stride`-th, (row, vector) `step_row` and `step_at` further on.
template <typename T, bool NT, bool TAIL>
__global__ void __launch_bounds__(256) dropout_kernel(DropoutRowsArgs a, uint32_t across, uint32_t step_row, uint32_t step_at) {
  constexpr int E = 16 / sizeof(T);
  const Draw draw(a.drop);
  const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row;
  uint32_t at;
  if (id >> 32 == 0) {  // 32-bit division
    row = (uint32_t)id / across;
    at = (uint32_t)id - (uint32_t)row * across;
  } else {
    row = (int64_t)(id / across);
    at = (uint32_t)(id - (uint64_t)row * across);
  }
  while (row < a.rows) {
    float f[kSteps][E], r[kSteps][E];
    int64_t rows[kSteps];
    uint32_t cols[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      rows[k] = row;
      cols[k] = at * E;
      const int left = a.channels - (int)cols[k];
      if (row < a.rows) {
        load<T, E, true, TAIL>((const T*)a.x + row * a.x_stride + cols[k], left, f[k]);
        if (a.residual) load<T, E, true, TAIL>((const T*)a.residual + row * a.r_stride + cols[k], left, r[k]);
      }
      row += step_row;
      at += step_at;
      if (at >= across) {
        at -= across;
        ++row;
      }
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      if (rows[k] >= a.rows) break;
      draw.apply<E>((uint32_t)rows[k], cols[k], f[k]);
      if (a.residual) {
#pragma unroll
        for (int e = 0; e < E; ++e) f[k][e] += r[k][e];
      }
      store<T, E, NT, TAIL>((T*)a.out + rows[k] * a.channels + cols[k], a.channels - (int)cols[k], f[k]);
    }
  }
}

template <typename T, bool NT>
hipError_t launch_as(const DropoutRowsArgs& a, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const uint32_t across = (uint32_t)((a.channels + E - 1) / E);
  const uint64_t vectors = (uint64_t)a.rows * across, want = (vectors + 256 * kSteps - 1) / (256 * kSteps);
  const uint64_t blocks = want < (uint64_t)kMostBlocks ? want : (uint64_t)kMostBlocks, stride = blocks * 256;
  const uint32_t step_row = (uint32_t)(stride / across), step_at = (uint32_t)(stride % across);
  if (a.channels % E)
    hipLaunchKernelGGL((dropout_kernel<T, NT, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a, across, step_row, step_at);
  else
    hipLaunchKernelGGL((dropout_kernel<T, NT, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a, across, step_row, step_at);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(int dtype, const DropoutRowsArgs& a, hipStream_t stream) {
  const bool stream_out = (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  if (dtype == FWN_F32) return stream_out ? launch_as<float, true>(a, stream) : launch_as<float, false>(a, stream);
  return stream_out ? launch_as<uint16_t, true>(a, stream) : launch_as<uint16_t, false>(a, stream);
}

}  // namespace fwn
