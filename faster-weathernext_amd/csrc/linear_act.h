// Interface between the launchers of the linear layers (linear_act_api.cpp) and their kernels (linear_act.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwn_rows.h"

namespace fwn {

enum : int32_t { kOpF32 = 0, kOpBf16 = 1, kOpE4m3 = 2 };  // element types of a product's operands

// c[i, j] = sum over k of a(i, k) b(j, k), then the epilogue. Strides in elements.
struct ProductArgs {
  const void* a;
  const void* b;
  int64_t a_row, a_k, b_row, b_k;
  int64_t m, n, k;
  int32_t op;     // of a and b
  int32_t dtype;  // of everything below but the scales
  const float* a_scale;  // [m] and [n], or null
  const float* b_scale;
  const void* bias;      // [n] or null
  const void* residual;  // [m, n], rows r_row apart, or null
  int64_t r_row;
  void* out;  // [m, n]
  void* pre;  // [m, n] or null
  int32_t activation;
};

hipError_t launch_product(const ProductArgs& a, hipStream_t stream);

struct SlopeArgs {
  const void* g;    // [rows, outs]
  const void* pre;  // [rows, outs], unread without an activation
  void* dz;         // [rows, outs] or null
  void* gb;         // [outs] or null
  int64_t rows;
  int32_t outs, dtype, activation;
};

// dz = g act'(pre) and its column sums.
hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream);

}  // namespace fwn
