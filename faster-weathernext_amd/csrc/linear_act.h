// Interface between the launchers of the linear layers (linear_act_api.cpp) and their kernels (linear_act.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwn_rows.h"

namespace fwn {

enum : int32_t { kOpF32 = 0, kOpBf16 = 1, kOpE4m3 = 2 };  // element types of a product's operands

// What happens to a product z[i, j]: z a_scale[i] b_scale[j] + bias[j] (in that order: the scales' own product may lie
// out of float32's range), kept in pre, activated, the residual added, stored in out. dtype is that of everything but the
// scales.
struct EpilogueArgs {
  const float* a_scale;  // [m] and [n], or both null
  const float* b_scale;
  const void* bias;      // [n] or null
  const void* residual;  // [m, n], rows r_row elements apart, or null
  void* out;             // [m, n]
  void* pre;             // [m, n] or null
  int64_t r_row;
  int64_t m, n;
  int32_t dtype, activation;
  bool vec;  // n and r_row are multiples of 8 (r_row at most FWN_LINEAR_ACT_MAX), every tensor is 16-byte aligned
};

// c[i, j] = sum over k of a(i, k) b(j, k). Each operand is either rows of contiguous k (inner) or k rows of
// contiguous i or j (outer). bf16 and e4m3 operands are 16-byte aligned, their strides and contiguous extents whole
// 16 bytes (what pads an extent is zeros).
struct ProductArgs {
  const char* a;
  const char* b;
  int64_t a_stride, b_stride;  // bytes between rows, at most kMaxStride
  int64_t k;
  int32_t splits;              // ranges of the sum, each `chunk` stages (the last may be shorter)
  int32_t chunk;
  float* part;                 // [splits, m, part_row] where splits > 1
  int64_t part_row;            // n padded to 8
  float* sums;                 // column sums of an outer a: [splits, m], or null
  void* sums_out;              // the sums in the dtype where splits is 1, or null
  EpilogueArgs e;
};

constexpr int64_t kMaxStride = 1 << 22;
constexpr int kStageBytes = 128;  // of an operand row in one pipeline stage
constexpr int kStageRows = 64;    // of an operand whose rows are k
constexpr int kStageF32 = 32;     // k of a stage of float32 operands

enum class Operands { kInnerInner, kInnerOuter, kOuterOuter };  // how a and b lie

// One product, by tiles of 256 x 256 or 128 x 128 (float32: 128 x 128, or 64 x 128 of an inner a). Of e4m3 operands
// kInnerInner alone.
hipError_t launch_product(Operands how, int32_t op, int tile, const ProductArgs& a, hipStream_t stream);
hipError_t launch_product_f32(Operands how, int tile, const ProductArgs& a, hipStream_t stream);
// One product of inner operands with at most kFewRows rows of a, unsplit.
hipError_t launch_product_rows(int32_t op, const ProductArgs& a, hipStream_t stream);
constexpr int64_t kFewRows = 32;

// A matrix copied to rows padded with zeros to 16 bytes.
struct LayoutArgs {
  const void* src;  // [rows, cols], rows `stride` elements apart
  int64_t rows, cols, stride;
  int32_t op;
  char* dst;
  int64_t dst_stride;  // bytes
};
hipError_t launch_layout(const LayoutArgs& a, hipStream_t stream);

// dz = g act'(pre) in rows padded to 16 bytes, and its column sums.
struct SlopeArgs {
  const void* g;    // [rows, outs]
  const void* pre;  // [rows, outs], unread without an activation
  char* dz;         // or null
  int64_t dz_stride;  // bytes, room for whole eights of columns
  float* part;      // [blocks, outs] partial sums, or null
  void* gb;         // the sums in the dtype where blocks is 1, or null
  int64_t rows, chunk;  // rows of a workgroup
  int32_t outs, dtype, activation, blocks;
};
hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream);

// out[c] = the sum of the `count` rows of part [count, n], in the dtype.
hipError_t launch_column_sums(const float* part, int64_t count, int64_t n, void* out, int dtype, hipStream_t stream);

}  // namespace fwn
