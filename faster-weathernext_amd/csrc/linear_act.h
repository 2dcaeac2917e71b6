// Interface between the launchers of the linear layers (linear_act_api.cpp) and their kernels (linear_act.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwn_rows.h"

namespace fwn {

enum : int32_t { kOpF32 = 0, kOpBf16 = 1, kOpE4m3 = 2 };  // element types of a product's operands

// What happens to a product z[i, j]: z a_scale[i] b_scale[j] + bias[j], kept in pre, activated, the residual
// added, stored in out. dtype is that of everything but the scales.
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

// c[i, j] = sum over k of a(i, k) b(j, k). Each operand is either rows of contiguous k (`inner`) or k rows of
// contiguous i or j; 16-byte aligned, strides and, in elements, the contiguous extent multiples of 16
// bytes. float32 operands lie as planes of three bf16 parts, side by side in each row, and the product is the
// sum of the six largest products of the parts.
struct ProductArgs {
  const char* a;
  const char* b;
  int64_t a_stride, b_stride;  // bytes between rows, at most kMaxStride
  int64_t a_plane, b_plane;    // bytes between planes of float32 operands
  int64_t k;                   // elements of the sum
  int32_t splits;              // ranges of the sum, each `chunk` stages (the last may be shorter)
  int32_t chunk;
  float* part;                 // [splits, m, part_row] where splits > 1
  int64_t part_row;            // n padded to 8
  float* sums;                 // column sums of a (a's rows are k): [splits, m], or null
  // float32 operands as they were given, for outputs that came out NaN: strides in elements, or null.
  const float* a_whole;
  const float* b_whole;
  int64_t aw_row, aw_k, bw_row, bw_k, whole_k;
  EpilogueArgs e;
};

constexpr int64_t kMaxStride = 1 << 22;
constexpr int kStageBytes = 128;  // of an operand row in one pipeline stage
constexpr int kStageRows = 64;   // of an operand whose rows are k

enum class Operands { kInnerInner, kInnerOuter, kOuterOuter };  // how a and b lie

// Output tiles of the product kernel.
struct TileShape {
  int m, n;
};
constexpr TileShape kTiles[] = {{256, 256}, {192, 128}, {128, 128}};
constexpr int kTileShapes = 3;

// One product, by tiles of kTiles[tile]. `op` is what the operands hold: bf16, float32 as planes, or e4m3
// (kInnerInner alone).
hipError_t launch_product(Operands how, int32_t op, int tile, const ProductArgs& a, hipStream_t stream);

// A matrix laid out for the product kernel: rows padded with zeros to 16 bytes, float32 as three planes of
// bf16 parts whose sum is the value.
struct LayoutArgs {
  const void* src;  // [rows, cols], rows `stride` elements apart
  int64_t rows, cols, stride;
  int32_t op;
  char* dst;
  int64_t dst_stride, dst_plane;  // bytes
};
hipError_t launch_layout(const LayoutArgs& a, hipStream_t stream);

// dz = g act'(pre) laid out for the product kernel, and its column sums.
struct SlopeArgs {
  const void* g;    // [rows, outs]
  const void* pre;  // [rows, outs], unread without an activation
  char* dz;         // or null
  int64_t dz_stride, dz_plane;  // bytes
  float* part;      // [blocks, outs] partial sums, or null: no sums
  int64_t rows, chunk;  // rows of a workgroup
  int32_t outs, dtype, activation, blocks;
};
hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream);

// out[c] = the sum of the `count` rows of part [count, n], in the dtype.
hipError_t launch_column_sums(const float* part, int64_t count, int64_t n, void* out, int dtype, hipStream_t stream);

}  // namespace fwn
