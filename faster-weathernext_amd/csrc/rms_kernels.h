// Interface between the RMS norm launchers (rms_api.cpp) and their kernels (rms.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwn_rows.h"

namespace fwn {

struct RmsArgs {
  const void* x;
  const void* y;       // added to x, or null
  const void* weight;  // [channels] or null
  void* sum;           // x + y, with y
  void* out;           // the norm in the dtype, or null with q
  uint8_t* q;          // its e4m3 codes, or null with out
  float* scale;        // a row's scale, with q
  int64_t rows, x_stride, y_stride;  // strides in elements
  int32_t channels;
  float eps;
  bool norm;        // false: the rows themselves are quantised
  bool weight_f32;  // the weight is float32 whatever the dtype
  bool stream;      // set by launch_rms: non-temporal stores
};

struct RmsBwdArgs {
  const void* s;       // the rows that were normalised
  const void* weight;  // or null
  const void* g_out;
  const void* g_sum;   // or null
  void* gx;
  float* part;  // [blocks, channels], or null: no weight gradient
  void* gw;     // [channels] in the weight's dtype
  int64_t rows;
  int32_t channels, blocks;
  float eps;
  bool weight_f32;
  bool stream;
};

hipError_t launch_rms(int dtype, const RmsArgs& a, hipStream_t stream);

// Workgroups of the backward pass.
int32_t rms_bwd_blocks(int64_t rows, int32_t channels);

// The backward pass and, with a.part, the reduction of its partial sums.
hipError_t launch_rms_bwd(int dtype, const RmsBwdArgs& a, hipStream_t stream);

}  // namespace fwn
