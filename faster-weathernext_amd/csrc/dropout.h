// Interface between the launchers of dropout and of the norms around a block (branch_api.cpp) and their kernels (dropout.hip,
// sandwich.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fwn_rows.h"

namespace fwn {

struct DropoutArgs {
  const uint64_t* state;  // {seed, offset} in the GPU's memory, or null: the two members below
  uint64_t seed, offset;
  uint32_t border;  // sixteen random bits below it: dropped
  float keep;       // what is kept is multiplied by it
};

struct DropoutRowsArgs {
  const void* x;
  const void* residual;  // or null
  void* out;             // contiguous
  int64_t rows, x_stride, r_stride;  // strides in elements
  int32_t channels;
  DropoutArgs drop;
};

hipError_t launch_dropout(int dtype, const DropoutRowsArgs& a, hipStream_t stream);

struct SandwichArgs {
  const void* x;
  const void* y;
  const void* gate;         // [rows / gate_rows, channels], or null: 1
  const void* post_weight;  // [channels] or null: 1
  const void* pre_weight;
  void* sum;
  void* out;
  int64_t rows, gate_rows, x_stride, y_stride;  // strides in elements
  int32_t channels;
  float eps, scale;
  bool post_norm;
  bool gate_f32, post_f32, pre_f32;  // float32 whatever the dtype
  bool drop;
  bool stream;  // set by the launch: non-temporal stores
  DropoutArgs draw;
};
hipError_t launch_sandwich(int dtype, const SandwichArgs& a, hipStream_t stream);

struct SandwichBwdArgs {
  const void* s;  // contiguous, as are the gradients
  const void* y;
  const void* gate;
  const void* post_weight;
  const void* pre_weight;
  const void* g_sum;  // or null: zeros
  const void* g_out;  // or null: zeros
  void* gx;           // or null: not wanted, as all below
  void* gy;
  void* g_gate;
  void* g_post;
  void* g_pre;
  float* part;  // [parts, blocks, channels] of the launch's SandwichGrid, or null
  int64_t rows, gate_rows, y_stride;
  int32_t channels;
  float eps, scale;
  bool post_norm;
  bool gate_f32, post_f32, pre_f32;
  bool drop;
  bool stream;  // set by the launch: non-temporal stores
  DropoutArgs draw;
};
// The workgroups of the backward pass: groups of rows that share a gate's row (one group without a gate, and with one of x's
// shape: gate_rows 1) go to `per` workgroups each, or several to one.
struct SandwichGrid {
  int64_t groups, group_rows;
  int32_t blocks, per, of_block;  // workgroups a group, groups a workgroup; one of the two is 1
  int32_t parts;                  // partial sums a workgroup leaves: of pre_weight's, post_weight's and the gate's gradients
};
SandwichGrid sandwich_grid(int64_t rows, int64_t gate_rows, int32_t channels, int32_t dtype);
hipError_t launch_sandwich_bwd(int dtype, const SandwichBwdArgs& a, hipStream_t stream);

}  // namespace fwn
