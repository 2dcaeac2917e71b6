// Interface between the launchers of the 4-bit linear layers (linear_act_api.cpp) and their kernels (linear_q4.hip).
#pragma once

#include "linear_act.h"

namespace fwn {

struct Q4Args {
  ProductArgs p;          // a, its stride, k and the epilogue
  const uint8_t* codes;   // [n, 16 groups], 16-byte aligned, the even input in a byte's low half
  const uint8_t* scales;  // [n, groups], rows scale_row bytes apart
  int64_t groups, scale_row;
};
// A product of at most kFewRows rows of bf16 or float32.
hipError_t launch_q4_rows(bool f32, const Q4Args& a, hipStream_t stream);

// A product of bf16 rows by tiles of 64 rows and 64 `waves` (2 or 4) outputs; `chunk` of its arguments counts kQ4Span inputs. Rows of scales are whole aligned
// fours of bytes.
hipError_t launch_q4_tiles(int waves, const Q4Args& a, hipStream_t stream);
constexpr int kQ4Span = 128;

struct WidenArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  char* dst;  // [outs, 32 groups] bf16 or float32
  int64_t outs, ins, groups;
};
hipError_t launch_widen(bool f32, const WidenArgs& a, hipStream_t stream);

struct QuantizeQ4Args {
  const void* x;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows, cols, x_stride;
};
hipError_t launch_quantize_q4(int dtype, const QuantizeQ4Args& a, hipStream_t stream);

}  // namespace fwn
