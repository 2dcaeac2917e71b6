// The linear layers' forward for few rows (gfx950): out = act(x w^T + b) + residual with up to 32 rows of x, a decoding
// step's tokens.
//
// Bound by the weight's trip from memory, so the launch is one pass over it with no partial products to join: a
// workgroup has 16 or 32 outputs, its waves share the sum, 128 bytes of each of the weight's rows at a time. A
// wave loads its operands straight into registers in the MFMA's layout (16 rows of 64 bytes an instruction; the
// order of k in a line does not matter as long as both operands have the same) and keeps several lines on
// their way; the waves' sums meet in LDS. float32 operands use float32 MFMAs, e4m3 ones are widened to bf16, which adds
// in float32 (linear_act.hip): the matrix units' rate is not what bounds this.
#include "linear_act_device.h"

namespace fwn {
namespace {

constexpr int LINE = 128;  // bytes of a row in one step of a wave

// Two 16-byte pieces of this lane's row in each line.
template <int OP>
struct Rows {
  rsrc_t r;
  uint32_t off;
  uint32_t bytes;  // of a row in the sum

  __device__ __forceinline__ void init(const char* p, int64_t stride, int64_t first, int64_t rows, int64_t k, int lane) {
    const int i = lane & 15, g = lane >> 4;
    r = make_rsrc(p + first * stride, kBuffer);
    off = first + i < rows ? (uint32_t)i * (uint32_t)stride + g * 16 : kNowhere;
    bytes = (uint32_t)k * (OP == kOpF32 ? 4 : OP == kOpBf16 ? 2 : 1);
  }
  // Piece p of line `line`; zeros past the row. A float32 row may end inside a piece, and is not read past its end.
  __device__ __forceinline__ u32x4 load(uint32_t line, int p, int g) const {
    const uint32_t at = line * LINE + p * 64, from = at + g * 16;
    if (OP != kOpF32 || bytes % 16 == 0 || at + 64 <= bytes) return bload16(r, (off + at) | (from < bytes ? 0 : kNowhere));
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)((off + at + 4 * e) | (from + 4 * e < bytes ? 0 : kNowhere)), 0, 0);
    return v;
  }
};

// c += a b over the k of one line: both pieces of both operands.
template <int OP>
__device__ __forceinline__ f32x4 multiply(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4 c) {
  const auto bf16 = [&](const u32x4& x, const u32x4& y) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  };
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    if constexpr (OP == kOpE4m3) {
#pragma unroll
      for (int h = 0; h < 4; h += 2) bf16(widen(a[p][h], a[p][h + 1]), widen(b[p][h], b[p][h + 1]));
    } else if constexpr (OP == kOpBf16) {
      bf16(a[p], b[p]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = a[p][e], y = b[p][e];
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(as_float(x), as_float(y), c, 0, 0, 0);
      }
    }
  }
  return c;
}

// GROUPS 16-row groups of x by COLS 16-row groups of the weight; AHEAD lines of a wave on their way.
template <int OP, int GROUPS, int COLS, int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) rows_kernel(ProductArgs a) {
  __shared__ float red[WAVES][GROUPS][16][16 * COLS + 1];
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * COLS);
  const EpilogueArgs& e = a.e;
  Rows<OP> weight[COLS], x[GROUPS];
#pragma unroll
  for (int n = 0; n < COLS; ++n) weight[n].init(a.b, a.b_stride, n0 + 16 * n, e.n, a.k, lane);
#pragma unroll
  for (int m = 0; m < GROUPS; ++m) x[m].init(a.a, a.a_stride, 16 * m, e.m, a.k, lane);
  const uint32_t lines = (weight[0].bytes + LINE - 1) / LINE;
  f32x4 acc[GROUPS][COLS];
#pragma unroll
  for (int m = 0; m < GROUPS; ++m)
#pragma unroll
    for (int n = 0; n < COLS; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Lines w, w + WAVES, ... of the rows, AHEAD of them at once (past the rows' end: zeros).
  for (uint32_t l0 = w; l0 < lines; l0 += WAVES * AHEAD) {
    u32x4 vw[AHEAD][COLS][2], vx[AHEAD][GROUPS][2];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int n = 0; n < COLS; ++n) vw[s][n][p] = weight[n].load(l0 + WAVES * s, p, g);
#pragma unroll
        for (int m = 0; m < GROUPS; ++m) vx[s][m][p] = x[m].load(l0 + WAVES * s, p, g);
      }
    __builtin_amdgcn_sched_barrier(0);  // all loads before the first product
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
#pragma unroll
      for (int m = 0; m < GROUPS; ++m)
#pragma unroll
        for (int n = 0; n < COLS; ++n) acc[m][n] = multiply<OP>(vw[s][n], vx[s][m], acc[m][n]);
  }
  // Lane (i, g) holds outputs 4 g .. 4 g + 3 of each group of columns in row i of each group of rows.
#pragma unroll
  for (int m = 0; m < GROUPS; ++m)
#pragma unroll
    for (int n = 0; n < COLS; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[w][m][lane & 15][16 * n + 4 * g + r] = acc[m][n][r];
  __syncthreads();
  with_activation<false>(e.activation, [&](auto act) {
    for (int t = threadIdx.x; t < GROUPS * COLS * 256; t += 64 * WAVES) {
      const int m = t / (COLS * 256), i = t / (COLS * 16) % 16, j = t % (COLS * 16);
      const int64_t row = 16 * m + i, col = n0 + j;
      if (row >= e.m || col >= e.n) continue;
      float z = red[0][m][i][j];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) z += red[v][m][i][j];
      if (OP == kOpE4m3) z = z * e.a_scale[row] * e.b_scale[col];
      if (e.bias) z += load_one(e.bias, col, e.dtype);
      if (e.pre) store_one(e.pre, row * e.n + col, e.dtype, z);
      z = activate<decltype(act)::kind, OP != kOpBf16>(z);
      if (e.residual) z += load_one(e.residual, row * e.r_row + col, e.dtype);
      store_one(e.out, row * e.n + col, e.dtype, z);
    }
  });
}

template <int OP, int GROUPS, int COLS, int WAVES, int AHEAD>
hipError_t launch(const ProductArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((rows_kernel<OP, GROUPS, COLS, WAVES, AHEAD>), dim3((unsigned)((a.e.n + 16 * COLS - 1) / (16 * COLS))),
                     dim3(64 * WAVES), 0, stream, a);
  return hipGetLastError();
}

// 32 outputs a workgroup where 16 would be more workgroups than CUs: the rows of x are then read half as often. bf16, us
// with 16 and with 32: 24 rows of 4,096 -> 4,096 12.5 and 15.9, of 5,120 -> 5,120 27.3 and 20.7, of 8,192 -> 8,192 40
// and 31; one row of 3,072 -> 768 5.9 and 8.8, of 768 -> 3,072 3.5 and 4.6, of 5,120 -> 5,120 15.1 and 13.9 (3.8
// TB/s), of 8,192 -> 8,192 23.3 (5.8 TB/s) and 26.4: one row is quicker with 16 where they fill the chip evenly, which the rule
// does not look at. From 33 rows on the tiles' kernels are quicker (48 rows
// of 4,096 -> 4,096: 15.8 against 22).
template <int OP>
hipError_t launch_op(const ProductArgs& a, hipStream_t stream) {
  const bool wide = a.e.n > 16 * 256;
  if (a.e.m <= 16) return wide ? launch<OP, 1, 2, 8, 4>(a, stream) : launch<OP, 1, 1, 16, 2>(a, stream);
  return wide ? launch<OP, 2, 2, 8, 2>(a, stream) : launch<OP, 2, 1, 8, 4>(a, stream);
}

}  // namespace

hipError_t launch_product_rows(int32_t op, const ProductArgs& a, hipStream_t stream) {
  if (op == kOpF32) return launch_op<kOpF32>(a, stream);
  return op == kOpE4m3 ? launch_op<kOpE4m3>(a, stream) : launch_op<kOpBf16>(a, stream);
}

}  // namespace fwn
