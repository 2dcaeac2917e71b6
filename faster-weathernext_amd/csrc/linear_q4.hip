// Linear layers of 4-bit weights with a scale for each group of 32 inputs (gfx950): out = act(x w^T + b) + residual with
// w = value(code) 2^(e - 127), the codes OCP e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and e the group's
// OCP e8m0 scale. Such a weight is exact in bfloat16, so that products of widened weights are exact and added in float32.
//
// Few rows of x: bound by the weight's trip from memory, one pass over it with no partial products to join. A
// workgroup has 16 or 32 outputs, its waves share the sum, 128 inputs at a time: a lane's 16 bytes of codes
// are one group of one weight row, widened in registers by its scale to the MFMAs' operands (the order of k does not
// matter as long as both operands have the same); the waves' sums meet in LDS. More rows: the weight is widened
// once into the workspace for the tiles' kernels.
#include "linear_act_device.h"
#include "linear_q4.h"

namespace fwn {
namespace {

constexpr int GROUP = 32, LINE = 128;  // inputs of a scale, and of one step of a wave

// Two codes of byte BYTE of `codes` times 2^(e - 127), given as the float with the exponent field e (255: NaN).
template <int BYTE>
__device__ __forceinline__ uint32_t widen_bf16(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
}
typedef float f32x2 __attribute__((ext_vector_type(2)));
template <int BYTE>
__device__ __forceinline__ f32x2 widen_f32(uint32_t codes, float scale) {
  return __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, BYTE));
}
__device__ __forceinline__ float scale_of(uint32_t e) { return as_float(e << 23); }

// 8 codes as bf16.
__device__ __forceinline__ u32x4 widen8(uint32_t codes, float scale) {
  return u32x4{widen_bf16<0>(codes, scale), widen_bf16<1>(codes, scale), widen_bf16<2>(codes, scale), widen_bf16<3>(codes, scale)};
}

// The codes of the inputs from `left` on, of the eight in a word: zeros.
__device__ __forceinline__ uint32_t first_codes(uint32_t codes, int left) {
  return left >= 8 ? codes : left <= 0 ? 0 : codes & ((1u << 4 * left) - 1);
}

// The lane's group of codes of 16 weight rows: lane (i, g) row i, group g of a line.
struct Codes {
  rsrc_t codes, scales;
  uint32_t off, soff, groups;

  __device__ __forceinline__ void init(const Q4Args& a, int64_t first, int lane) {
    const int i = lane & 15, g = lane >> 4;
    groups = (uint32_t)a.groups;
    codes = make_rsrc(a.codes + first * groups * 16, kBuffer);
    scales = make_rsrc(a.scales + first * groups, kBuffer);
    const bool in = first + i < a.p.e.n;
    off = in ? ((uint32_t)i * groups + g) * 16 : kNowhere;
    soff = in ? (uint32_t)i * groups + g : kNowhere;
  }
  __device__ __forceinline__ u32x4 load(uint32_t line, int g) const {
    return bload16(codes, (off + line * 64) | (line * 4 + g < groups ? 0 : kNowhere));
  }
  __device__ __forceinline__ uint32_t scale(uint32_t line, int g) const {
    return __builtin_amdgcn_raw_buffer_load_b8(scales, (int)((soff + line * 4) | (line * 4 + g < groups ? 0 : kNowhere)), 0, 0);
  }
};

// The lane's group of x in 16 rows: as many pieces of 16 bytes as a group has.
template <bool F32>
struct Inputs {
  static constexpr int PIECES = F32 ? 8 : 4;
  rsrc_t r;
  uint32_t off, bytes;

  __device__ __forceinline__ void init(const ProductArgs& a, int64_t first, int lane) {
    const int i = lane & 15, g = lane >> 4;
    r = make_rsrc(a.a + first * a.a_stride, kBuffer);
    off = first + i < a.e.m ? (uint32_t)i * (uint32_t)a.a_stride + g * (PIECES * 16) : kNowhere;
    bytes = (uint32_t)a.k * (F32 ? 4 : 2);
  }
  // Zeros past the row. A float32 row may end inside a piece, and is not read past its end.
  __device__ __forceinline__ void load(uint32_t line, int g, u32x4 (&v)[PIECES]) const {
    const uint32_t at = line * (4 * PIECES * 16);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const uint32_t from = at + (g * PIECES + p) * 16, o = off + at + p * 16;
      if (!F32 || bytes % 16 == 0) {
        v[p] = bload16(r, o | (from < bytes ? 0 : kNowhere));
      } else if (at + 4 * PIECES * 16 <= bytes) {
        v[p] = bload16(r, o);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[p][e] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)((o + 4 * e) | (from + 4 * e < bytes ? 0 : kNowhere)), 0, 0);
      }
    }
  }
};

// c += the lane's group of codes times its group of x.
template <bool F32>
__device__ __forceinline__ f32x4 multiply(const u32x4& codes, float scale, const u32x4 (&x)[Inputs<F32>::PIECES], f32x4 c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t u = codes[t];
    if constexpr (F32) {
      const f32x2 w[4] = {widen_f32<0>(u, scale), widen_f32<1>(u, scale), widen_f32<2>(u, scale), widen_f32<3>(u, scale)};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t v = x[2 * t + e / 4][e % 4];
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e / 2][e % 2], as_float(v), c, 0, 0, 0);
      }
    } else {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, widen8(u, scale)), __builtin_bit_cast(bf16x8, x[t]), c, 0,
                                                  0, 0);
    }
  }
  return c;
}

// GROUPS 16-row groups of x by COLS 16-row groups of the weight; AHEAD lines of a wave on their way.
template <bool F32, int GROUPS, int COLS, int WAVES, int AHEAD>
__global__ void __launch_bounds__(64 * WAVES) q4_rows_kernel(Q4Args a) {
  __shared__ float red[WAVES][GROUPS][16][16 * COLS + 1];
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * COLS);
  const EpilogueArgs& e = a.p.e;
  Codes weight[COLS];
  Inputs<F32> x[GROUPS];
#pragma unroll
  for (int n = 0; n < COLS; ++n) weight[n].init(a, n0 + 16 * n, lane);
#pragma unroll
  for (int m = 0; m < GROUPS; ++m) x[m].init(a.p, 16 * m, lane);
  const uint32_t lines = (uint32_t)((a.p.k + LINE - 1) / LINE);
  f32x4 acc[GROUPS][COLS];
#pragma unroll
  for (int m = 0; m < GROUPS; ++m)
#pragma unroll
    for (int n = 0; n < COLS; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (uint32_t l0 = w; l0 < lines; l0 += WAVES * AHEAD) {
    u32x4 vw[AHEAD][COLS], vx[AHEAD][GROUPS][Inputs<F32>::PIECES];
    uint32_t vs[AHEAD][COLS];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const uint32_t line = l0 + WAVES * s;
#pragma unroll
      for (int n = 0; n < COLS; ++n) {
        vw[s][n] = weight[n].load(line, g);
        vs[s][n] = weight[n].scale(line, g);
      }
#pragma unroll
      for (int m = 0; m < GROUPS; ++m) x[m].load(line, g, vx[s][m]);
    }
    __builtin_amdgcn_sched_barrier(0);  // all loads before the first product
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const int left = (int)((int64_t)a.p.k - (int64_t)((l0 + WAVES * s) * 4 + g) * GROUP);
#pragma unroll
      for (int n = 0; n < COLS; ++n) {
        u32x4 codes = vw[s][n];
        if (left < GROUP) {
#pragma unroll
          for (int t = 0; t < 4; ++t) codes[t] = first_codes(codes[t], left - 8 * t);
        }
        const float scale = scale_of(vs[s][n]);
#pragma unroll
        for (int m = 0; m < GROUPS; ++m) acc[m][n] = multiply<F32>(codes, scale, vx[s][m], acc[m][n]);
      }
    }
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
      if (e.bias) z += load_one(e.bias, col, e.dtype);
      z = activate<decltype(act)::kind, F32>(z);
      if (e.residual) z += load_one(e.residual, row * e.r_row + col, e.dtype);
      store_one(e.out, row * e.n + col, e.dtype, z);
    }
  });
}

// The weight as bf16 or float32 [outs, 32 groups], zeros past the inputs: 16 bytes a thread.
template <bool F32>
__global__ void __launch_bounds__(256) widen_kernel(WidenArgs a) {
  constexpr int PER = F32 ? 8 : 4;  // threads a group
  const int64_t across = a.groups * PER, total = a.outs * across;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / across, at = id - row * across;
    const float scale = scale_of(a.scales[row * a.groups + at / PER]);
    const int64_t left = a.ins - at * (GROUP / PER);
    u32x4 v;
    if constexpr (F32) {
      const uint32_t u = first_codes(((const uint16_t*)a.codes)[id], left < 4 ? (int)left : 4);
      const f32x2 lo = widen_f32<0>(u, scale), hi = widen_f32<1>(u, scale);
      v = u32x4{as_bits(lo[0]), as_bits(lo[1]), as_bits(hi[0]), as_bits(hi[1])};
    } else {
      v = widen8(first_codes(((const uint32_t*)a.codes)[id], left < 8 ? (int)left : 8), scale);
    }
    *(u32x4*)(a.dst + id * 16) = v;
  }
}

// Codes and scales of rows: a group a thread.
template <typename T>
__global__ void __launch_bounds__(256) quantize_q4_kernel(QuantizeQ4Args a) {
  const int64_t groups = (a.cols + GROUP - 1) / GROUP, total = a.rows * groups;
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < total; id += (int64_t)gridDim.x * 256) {
    const int64_t row = id / groups, c0 = (id - row * groups) * GROUP;
    const T* x = (const T*)a.x + row * a.x_stride + c0;
    const int left = (int)(a.cols - c0 < GROUP ? a.cols - c0 : GROUP);
    float f[GROUP];
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < GROUP; ++k) {
      f[k] = k < left ? load_one(x, k, sizeof(T) == 4 ? FWN_F32 : FWN_BF16) : 0.f;
      const uint32_t u = as_bits(f[k]) & 0x7fffffffu;
      most = u > most ? u : most;
    }
    // The least 2^k of which the largest magnitude is at most seven: beyond six it is cut to six, where the next scale's codes
    // would be six and eight, as far off. Numbers that are not finite: the scale NaN.
    int32_t e = (int32_t)(most >> 23) - ((most & 0x7fffffu) > 0x600000u ? 1 : 2);
    e = e < 0 ? 0 : e;
    if (most >= 0x7f800000u) e = 255;
    a.scales[id] = (uint8_t)e;
    const float inv = e == 255 ? 0.f : as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e)
    uint32_t d[4] = {};
#pragma unroll
    for (int k = 0; k < GROUP; ++k) {
      const float v = __builtin_fabsf(f[k]) * inv;  // exact; to the nearest code, middles to even ones
      const uint32_t code = (uint32_t)(v > 0.25f) + (v >= 0.75f) + (v > 1.25f) + (v >= 1.75f) + (v > 2.5f) + (v >= 3.5f) + (v > 5.f);
      d[k / 8] |= (e == 255 ? 0 : code | (as_bits(f[k]) >> 31) << 3) << 4 * (k % 8);
    }
    *(u32x4*)(a.codes + id * 16) = u32x4{d[0], d[1], d[2], d[3]};
  }
}

constexpr int64_t kMostBlocks = 1 << 20;  // of a pass; more are looped over

dim3 pass_grid(int64_t threads) {
  const int64_t blocks = (threads + 255) / 256;
  return dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks));
}

template <bool F32, int GROUPS, int COLS, int WAVES, int AHEAD>
hipError_t launch(const Q4Args& a, hipStream_t stream) {
  hipLaunchKernelGGL((q4_rows_kernel<F32, GROUPS, COLS, WAVES, AHEAD>), dim3((unsigned)((a.p.e.n + 16 * COLS - 1) / (16 * COLS))),
                     dim3(64 * WAVES), 0, stream, a);
  return hipGetLastError();
}

template <bool F32>
hipError_t launch_as(const Q4Args& a, hipStream_t stream) {
  const bool wide = a.p.e.n > 16 * 256;
  if (a.p.e.m <= 16) return wide ? launch<F32, 1, 2, 8, 2>(a, stream) : launch<F32, 1, 1, 16, 2>(a, stream);
  return wide ? launch<F32, 2, 2, 8, 2>(a, stream) : launch<F32, 2, 1, 8, 2>(a, stream);
}

}  // namespace

hipError_t launch_q4_rows(bool f32, const Q4Args& a, hipStream_t stream) {
  return f32 ? launch_as<true>(a, stream) : launch_as<false>(a, stream);
}

hipError_t launch_widen(bool f32, const WidenArgs& a, hipStream_t stream) {
  if (f32)
    hipLaunchKernelGGL(widen_kernel<true>, pass_grid(a.outs * a.groups * 8), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(widen_kernel<false>, pass_grid(a.outs * a.groups * 4), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_quantize_q4(int dtype, const QuantizeQ4Args& a, hipStream_t stream) {
  const dim3 grid = pass_grid(a.rows * ((a.cols + GROUP - 1) / GROUP));
  if (dtype == FWN_F32)
    hipLaunchKernelGGL(quantize_q4_kernel<float>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(quantize_q4_kernel<uint16_t>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace fwn
