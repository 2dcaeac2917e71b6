// Device-side building blocks of the linear layers' kernels: elements, activations, the epilogue of a product's
// tile and the order of the tiles (gfx950).
#pragma once

#include <type_traits>

#include "attn_bf16_tiles.h"
#include "linear_act.h"

namespace fwn {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ uint32_t bf16_bits(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

__device__ __forceinline__ float load_one(const void* p, int64_t i, int dtype) {
  if (dtype == FWN_F32) return ((const float*)p)[i];
  return as_float((uint32_t)((const uint16_t*)p)[i] << 16);
}

__device__ __forceinline__ void store_one(void* p, int64_t i, int dtype, float v) {
  if (dtype == FWN_F32)
    ((float*)p)[i] = v;
  else
    ((uint16_t*)p)[i] = (uint16_t)bf16_bits(v);
}

// Eight consecutive elements, 16-byte aligned.
__device__ __forceinline__ void load8(const void* p, int64_t i, int dtype, float (&f)[8]) {
  if (dtype == FWN_F32) {
    const u32x4* q = (const u32x4*)((const float*)p + i);
    const u32x4 v0 = q[0], v1 = q[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t a = v0[k], b = v1[k];
      f[k] = as_float(a);
      f[4 + k] = as_float(b);
    }
  } else {
    const u32x4 v = *(const u32x4*)((const uint16_t*)p + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t u = v[k];
      f[2 * k] = as_float(u << 16);
      f[2 * k + 1] = as_float(u & 0xffff0000u);
    }
  }
}

__device__ __forceinline__ u32x4 pack8(const float (&f)[8]) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = bf16_bits(f[2 * k]) | bf16_bits(f[2 * k + 1]) << 16;
  return v;
}

__device__ __forceinline__ void store8(void* p, int64_t i, int dtype, const float (&f)[8]) {
  if (dtype == FWN_F32) {
    u32x4* q = (u32x4*)((float*)p + i);
    q[0] = u32x4{as_bits(f[0]), as_bits(f[1]), as_bits(f[2]), as_bits(f[3])};
    q[1] = u32x4{as_bits(f[4]), as_bits(f[5]), as_bits(f[6]), as_bits(f[7])};
  } else {
    *(u32x4*)((uint16_t*)p + i) = pack8(f);
  }
}

// Eight e4m3 codes as the bf16 values that they are exactly.
__device__ __forceinline__ u32x4 widen(uint32_t lo, uint32_t hi) {
  const auto two = [](uint32_t codes, auto high) {
    return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, decltype(high)::value));
  };
  return u32x4{two(lo, std::false_type()), two(lo, std::true_type()), two(hi, std::false_type()), two(hi, std::true_type())};
}

// The activations' functions for outputs of float32 (F32), and of bf16: e^x on the transcendental unit, off by up to
// (1 + |x|) 2^-23 of itself, its reciprocal there, zero below 2^-126, and erfc by Abramowitz and Stegun's 7.1.26, off by
// up to 1e-6 in float32 (1.5e-7 without its roundings) and, where it is small itself, by up to 0.4% of it for z down to -6.2,
// one rounding of a bf16 output. float32 outputs with bf16's functions and with their own, us of 10,242 x 768 -> 3,072: gelu 267
// and 286, gelu_tanh 258 and 264, silu 257 and 262.
template <bool F32>
constexpr float kLog = F32 ? 1.f : LOG2E;
template <bool F32>
__device__ __forceinline__ float power(float x) {  // e^(x / kLog)
  if constexpr (F32) return expf(x);
  return fast_exp2(x);
}

// (1 + erf(z / sqrt 2)) / 2, formed of erfc so that the small values of negative z keep their digits: the sum leaves
// none from z = -5.5 on.
template <bool F32>
__device__ __forceinline__ float normal_cdf(float z) {
  const float x = z * 0.7071067811865476f;
  if constexpr (F32) return 0.5f * erfcf(-x);
  const float y = __builtin_fabsf(x), t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, y, 1.f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float c = 0.5f * p * t * fast_exp2(-y * y * LOG2E);
  return z > 0.f ? 1.f - c : c;
}

// p = 1 / (1 + e^(x / kLog)) and q = 1 - p. float32: of e^-|x|, which leaves neither the range nor digits behind.
struct Logistic {
  float p, q;
};
template <bool F32>
__device__ __forceinline__ Logistic logistic(float x) {
  if constexpr (F32) {
    const float e = expf(-__builtin_fabsf(x)), r = __builtin_amdgcn_rcpf(1.f + e);
    return x > 0.f ? Logistic{e * r, r} : Logistic{r, e * r};
  }
  const float p = __builtin_amdgcn_rcpf(1.f + fast_exp2(x));
  return {p, 1.f - p};
}

constexpr float kTanh = 0.7978845608028654f, kCube = 0.044715f;  // gelu_tanh: u = kTanh (z + kCube z^3)

// -2 u kLog of z, z2 = z^2.
template <bool F32>
__device__ __forceinline__ float tanh_arg(float z, float z2) {
  return z * fmaf(z2, -2.f * kTanh * kCube * kLog<F32>, -2.f * kTanh * kLog<F32>);
}

// act(z). The tanh form is z / (1 + e^(-2u)).
template <int KIND, bool F32>
__device__ __forceinline__ float activate(float z) {
  if constexpr (KIND == FWN_ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if constexpr (KIND == FWN_ACT_GELU) return z * normal_cdf<F32>(z);
  if constexpr (KIND == FWN_ACT_GELU_TANH) return z * logistic<F32>(tanh_arg<F32>(z, z * z)).p;
  if constexpr (KIND == FWN_ACT_SILU) return z * logistic<F32>(-z * kLog<F32>).p;
  return z;
}

// act'(z).
template <int KIND, bool F32>
__device__ __forceinline__ float slope(float z) {
  if constexpr (KIND == FWN_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (KIND == FWN_ACT_GELU)
    return normal_cdf<F32>(z) + z * power<F32>(-0.5f * z * z * kLog<F32>) * 0.3989422804014327f;
  if constexpr (KIND == FWN_ACT_GELU_TANH) {
    // p + 2 z p (1 - p) u'; beyond 12 p is 0 or 1, and a large z^2 would meet that 0.
    const float y = z > 12.f ? 12.f : z < -12.f ? -12.f : z, y2 = y * y;
    const Logistic l = logistic<F32>(tanh_arg<F32>(y, y2));
    return fmaf(2.f * y * l.p * l.q, fmaf(y2, 3.f * kTanh * kCube, kTanh), l.p);
  }
  if constexpr (KIND == FWN_ACT_SILU) {
    const Logistic l = logistic<F32>(-z * kLog<F32>);
    return l.p * fmaf(l.p > 0.f ? z : 0.f, l.q, 1.f);
  }
  return 1.f;
}

// Calls f with the activation as a compile-time constant.
template <int KIND>
struct Act {
  static constexpr int kind = KIND;
};
template <bool PLAIN, typename F>
__device__ __forceinline__ void with_activation(int kind, F&& f) {
  if constexpr (PLAIN) return f(Act<FWN_ACT_NONE>());
  switch (kind) {
    case FWN_ACT_RELU: return f(Act<FWN_ACT_RELU>());
    case FWN_ACT_GELU: return f(Act<FWN_ACT_GELU>());
    case FWN_ACT_GELU_TANH: return f(Act<FWN_ACT_GELU_TANH>());
    case FWN_ACT_SILU: return f(Act<FWN_ACT_SILU>());
    default: return f(Act<FWN_ACT_NONE>());
  }
}

// What the epilogue needs of the columns col .. col + 7.
struct Columns {
  float bias[8], scale[8];

  __device__ __forceinline__ void load(const EpilogueArgs& e, int64_t col) {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const bool in = col + k < e.n;
      bias[k] = e.bias && in ? load_one(e.bias, col + k, e.dtype) : 0.f;
      scale[k] = e.b_scale && in ? e.b_scale[col + k] : 1.f;
    }
  }
};

// The epilogue of z[row, col .. col + 7] in rows of whole aligned eights.
template <int KIND, bool F32>
__device__ __forceinline__ void finish(const EpilogueArgs& e, int64_t row, int64_t col, float (&v)[8], const Columns& c) {
  if (e.a_scale) {
    const float s = e.a_scale[row];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = v[k] * s * c.scale[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += c.bias[k];
  const int64_t at = row * e.n + col;
  if (e.pre) store8(e.pre, at, e.dtype, v);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = activate<KIND, F32>(v[k]);
  if (e.residual) {
    float r[8];
    load8(e.residual, row * e.r_row + col, e.dtype, r);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += r[k];
  }
  store8(e.out, at, e.dtype, v);
}

// Offsets with the top bit set lie past every buffer's end: loads give zeros and stores are dropped.
constexpr uint32_t kNowhere = 0x80000000u, kBuffer = 0x7fffffffu;

// What a workgroup computes: a tile of c and a range of the sum.
struct Work {
  int split;
  int64_t i0, j0;
};

constexpr int kBand = 8;

// Workgroups go to the 8 XCDs in turn: each takes a contiguous range of (range of the sum, tile). Tiles run in
// bands of kBand rows of them, column by column: what runs at once on an XCD shares rows of both operands.
template <int BM, int BN>
__device__ __forceinline__ Work work_of(const EpilogueArgs& e) {
  const int total = (int)gridDim.x, xcd = (int)blockIdx.x & 7, per = total >> 3, rem = total & 7;
  const int id = xcd * per + (xcd < rem ? xcd : rem) + ((int)blockIdx.x >> 3);
  const int tn = (int)((e.n + BN - 1) / BN), tm = (int)((e.m + BM - 1) / BM), tiles = tm * tn;
  Work k;
  k.split = id / tiles;
  const int tile = id - k.split * tiles, band = tile / (kBand * tn), in = tile - band * (kBand * tn);
  const int high = tm - band * kBand < kBand ? tm - band * kBand : kBand;
  k.i0 = (int64_t)(band * kBand + in % high) * BM;
  k.j0 = (int64_t)(in / high) * BN;
  return k;
}

typedef __attribute__((address_space(3))) float* strip_ptr;
// Fours at any address of an element.
typedef uint32_t bf16x4_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kStrip = 72;                      // floats from one row of a strip to the next: eight rows' fours fall in other banks
constexpr int kStripBytes = 32 * kStrip * 4;    // of LDS, for each wave
static_assert(kStripBytes >= 64 * 128, "a strip of 64 rows of bf16, chunk c of row r at c ^ (r / 2 % 8)");

// Whether a product's outputs are bf16 that nothing but their column's bias is added to, in rows of whole aligned eights.
template <bool PLAIN>
__device__ __forceinline__ bool bf16_rows(const ProductArgs& g) {
  return !g.part && g.e.vec && g.e.dtype == FWN_BF16 && (PLAIN || (!g.e.pre && !g.e.residual));
}

// What the epilogue of those needs of memory for a wave's part, in the layout of its registers: asked for before the last
// barrier, and before the stores, which a later load would wait for.
template <int MI, bool PLAIN, bool SCALED>
struct Bf16Terms {
  u32x2 bias[2][4];
  u32x4 scale[2][4];
  float a_scale[MI];

  __device__ __forceinline__ void load(const EpilogueArgs& e, const Work& k, int rows, int wm, int wn, int lane) {
    const int j = lane & 31, half = lane >> 5;
    if constexpr (!PLAIN) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t col = k.j0 + wn + 32 * n + 8 * q + 4 * half;
          bias[n][q] = e.bias && col < e.n ? *(const bf16x4_any*)((const uint16_t*)e.bias + col) : u32x2{0, 0};
          if constexpr (SCALED) scale[n][q] = col < e.n ? *(const f32x4_any*)(e.b_scale + col) : u32x4{0, 0, 0, 0};
        }
    }
    if constexpr (SCALED) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int row = wm + 32 * m + j;
        a_scale[m] = row < rows ? e.a_scale[k.i0 + row] : 0.f;
      }
    }
  }
};

// The epilogue of a wave's 32 MI x 64 part (from row wm and column wn) of a BM-row tile. The products are formed with
// the weight's side as the MFMA's rows, so that a lane's registers are fours of columns of one row (acc[m][n][4 q + i]:
// row 32 m + lane % 32, column 32 n + 8 q + 4 (lane / 32) + i), which go to LDS whole (gx of 10,242 x 768 with 3,072
// outputs 62 us with single columns, 57 so): 32 rows at a time through the wave's strip to rows of eight columns a
// lane, or of one column a lane where rows are not whole aligned eights. bf16 outputs that nothing but their column's
// bias is added to are finished where the MFMAs leave them and go through LDS as bf16, 64 rows at a time. PLAIN: no
// epilogue but the rounding (gradients). F32: the outputs are float32, else bf16. mend(row, col, v) may change outputs
// before the epilogue.
template <int BM, int MI, bool PLAIN, bool F32, bool SCALED, typename Mend>
__device__ __forceinline__ void write_tile(const ProductArgs& g, const Work& k, const f32x16 (&acc)[MI][2], strip_ptr strip,
                                           int wm, int wn, int lane, const Bf16Terms<MI, PLAIN, SCALED>& terms, const Mend& mend) {
  const int j = lane & 31, half = lane >> 5;
  const auto to_strip = [&](int m) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(__attribute__((address_space(3))) f32x4*)(strip + j * kStrip + 32 * n + 8 * q + 4 * half) =
            f32x4{acc[m][n][4 * q], acc[m][n][4 * q + 1], acc[m][n][4 * q + 2], acc[m][n][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
  };
  const EpilogueArgs& e = g.e;
  const int rows = (int)(e.m - k.i0 < BM ? e.m - k.i0 : BM);  // of the tile
  if constexpr (!F32) {
    if (bf16_rows<PLAIN>(g)) {
      static_assert(MI % 2 == 0, "64 rows at a time");
      typedef __attribute__((address_space(3))) char* bytes_ptr;
      bytes_ptr const half_strip = (bytes_ptr)strip;
      const rsrc_t ro = make_rsrc((char*)e.out + (k.i0 * e.n + k.j0) * 2, kBuffer);
      const int sub = lane >> 3, at_col = wn + 8 * (lane & 7);
      const uint32_t nowhere = k.j0 + at_col < e.n ? 0 : kNowhere;
      with_activation<PLAIN>(e.activation, [&](auto act) {
#pragma unroll
        for (int m0 = 0; m0 < MI; m0 += 2) {
#pragma unroll
          for (int m = m0; m < m0 + 2; ++m) {
            const int strip_row = 32 * (m - m0) + j;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                float v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  v[i] = acc[m][n][4 * q + i];
                  if constexpr (SCALED) {
                    const uint32_t u = terms.scale[n][q][i];
                    v[i] = v[i] * terms.a_scale[m] * as_float(u);
                  }
                  if constexpr (!PLAIN) {
                    const uint32_t u = terms.bias[n][q][i / 2];
                    v[i] = activate<decltype(act)::kind, false>(v[i] + as_float(i % 2 ? u & 0xffff0000u : u << 16));
                  }
                }
                *(__attribute__((address_space(3))) u32x2*)(half_strip + strip_row * 128 +
                                                            (((4 * n + q) ^ (strip_row / 2 % 8)) << 4) + 8 * half) =
                    u32x2{bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16};
              }
          }
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int p = 0; p < 8; ++p) {
            const int strip_row = 8 * p + sub, row = wm + 32 * m0 + strip_row;
            const u32x4 v = *(const __attribute__((address_space(3))) u32x4*)(half_strip + strip_row * 128 +
                                                                              (((lane & 7) ^ (strip_row / 2 % 8)) << 4));
            __builtin_amdgcn_raw_buffer_store_b128(
                v, ro, (int)(((uint32_t)row * (uint32_t)e.n + (uint32_t)at_col) * 2 | (row < rows ? 0 : kNowhere) | nowhere), 0, 0);
          }
          __builtin_amdgcn_wave_barrier();
        }
      });
      return;
    }
  }
  if (g.part || e.vec) {
    // Offsets in the tile.
    const bool f32 = g.part || F32;
    const int64_t width = g.part ? g.part_row : e.n;
    const uint32_t shift = f32 ? 2 : 1;
    char* const to = g.part ? (char*)(g.part + (int64_t)k.split * e.m * g.part_row) : (char*)e.out;
    const rsrc_t ro = make_rsrc(to + ((k.i0 * width + k.j0) << shift), kBuffer);
    const rsrc_t rp = make_rsrc((char*)e.pre + ((k.i0 * width + k.j0) << shift), kBuffer);
    const rsrc_t rr = make_rsrc((const char*)e.residual + ((k.i0 * e.r_row + k.j0) << shift), kBuffer);
    const bool pre = !PLAIN && !g.part && e.pre, residual = !PLAIN && !g.part && e.residual;
    const int sub = lane >> 3, at_col = wn + 8 * (lane & 7);  // this lane's row of eight and its columns of the tile
    const int64_t col = k.j0 + at_col;
    const uint32_t nowhere = col < e.n ? 0 : kNowhere;
    Columns c;
    if (!PLAIN && !g.part) c.load(e, col);
    // The residual of 32 rows is asked for before the stores of the 32 before them, which a later load would wait for (where
    // registers allow it).
    constexpr bool AHEAD = F32 || !SCALED;
    u32x4 next[AHEAD ? 2 : 1][4][2];
    const auto ask = [&](int m) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int row = wm + 32 * m + 8 * p + sub;
        const uint32_t o = (row < rows ? 0 : kNowhere) | nowhere | (((uint32_t)row * (uint32_t)e.r_row + (uint32_t)at_col) << shift);
        next[AHEAD ? m & 1 : 0][p][0] = bload16(rr, o);
        if (F32) next[AHEAD ? m & 1 : 0][p][1] = bload16(rr, o + 16);
      }
    };
    const auto asked = [&](int m, int p, float(&f)[8]) {
      const u32x4 lo = next[AHEAD ? m & 1 : 0][p][0], hi = next[AHEAD ? m & 1 : 0][p][1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t x = lo[i], y = hi[i];
        if (F32) {
          f[i] = as_float(x);
          f[4 + i] = as_float(y);
        } else {
          f[2 * i] = as_float(x << 16);
          f[2 * i + 1] = as_float(x & 0xffff0000u);
        }
      }
    };
    const auto store = [&](rsrc_t r, uint32_t o, const float(&f)[8]) {
      if (f32) {
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{as_bits(f[0]), as_bits(f[1]), as_bits(f[2]), as_bits(f[3])}, r, (int)o, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{as_bits(f[4]), as_bits(f[5]), as_bits(f[6]), as_bits(f[7])}, r, (int)(o + 16), 0, 0);
      } else {
        __builtin_amdgcn_raw_buffer_store_b128(pack8(f), r, (int)o, 0, 0);
      }
    };
    if (AHEAD && residual) ask(0);
    with_activation<PLAIN>(g.part ? FWN_ACT_NONE : e.activation, [&](auto act) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        to_strip(m);
        if (residual && m + AHEAD < MI) ask(m + AHEAD);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int row = wm + 32 * m + 8 * p + sub;
          const uint32_t out = (row < rows ? 0 : kNowhere) | nowhere;
          const uint32_t o = out | (((uint32_t)row * (uint32_t)width + (uint32_t)at_col) << shift);
          float v[8];
          const auto* q = (const __attribute__((address_space(3))) f32x4*)(strip + (8 * p + sub) * kStrip + 8 * (lane & 7));
          const f32x4 lo = q[0], hi = q[1];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = lo[i], y = hi[i];
            v[i] = x;
            v[4 + i] = y;
          }
          if (!g.part) {
            if (out == 0) mend(k.i0 + row, col, v);
            if (SCALED) {
              const float s = row < rows ? e.a_scale[k.i0 + row] : 0.f;
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = v[i] * s * c.scale[i];
            }
            if (!PLAIN) {
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] += c.bias[i];
              if (pre) store(rp, o, v);
#pragma unroll
              for (int i = 0; i < 8; ++i) v[i] = activate<decltype(act)::kind, F32>(v[i]);
              if (residual) {
                float r[8];
                asked(m, p, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += r[i];
              }
            }
          }
          store(ro, o, v);
        }
        __builtin_amdgcn_wave_barrier();
      }
    });
    return;
  }
  const int64_t col = k.j0 + wn + lane;
  const bool in = col < e.n;
  const float bias = !PLAIN && e.bias && in ? load_one(e.bias, col, e.dtype) : 0.f;
  const float scale = SCALED && in ? e.b_scale[col] : 1.f;
  const uint32_t shift = F32 ? 2 : 1;
  const rsrc_t ro = make_rsrc((char*)e.out + ((k.i0 * e.n + k.j0) << shift), kBuffer);
  const rsrc_t rp = make_rsrc((char*)e.pre + ((k.i0 * e.n + k.j0) << shift), kBuffer);
  const rsrc_t rr = make_rsrc((const char*)e.residual + ((k.i0 * e.r_row + k.j0) << shift), kBuffer);
  const auto store = [&](rsrc_t r, uint32_t o, float v) {
    if (F32)
      __builtin_amdgcn_raw_buffer_store_b32(as_bits(v), r, (int)o, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b16((uint16_t)bf16_bits(v), r, (int)o, 0, 0);
  };
  with_activation<PLAIN>(e.activation, [&](auto act) {
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      to_strip(m);
#pragma unroll 1
      for (int r0 = 0; r0 < 32; r0 += 8) {  // eight rows' residuals are on their way at once
        uint32_t out[8];
        float z[8], res[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int row = wm + 32 * m + r0 + r;
          out[r] = in && row < rows ? 0 : kNowhere;
          res[r] = 0.f;
          if (!PLAIN && e.residual) {
            const uint32_t o = out[r] | (((uint32_t)row * (uint32_t)e.r_row + (uint32_t)(wn + lane)) << shift);
            res[r] = F32 ? as_float(__builtin_amdgcn_raw_buffer_load_b32(rr, (int)o, 0, 0))
                         : as_float((uint32_t)__builtin_amdgcn_raw_buffer_load_b16(rr, (int)o, 0, 0) << 16);
          }
          z[r] = strip[(r0 + r) * kStrip + lane];
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const int row = wm + 32 * m + r0 + r;
          const uint32_t o = out[r] | (((uint32_t)row * (uint32_t)e.n + (uint32_t)(wn + lane)) << shift);
          float v[1] = {z[r]};
          if (out[r] == 0) mend(k.i0 + row, col, v);
          if (SCALED && row < rows) v[0] = v[0] * e.a_scale[k.i0 + row] * scale;
          if (!PLAIN) {
            v[0] += bias;
            if (e.pre) store(rp, o, v[0]);
            v[0] = activate<decltype(act)::kind, F32>(v[0]);
            if (e.residual) v[0] += res[r];
          }
          store(ro, o, v[0]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  });
}

constexpr float kUp = 65536.f;  // of a float32 operand's parts, see linear_act_f32.hip

// float32 products are formed of three bf16 parts of each value times kUp: outputs are divided by kUp^2, and those that
// came out infinite or NaN formed anew of the whole values. OUTER: the operand's rows are k.
template <bool OA, bool OB>
struct MendParts {
  const ProductArgs& g;

  template <bool OUTER>
  __device__ __forceinline__ static float value(const char* p, int64_t stride, int64_t i, int64_t k) {
    return *(const float*)(OUTER ? p + k * stride + i * 4 : p + i * stride + k * 4);
  }

  template <int N>
  __device__ __forceinline__ void operator()(int64_t row, int64_t col, float (&v)[N]) const {
    const auto lost = [&](int e) { return !(__builtin_fabsf(v[e]) < __builtin_inff()); };
    bool bad = false;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      v[e] *= 1.f / (kUp * kUp);
      bad |= lost(e);
    }
    if (!bad) return;
    float s[N] = {};
    for (int64_t k = 0; k < g.k && bad; ++k) {  // until every one is NaN for good
      const float x = value<OA>(g.a, g.a_stride, row, k);
      bad = false;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (col + e < g.e.n) s[e] = fmaf(x, value<OB>(g.b, g.b_stride, col + e, k), s[e]);
        bad |= lost(e) && s[e] == s[e];
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (lost(e)) v[e] = s[e];
  }
};

struct MendNothing {
  template <int N>
  __device__ __forceinline__ void operator()(int64_t, int64_t, float (&)[N]) const {}
};

// The partial products added in the order of the splits, then the epilogue: N columns a thread, eight where rows are
// whole aligned eights, else one, so that a wave's accesses still lie side by side. F32: the outputs are float32.
template <bool PLAIN, bool F32, int N, typename Mend>
__device__ __forceinline__ void join(const ProductArgs& g, const Mend& mend) {
  const EpilogueArgs& e = g.e;
  const int64_t across = N == 8 ? g.part_row / 8 : e.n, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / across, col = (id - row * across) * N;
  if (row >= e.m) return;
  float v[N] = {};
#pragma unroll 4
  for (int s = 0; s < g.splits; ++s) {
    const int64_t at = ((int64_t)s * e.m + row) * g.part_row + col;
    if constexpr (N == 8) {
      float p[8];
      load8(g.part, at, FWN_F32, p);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += p[k];
    } else {
      v[0] += g.part[at];
    }
  }
  mend(row, col, v);
  with_activation<PLAIN>(e.activation, [&](auto act) {
    if constexpr (N == 8) {
      Columns c;
      c.load(e, col);
      finish<decltype(act)::kind, F32>(e, row, col, v, c);
    } else {
      float z = v[0];
      if (e.a_scale) z = z * e.a_scale[row] * e.b_scale[col];
      if (e.bias) z += load_one(e.bias, col, e.dtype);
      if (e.pre) store_one(e.pre, row * e.n + col, e.dtype, z);
      z = activate<decltype(act)::kind, F32>(z);
      if (e.residual) z += load_one(e.residual, row * e.r_row + col, e.dtype);
      store_one(e.out, row * e.n + col, e.dtype, z);
    }
  });
}

inline dim3 join_grid(const ProductArgs& g) {
  return dim3((unsigned)((g.e.m * (g.e.vec ? g.part_row / 8 : g.e.n) + 255) / 256));
}

}  // namespace
}  // namespace fwn
