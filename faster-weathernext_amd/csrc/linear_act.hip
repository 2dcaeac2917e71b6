// Matrix products with bias, activation and residual in their epilogue, and their gradients (gfx950):
//
//   z = x w^T + b,  out = act(z) + residual;   dz = g act'(z),  gx = dz w,  gw = dz^T x,  gb = sum of dz
//
// One kernel for the three products c[i, j] = sum over k of a(i, k) b(j, k): an operand whose rows are
// contiguous in k ("inner": x, w and dz in the first two) is read from LDS row by row, one whose rows are k
// ("outer": w in gx, dz and x in gw) by transpose reads, and both arrive as the same MFMA operands.
// float32 operands are laid out as three bf16 parts, 8 bits of the value each, and the product is the sum of
// the six products of parts above 2^-24 of it, accumulated in float32 on the bf16 matrix units.
#include "attn_bf16_tiles.h"
#include "linear_act.h"

namespace fwn {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

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

// e^x and 1 / x on the transcendental unit, within two units in the last place.
__device__ __forceinline__ float fast_exp(float x) { return fast_exp2(x * LOG2E); }
__device__ __forceinline__ float fast_rcp(float x) { return __builtin_amdgcn_rcpf(x); }

// erf by Abramowitz and Stegun's 7.1.26, off by at most 1.5e-7 (a value times z / 2 here).
__device__ __forceinline__ float erf_of(float x) {
  const float y = __builtin_fabsf(x), t = fast_rcp(fmaf(0.3275911f, y, 1.f));
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  return __builtin_copysignf(1.f - p * t * fast_exp(-y * y), x);
}

constexpr float kTanh = 0.7978845608028654f, kCube = 0.044715f;  // gelu_tanh: u = kTanh (z + kCube z^3)

// act(z). The tanh form is z / (1 + e^(-2u)).
template <int KIND>
__device__ __forceinline__ float activate(float z) {
  if constexpr (KIND == FWN_ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if constexpr (KIND == FWN_ACT_GELU) return 0.5f * z * (1.f + erf_of(z * 0.7071067811865476f));
  if constexpr (KIND == FWN_ACT_GELU_TANH)
    return z * fast_rcp(1.f + fast_exp2(z * fmaf(z * z, -2.f * kTanh * kCube * LOG2E, -2.f * kTanh * LOG2E)));
  if constexpr (KIND == FWN_ACT_SILU) return z * fast_rcp(1.f + fast_exp(-z));
  return z;
}

// act'(z).
template <int KIND>
__device__ __forceinline__ float slope(float z) {
  if constexpr (KIND == FWN_ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if constexpr (KIND == FWN_ACT_GELU)
    return 0.5f * (1.f + erf_of(z * 0.7071067811865476f)) + z * fast_exp(-0.5f * z * z) * 0.3989422804014327f;
  if constexpr (KIND == FWN_ACT_GELU_TANH) {
    // p = 1 / (1 + e^(-2u)), p + 2 z p (1 - p) u'; beyond 12 it is 0 or 1, and a large z^2 would meet that 0.
    const float y = z > 12.f ? 12.f : z < -12.f ? -12.f : z, q = y * y;
    const float p = fast_rcp(1.f + fast_exp2(y * fmaf(q, -2.f * kTanh * kCube * LOG2E, -2.f * kTanh * LOG2E)));
    return fmaf(2.f * y * p * (1.f - p), fmaf(q, 3.f * kTanh * kCube, kTanh), p);
  }
  if constexpr (KIND == FWN_ACT_SILU) {
    const float p = fast_rcp(1.f + fast_exp(-z)), y = p > 0.f ? z : 0.f;
    return p * fmaf(y, 1.f - p, 1.f);
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

// The epilogue of z[row, col .. col + 7], row < m; columns from n on are dropped.
template <int KIND>
__device__ __forceinline__ void finish(const EpilogueArgs& e, int64_t row, int64_t col, float (&v)[8], const Columns& c) {
  if (e.a_scale) {
    const float s = e.a_scale[row];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] *= s * c.scale[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] += c.bias[k];
  const int64_t at = row * e.n + col;
  if (e.vec) {
    if (col >= e.n) return;
    if (e.pre) store8(e.pre, at, e.dtype, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = activate<KIND>(v[k]);
    if (e.residual) {
      float r[8];
      load8(e.residual, row * e.r_row + col, e.dtype, r);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] += r[k];
    }
    store8(e.out, at, e.dtype, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (col + k >= e.n) break;
      if (e.pre) store_one(e.pre, at + k, e.dtype, v[k]);
      float o = activate<KIND>(v[k]);
      if (e.residual) o += load_one(e.residual, row * e.r_row + col + k, e.dtype);
      store_one(e.out, at + k, e.dtype, o);
    }
  }
}

// Planes of a and b in each term of a product of parts, a digit a term from the right. The small terms come
// first, where the accumulator's rounding hurts them least.
constexpr uint32_t kPlaneA = 0x001102, kPlaneB = 0x010120;

// An operand's float32 value at (row, k) from its three parts.
template <bool OUTER>
__device__ __forceinline__ float whole(const char* p, int64_t stride, int64_t plane, int64_t row, int64_t k) {
  const char* q = OUTER ? p + k * stride + row * 2 : p + row * stride + k * 2;
  float s = 0.f;
  for (int i = 2; i >= 0; --i) s += as_float((uint32_t)*(const uint16_t*)(q + i * plane) << 16);
  return s;
}

// Outputs of a product of parts that are NaN, formed from whole values: an infinity's parts beside it are
// zeros, and so are those of a short number, whose product is NaN where the whole one is infinite.
template <bool OA, bool OB>
__device__ __forceinline__ void mend(const ProductArgs& g, int64_t row, int64_t col, float (&v)[8]) {
  bool bad = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) bad |= v[e] != v[e] && col + e < g.e.n;
  if (!bad) return;
  float s[8] = {};
  for (int64_t k = 0; k < g.k; ++k) {
    const float x = whole<OA>(g.a, g.a_stride, g.a_plane, row, k);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < g.e.n) s[e] = fmaf(x, whole<OB>(g.b, g.b_stride, g.b_plane, col + e, k), s[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (v[e] != v[e]) v[e] = s[e];
}

// ------------------------------------------------------------------------------------------
// Copies of an operand's stages into LDS, 1 KB a wave instruction, a few a wave and stage.
//   inner: 8 rows of 128 bytes; 16-byte chunk c of row r lies at c ^ (r / 2 % 8), so that a chunk of sixteen
//          rows, which a ds_read_b128 serves at once, lies in sixteen different parts of a 256-byte line (4 clocks
//          a read measured, 256 bytes a clock). Whole 128-byte lines: with 64-byte rows each line was fetched
//          twice, the L1 holding less than a stage, and the product ran at two thirds of its rate;
//   outer: 4 rows of k by 128 columns, in the swizzled layout of the transpose reads.
// Rows and columns past the operand, k past the sum and stages past the range are copied as zeros: their
// offsets lie past the buffer's end.
constexpr uint32_t kNowhere = 0x80000000u, kBuffer = 0x7fffffffu;
template <bool OUTER, int WAVES, int COUNT>
struct Copy {
  const char* base;  // of the tile
  int64_t step;      // bytes from one stage to the next
  int64_t plane;
  uint32_t off[COUNT], tail[COUNT];  // of this lane's 16 bytes, and kNowhere where they lie past the sum in its last stage

  // Tile from row (or column) `first` of `rows`; `k` elements of `size` bytes in the sum, whose last stage is `last`.
  __device__ __forceinline__ void init(const char* p, int64_t stride, int64_t plane_bytes, int64_t first, int64_t rows,
                                       int64_t k, int size, int64_t last, int w, int lane) {
    plane = plane_bytes;
    base = p + (OUTER ? first * 2 : first * stride);
    step = OUTER ? kStageRows * stride : kStageBytes;
#pragma unroll
    for (int h = 0; h < COUNT; ++h) {
      const int q = w + WAVES * h;
      if constexpr (OUTER) {
        const int row = 4 * (q & 15) + lane / 16, chunk = (lane % 16) ^ swz<16>(row), col = (q >> 4) * 128 + chunk * 8;
        off[h] = first + col < rows ? (uint32_t)row * (uint32_t)stride + (uint32_t)col * 2 : kNowhere;
        tail[h] = last * kStageRows + row < k ? 0 : kNowhere;
      } else {
        const int row = 8 * q + lane / 8, chunk = (lane % 8) ^ (row / 2 % 8);
        off[h] = first + row < rows ? (uint32_t)row * (uint32_t)stride + (uint32_t)chunk * 16 : kNowhere;
        tail[h] = last * kStageBytes + chunk * 16 < k * size ? 0 : kNowhere;
      }
    }
  }

  // Stage `t` of plane `p` to `dst`; `last` all ones: the sum's last stage; `none` kNowhere: zeros.
  __device__ __forceinline__ void issue(lds_char* dst, int64_t t, int p, uint32_t last, uint32_t none, int w) const {
    const rsrc_t r = make_rsrc(base + p * plane + t * step, kBuffer);
#pragma unroll
    for (int h = 0; h < COUNT; ++h) {
      const uint32_t o = off[h] | (tail[h] & last) | none;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + (w + WAVES * h) * 1024),
                                               16, (int)o, 0, 0, 0);
    }
  }
};

// LDS byte offsets of an operand's 32-row blocks for one wave: quarter c of a stage is 16 bf16 k.
template <bool OUTER, int BLOCKS>
struct Reads {
  uint32_t at[OUTER ? 2 * BLOCKS : 4];

  __device__ __forceinline__ void init(uint32_t region, int first, int lane) {  // first: row or column of the tile
    const int i = lane & 31, g = lane >> 5;
    if constexpr (OUTER) {  // k 8 g + 4 h .. of a quarter
      const int G = lane >> 4, t = lane & 15, e = t >> 2, q = t & 3;
#pragma unroll
      for (int m = 0; m < BLOCKS; ++m) {
        const int c0 = first + 32 * m;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 8 * g + 4 * h + e, chunk = 4 * ((c0 & 127) >> 5) + 2 * (G & 1) + (q >> 1);
          at[2 * m + h] = region + (uint32_t)(c0 >> 7) * 16384 + r * 256 + ((chunk ^ swz<16>(r)) << 4) + (q & 1) * 8;
        }
      }
    } else {
      const int r = first + i;
#pragma unroll
      for (int c = 0; c < 4; ++c) at[c] = region + r * 128 + (((2 * c + g) ^ (r / 2 % 8)) << 4);
    }
  }

  __device__ __forceinline__ u32x4 read(const lds_char* stage, int m, int c) const {
    if constexpr (OUTER) {
      const u32x2 lo = tr_read(stage + c * 4096, at[2 * m]), hi = tr_read(stage + c * 4096, at[2 * m + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return row_read(stage + m * 4096, at[c]);
    }
  }
};

// This wave's copies have landed and its LDS reads have returned, and so have every other wave's.
__device__ __forceinline__ void stage_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int kBand = 8;
constexpr int kStrip = 72;  // floats from one row of a strip to the next: its halves' rows fall in other banks

constexpr int threads_of(int bm, int bn) { return bm * bn > 192 * 128 ? 512 : 256; }

enum class Form { kBf16, kParts, kE4m3 };

// One BM x BN tile of c over one range of the sum. A wave has 32 MI x 64 of the tile.
template <bool OA, bool OB, Form FORM, int BM, int BN>
__global__ void __launch_bounds__((threads_of(BM, BN)), 2) product_kernel(ProductArgs g) {
  constexpr int WAVES = (threads_of(BM, BN)) / 64, NI = 2, WN = BN / 64, WM = WAVES / WN, MI = BM / WM / 32;
  constexpr int STAGE = (BM + BN) * kStageBytes;
  constexpr bool E4M3 = FORM == Form::kE4m3, PARTS = FORM == Form::kParts;
  constexpr bool PLAIN = OB;  // a gradient: no epilogue but the rounding
  constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;  // copies a wave and operand
  static_assert(CA * WAVES * 8 == BM && CB * WAVES * 8 == BN && WM * MI * 32 == BM, "whole copies and blocks");
  static_assert((!OA || BM % 128 == 0) && (!OB || BN % 128 == 0), "outer operands lie in 128 columns");
  // One array a stage: the compiler waits for the copies into the array that a read names, and for those alone.
  __shared__ __align__(256) char lds0[STAGE], lds1[STAGE];
  lds_char *const s0 = (lds_char*)lds0, *const s1 = (lds_char*)lds1;
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // Workgroups go to the 8 XCDs in turn: each takes a contiguous range of (range of the sum, tile).
  const int total = (int)gridDim.x, xcd = (int)blockIdx.x & 7, per = total >> 3, rem = total & 7;
  const int id = xcd * per + (xcd < rem ? xcd : rem) + ((int)blockIdx.x >> 3);
  const int tn = (int)((g.e.n + BN - 1) / BN), tiles = (int)((g.e.m + BM - 1) / BM) * tn;
  const int split = id / tiles, tile = id - split * tiles;
  // Bands of kBand rows of tiles, column by column: what runs at once on an XCD shares rows of both operands.
  const int tm = tiles / tn, band = tile / (kBand * tn), in = tile - band * (kBand * tn);
  const int high = tm - band * kBand < kBand ? tm - band * kBand : kBand;
  const int64_t i0 = (int64_t)(band * kBand + in % high) * BM, j0 = (int64_t)(in / high) * BN;
  const int size = E4M3 ? 1 : 2, per_stage = kStageBytes / size;
  const int64_t stages = (g.k + per_stage - 1) / per_stage, t0 = (int64_t)split * g.chunk;
  const int64_t t1 = t0 + g.chunk < stages ? t0 + g.chunk : stages;
  const int steps = (int)(t1 - t0) * (PARTS ? 6 : 1);

  Copy<OA, WAVES, CA> ca;
  Copy<OB, WAVES, CB> cb;
  ca.init(g.a, g.a_stride, g.a_plane, i0, g.e.m, g.k, size, stages - 1, w, lane);
  cb.init(g.b, g.b_stride, g.b_plane, j0, g.e.n, g.k, size, stages - 1, w, lane);
  int64_t at = t0;  // the stage copied next, and its term
  uint32_t pa = PARTS ? kPlaneA : 0, pb = PARTS ? kPlaneB : 0;
  int left = steps;
  const auto copy = [&](lds_char* stage) {
    const uint32_t none = left <= 0 ? kNowhere : 0, last = at == stages - 1 ? ~0u : 0;
    ca.issue(stage, at, pa & 3, last, none, w);
    cb.issue(stage + BM * kStageBytes, at, pb & 3, last, none, w);
    --left;
    if (++at == t1) {
      at = t0;
      pa >>= 4;
      pb >>= 4;
    }
  };

  const int wm = w / WN * (32 * MI), wn = w % WN * 64;  // this wave's part of the tile
  Reads<OA, MI> ra;
  Reads<OB, NI> rb;
  ra.init(0, wm, lane);
  rb.init(BM * kStageBytes, wn, lane);
  f32x16 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = zero16();
  constexpr int SETS = E4M3 ? 4 : 2;  // operands in registers: those multiplied and those being read
  u32x4 fa[SETS][MI], fb[SETS][NI];
  const auto read = [&](const lds_char* stage, int c, int set) {
#pragma unroll
    for (int m = 0; m < MI; ++m) fa[set][m] = ra.read(stage, m, c);
#pragma unroll
    for (int n = 0; n < NI; ++n) fb[set][n] = rb.read(stage, n, c);
  };
  const auto multiply = [&](int set) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n) acc[m][n] = mfma_bf16(fa[set][m], fb[set][n], acc[m][n]);
  };
  // The same for half a stage of e4m3: 64 k, the bytes of two quarters, scales 2^0.
  const auto multiply8 = [&](int set) {
    const auto join = [](const u32x4& x, const u32x4& y) {
      return i32x8{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    };
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(fa[set][m], fa[set + 1][m]),
                                                                    join(fb[set][n], fb[set + 1][n]), acc[m][n], 0, 0, 0,
                                                                    0x7f7f7f7f, 0, 0x7f7f7f7f);
  };
  // Column sums of a, in the workgroups of the first column tile: wave w takes 32 columns.
  const bool sums = OA && g.sums != nullptr && j0 == 0 && w < BM / 32;
  float sum = 0.f;
  Reads<OA, 1> rs;
  rs.init(0, 32 * (w < BM / 32 ? w : 0), lane);
  const auto add = [&](const lds_char* stage) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u32x4 v = rs.read(stage, 0, c);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u = v[k];
        sum += as_float(u << 16) + as_float(u & 0xffff0000u);
      }
    }
  };

  copy(s0);
  stage_barrier();
  copy(s1);
  read(s0, 0, 0);
  if constexpr (E4M3) read(s0, 1, 1);
  const auto step = [&](lds_char* now, lds_char* next) {
    if constexpr (E4M3) {
      read(now, 2, 2);
      read(now, 3, 3);
      multiply8(0);
    } else {
      read(now, 1, 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(0);
      if constexpr (OA) {
        if (sums) add(now);
      }
      read(now, 2, 0);
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
      read(now, 3, 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(0);
    }
    // Every wave has read all of this stage, whose place the stage after the next takes, and the next has landed.
    stage_barrier();
    copy(now);
    read(next, 0, 0);
    if constexpr (E4M3) {
      read(next, 1, 1);
      multiply8(2);
    } else {
      __builtin_amdgcn_sched_barrier(0);
      multiply(1);
    }
  };
  for (int t = 0; t < steps; t += 2) {  // a stage past the last is zeros
    step(s0, s1);
    step(s1, s0);
  }
  wait_vmem();  // no copy outlives the stages
  __syncthreads();

  if constexpr (OA) {
    if (sums) {
      sum += __shfl_xor(sum, 32);
      if (lane < 32 && i0 + 32 * w + lane < g.e.m) g.sums[(int64_t)split * g.e.m + i0 + 32 * w + lane] = sum;
    }
  }
  // Through LDS, 32 rows of the wave's part at a time, to rows of eight columns a lane.
  constexpr int PER = WAVES / 2;  // waves that share a stage's array
  auto* const strip = (__attribute__((address_space(3))) float*)((w < PER ? s0 : s1) + (w % PER) * (32 * kStrip * 4));
  const int j = lane & 31, half = lane >> 5;
  const auto to_strip = [&](int m) {
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) strip[(8 * (r >> 2) + 4 * half + (r & 3)) * kStrip + 32 * n + j] = acc[m][n][r];
  };
  const int sub = lane >> 3, at_col = wn + 8 * (lane & 7);  // this lane's row of eight and its columns of the tile
  const int64_t col = j0 + at_col;
  const auto from_strip = [&](int p, float(&v)[8]) {
    const auto* q = (const __attribute__((address_space(3))) f32x4*)(strip + (8 * p + sub) * kStrip + 8 * (lane & 7));
    const f32x4 lo = q[0], hi = q[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = lo[k], y = hi[k];
      v[k] = x;
      v[4 + k] = y;
    }
  };
  const EpilogueArgs& e = g.e;
  const int rows = (int)(e.m - i0 < BM ? e.m - i0 : BM);  // of the tile
  if (g.part || (e.vec && !PARTS)) {
    // Offsets in the tile, past the buffers' ends for rows and columns outside.
    const bool f32 = g.part || (E4M3 && e.dtype == FWN_F32);
    const int64_t width = g.part ? g.part_row : e.n;
    const uint32_t shift = f32 ? 2 : 1;
    char* const to = g.part ? (char*)(g.part + (int64_t)split * e.m * g.part_row) : (char*)e.out;
    const rsrc_t ro = make_rsrc(to + ((i0 * width + j0) << shift), kBuffer);
    const rsrc_t rp = make_rsrc((char*)e.pre + ((i0 * width + j0) << shift), kBuffer);
    const rsrc_t rr = make_rsrc((const char*)e.residual + ((i0 * e.r_row + j0) << shift), kBuffer);
    const bool scaled = E4M3 && !g.part, pre = !PLAIN && !g.part && e.pre,
               residual = !PLAIN && !g.part && e.residual;
    const uint32_t nowhere = col < e.n ? 0 : kNowhere;
    Columns c;
    if (!PLAIN && !g.part) c.load(e, col);
    const auto load = [&](rsrc_t r, uint32_t o, float(&f)[8]) {
      const u32x4 lo = bload16(r, o), hi = f32 ? bload16(r, o + 16) : lo;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t x = lo[k], y = hi[k];
        if (f32) {
          f[k] = as_float(x);
          f[4 + k] = as_float(y);
        } else {
          f[2 * k] = as_float(x << 16);
          f[2 * k + 1] = as_float(x & 0xffff0000u);
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
    with_activation<PLAIN>(g.part ? FWN_ACT_NONE : e.activation, [&](auto act) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        to_strip(m);
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const int row = wm + 32 * m + 8 * p + sub;
          const uint32_t out = (row < rows ? 0 : kNowhere) | nowhere;
          const uint32_t o = out | (((uint32_t)row * (uint32_t)width + (uint32_t)at_col) << shift);
          float v[8], r[8];
          if (residual) load(rr, out | (((uint32_t)row * (uint32_t)e.r_row + (uint32_t)at_col) << shift), r);
          from_strip(p, v);
          if (scaled) {
            const float s = row < rows ? e.a_scale[i0 + row] : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= s * c.scale[k];
          }
          if (!PLAIN && !g.part) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] += c.bias[k];
            if (pre) store(rp, o, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = activate<decltype(act)::kind>(v[k]);
            if (residual) {
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] += r[k];
            }
          }
          store(ro, o, v);
        }
        __builtin_amdgcn_wave_barrier();
      }
    });
    return;
  }
  // Outputs that are not whole aligned eights, and those of parts, which may need their wholes.
  Columns c;
  c.load(e, col);
  with_activation<PLAIN>(e.activation, [&](auto act) {
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      to_strip(m);
      __builtin_amdgcn_wave_barrier();
#pragma unroll 1
      for (int p = 0; p < 4; ++p) {
        const int row = wm + 32 * m + 8 * p + sub;
        if (row >= rows || col >= e.n) continue;
        float v[8];
        from_strip(p, v);
        if constexpr (PARTS) mend<OA, OB>(g, i0 + row, col, v);
        finish<decltype(act)::kind>(e, i0 + row, col, v, c);
      }
      __builtin_amdgcn_wave_barrier();
    }
  });
}

// The partial products added in the order of the splits, then the epilogue: eight columns a thread.
template <bool OA, bool OB, Form FORM>
__global__ void __launch_bounds__(256) join_kernel(ProductArgs g) {
  const int64_t across = g.part_row / 8, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / across, col = (id - row * across) * 8;
  if (row >= g.e.m) return;
  float v[8] = {};
#pragma unroll 4
  for (int s = 0; s < g.splits; ++s) {
    float p[8];
    load8(g.part, ((int64_t)s * g.e.m + row) * g.part_row + col, FWN_F32, p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] += p[k];
  }
  Columns c;
  c.load(g.e, col);
  if constexpr (FORM == Form::kParts) mend<OA, OB>(g, row, col, v);
  with_activation<OB>(g.e.activation, [&](auto act) { finish<decltype(act)::kind>(g.e, row, col, v, c); });
}

template <bool OA, bool OB, Form FORM, int BM, int BN>
hipError_t launch_tile(const ProductArgs& g, hipStream_t stream) {
  const int64_t tiles = ((g.e.m + BM - 1) / BM) * ((g.e.n + BN - 1) / BN);
  hipLaunchKernelGGL((product_kernel<OA, OB, FORM, BM, BN>), dim3((unsigned)(tiles * g.splits)), dim3((threads_of(BM, BN))), 0, stream, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !g.part) return e;
  const int64_t threads = g.e.m * (g.part_row / 8);
  hipLaunchKernelGGL((join_kernel<OA, OB, FORM>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, g);
  return hipGetLastError();
}

template <bool OA, bool OB, Form FORM>
hipError_t launch_operands(int tile, const ProductArgs& g, hipStream_t stream) {
  if (tile == 0) return launch_tile<OA, OB, FORM, 256, 256>(g, stream);
  if constexpr (!OA) {
    if (tile == 1) return launch_tile<OA, OB, FORM, 192, 128>(g, stream);
  }
  return launch_tile<OA, OB, FORM, 128, 128>(g, stream);
}

template <Form FORM>
hipError_t launch_kind(Operands how, int tile, const ProductArgs& g, hipStream_t stream) {
  if (how == Operands::kInnerInner) return launch_operands<false, false, FORM>(tile, g, stream);
  if (how == Operands::kInnerOuter) return launch_operands<false, true, FORM>(tile, g, stream);
  return launch_operands<true, true, FORM>(tile, g, stream);
}

// ------------------------------------------------------------------------------------------
// Layouts. A thread forms 16 bytes of each plane of a row.

// Eight values of a row as the product kernel reads them: rounded to bf16, or three parts of 8 bits each.
__device__ __forceinline__ void store_parts(char* dst, int64_t plane, bool parts, const float (&f)[8]) {
  if (!parts) {
    *(u32x4*)dst = pack8(f);
    return;
  }
  u32x4 hi, mid, lo;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t h[2], m[2], l[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float v = f[2 * k + e];
      const uint32_t u = as_bits(v);
      if ((u & 0x7f800000u) == 0x7f800000u) {  // an infinity, or a NaN whose bits may all lie in the cut part
        h[e] = u << 9 ? 0x7fc0u : u >> 16;
        m[e] = l[e] = 0;
        continue;
      }
      const float r1 = v - as_float(u & 0xffff0000u);
      const uint32_t u1 = as_bits(r1);
      const float r2 = r1 - as_float(u1 & 0xffff0000u);
      h[e] = u >> 16;
      m[e] = u1 >> 16;
      l[e] = as_bits(r2) >> 16;
    }
    hi[k] = h[0] | h[1] << 16;
    mid[k] = m[0] | m[1] << 16;
    lo[k] = l[0] | l[1] << 16;
  }
  *(u32x4*)dst = hi;
  *(u32x4*)(dst + plane) = mid;
  *(u32x4*)(dst + 2 * plane) = lo;
}

__global__ void __launch_bounds__(256) layout_kernel(LayoutArgs a) {
  const int per = a.op == kOpE4m3 ? 16 : 8;  // columns a thread
  const int64_t across = (a.cols + per - 1) / per, id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / across, col = (id - row * across) * per;
  if (row >= a.rows) return;
  char* dst = a.dst + row * a.dst_stride + (id - row * across) * 16;
  if (a.op == kOpE4m3) {
    const uint8_t* p = (const uint8_t*)a.src + row * a.stride + col;
    uint32_t d[4] = {};
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (col + k < a.cols) d[k / 4] |= (uint32_t)p[k] << 8 * (k % 4);
    *(u32x4*)dst = u32x4{d[0], d[1], d[2], d[3]};
    return;
  }
  float f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    f[k] = col + k < a.cols ? load_one(a.src, row * a.stride + col + k, a.op == kOpF32 ? FWN_F32 : FWN_BF16) : 0.f;
  store_parts(dst, a.dst_plane, a.op == kOpF32, f);
}

// 256 columns by `chunk` rows a workgroup, eight columns of every eighth row a thread.
template <int KIND>
__global__ void __launch_bounds__(256) slope_kernel(SlopeArgs a) {
  __shared__ float red[8][256];
  const int across = (a.outs + 255) / 256, block = (int)blockIdx.x / across;
  const int lane = (int)threadIdx.x & 31, own = (int)threadIdx.x >> 5;
  const int col = ((int)blockIdx.x - block * across) * 256 + 8 * lane;
  const int64_t r0 = (int64_t)block * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  const bool vec = a.outs % 8 == 0 && (((uintptr_t)a.g | (uintptr_t)a.pre) & 15) == 0;
  float sum[8] = {};
  if (col < a.outs) {
    for (int64_t r = r0 + own; r < r1; r += 8) {
      const int64_t at = r * a.outs + col;
      float dz[8], z[8];
      if (vec) {
        load8(a.g, at, a.dtype, dz);
        if (KIND != FWN_ACT_NONE) load8(a.pre, at, a.dtype, z);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool in = col + k < a.outs;
          dz[k] = in ? load_one(a.g, at + k, a.dtype) : 0.f;
          z[k] = in && KIND != FWN_ACT_NONE ? load_one(a.pre, at + k, a.dtype) : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if constexpr (KIND != FWN_ACT_NONE) dz[k] *= slope<KIND>(z[k]);
        sum[k] += dz[k];
      }
      if (a.dz) store_parts(a.dz + r * a.dz_stride + (int64_t)col * 2, a.dz_plane, a.dtype == FWN_F32, dz);
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) red[own][8 * lane + k] = sum[k];
  __syncthreads();
  const int c = (int)threadIdx.x, to = col - 8 * lane + c;
  if (to >= a.outs) return;
  float s = red[0][c];
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][c];
  a.part[(int64_t)block * a.outs + to] = s;
}

constexpr int kGroups = 16;  // shares of the partial rows that a workgroup adds in parallel

__global__ void __launch_bounds__(64 * kGroups) column_sums_kernel(const float* part, int64_t count, int64_t n, void* out,
                                                                   int dtype) {
  __shared__ float red[kGroups][64];
  const int lane = threadIdx.x & 63, grp = (int)threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int64_t b = grp; b < count; b += kGroups) s += part[b * n + c];
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || c >= n) return;
#pragma unroll
  for (int k = 1; k < kGroups; ++k) s += red[k][lane];
  store_one(out, c, dtype, s);
}

}  // namespace

hipError_t launch_product(Operands how, int32_t op, int tile, const ProductArgs& a, hipStream_t stream) {
  if (op == kOpE4m3) return launch_operands<false, false, Form::kE4m3>(tile, a, stream);
  return op == kOpF32 ? launch_kind<Form::kParts>(how, tile, a, stream) : launch_kind<Form::kBf16>(how, tile, a, stream);
}

hipError_t launch_layout(const LayoutArgs& a, hipStream_t stream) {
  const int per = a.op == kOpE4m3 ? 16 : 8;
  const int64_t threads = a.rows * ((a.cols + per - 1) / per);
  if (threads == 0) return hipSuccess;
  hipLaunchKernelGGL(layout_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_slope(const SlopeArgs& a, hipStream_t stream) {
  const unsigned across = (unsigned)(a.outs + 255) / 256;
  const dim3 grid(across * (unsigned)a.blocks), block(256);
  switch (a.activation) {
    case FWN_ACT_RELU: hipLaunchKernelGGL(slope_kernel<FWN_ACT_RELU>, grid, block, 0, stream, a); break;
    case FWN_ACT_GELU: hipLaunchKernelGGL(slope_kernel<FWN_ACT_GELU>, grid, block, 0, stream, a); break;
    case FWN_ACT_GELU_TANH: hipLaunchKernelGGL(slope_kernel<FWN_ACT_GELU_TANH>, grid, block, 0, stream, a); break;
    case FWN_ACT_SILU: hipLaunchKernelGGL(slope_kernel<FWN_ACT_SILU>, grid, block, 0, stream, a); break;
    default: hipLaunchKernelGGL(slope_kernel<FWN_ACT_NONE>, grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_column_sums(const float* part, int64_t count, int64_t n, void* out, int dtype, hipStream_t stream) {
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((n + 63) / 64)), dim3(64 * kGroups), 0, stream, part, count, n,
                     out, dtype);
  return hipGetLastError();
}

}  // namespace fwn
