// Linear layers of 4-bit weights with a scale for each group of 32 inputs (gfx950): out = act(x w^T + b) + residual with
// w = value(code) 2^(e - 127), the codes OCP e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) and e the group's
// OCP e8m0 scale. Such a weight is exact in bfloat16, so that products of widened weights are exact and added in float32.
//
// Few rows of x: bound by the weight's trip from memory and the waits for the rows' from L2, one pass over the weight with no
// partial products to join. A workgroup has 16 to 64 outputs, its waves share the sum, 128 inputs at a time: a lane's 16 bytes of codes are one
// group of one weight row, exchanged between the four lanes of a row so that each has eight inputs of each group and widened in
// registers by the groups' scales to the MFMAs' operands; the waves' sums meet in LDS. From a captured graph one row of
// 4,096 -> 4,096 takes 5.5 to 5.9 us, of 8,192 -> 8,192 12.4 to 14 (2.5 to 2.9 TB/s; as bf16 33 to 35), 24 rows of 5,120 -> 8,192 16 to 17;
// with a profiler 7.0 and 18 for the first and the last.
// More rows of bf16: tiles that read the codes (q4_tile_kernel); float32, and rows enough to pay for it: the weight is widened
// into the workspace for the kernels of linear_act.
#include "linear_act_device.h"
#include "linear_act_stage.h"
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
    scales = make_rsrc(a.scales + first * a.scale_row, kBuffer);
    const bool in = first + i < a.p.e.n;
    off = in ? ((uint32_t)i * groups + g) * 16 : kNowhere;
    soff = in ? (uint32_t)i * (uint32_t)a.scale_row + g : kNowhere;
  }
  __device__ __forceinline__ u32x4 load(uint32_t line, int g) const {
    return bload16(codes, (off + line * 64) | (line * 4 + g < groups ? 0 : kNowhere));
  }
  __device__ __forceinline__ uint32_t scale(uint32_t line, int g) const {
    return __builtin_amdgcn_raw_buffer_load_b8(scales, (int)((soff + line * 4) | (line * 4 + g < groups ? 0 : kNowhere)), 0, 0);
  }
};

// The lane's part of x in 16 rows and a line: the inputs 32 t + 8 g .. + 7 of it for t = 0 to 3, a piece of 16 bytes each in bf16
// and two in float32, so that the four lanes of a row read 64 or 128 bytes side by side. (The inputs 32 g .. of the lane's own group of
// codes, which need no exchange of codes between lanes, lie in a line of their own: float32, 24 rows of 4,096 -> 4,096: 35 us, 24 so.)
template <bool F32>
struct Inputs {
  static constexpr int PER = F32 ? 2 : 1, PIECES = 4 * PER, LINE_BYTES = LINE * (F32 ? 4 : 2);
  rsrc_t r;
  uint32_t off, at0, bytes;

  __device__ __forceinline__ void init(const ProductArgs& a, int64_t first, int lane) {
    const int i = lane & 15, g = lane >> 4;
    r = make_rsrc(a.a + first * a.a_stride, kBuffer);
    at0 = g * PER * 16;
    off = first + i < a.e.m ? (uint32_t)i * (uint32_t)a.a_stride : kNowhere;
    bytes = (uint32_t)a.k * (F32 ? 4 : 2);
  }
  // Zeros past the row. A float32 row may end inside a piece, and is not read past its end.
  __device__ __forceinline__ void load(uint32_t line, int, u32x4 (&v)[PIECES]) const {
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const uint32_t at = line * LINE_BYTES + at0 + p / PER * (64 * PER) + p % PER * 16;
      if (!F32 || bytes % 16 == 0) {
        v[p] = bload16(r, (off + at) | (at < bytes ? 0 : kNowhere));
      } else if ((line + 1) * LINE_BYTES <= bytes) {
        v[p] = bload16(r, off + at);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[p][e] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)((off + at + 4 * e) | (at + 4 * e < bytes ? 0 : kNowhere)), 0, 0);
      }
    }
  }
};

// Rows of 16 lanes of the arguments exchanged: see transpose.
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {  // a's upper half with b's lower half
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0], b = r[1];
}
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {  // a's odd rows with b's even rows
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  a = r[0], b = r[1];
}
// Word t of row g to word g of row t.
__device__ __forceinline__ void transpose(uint32_t (&d)[4]) {
  swap32(d[0], d[2]);
  swap32(d[1], d[3]);
  swap16(d[0], d[1]);
  swap16(d[2], d[3]);
}
// Row t's value, in every row, to d[t].
__device__ __forceinline__ void broadcast(uint32_t v, uint32_t (&d)[4]) {
  uint32_t lo = v, hi = v;
  swap32(lo, hi);
  d[0] = d[1] = lo;
  swap16(d[0], d[1]);
  d[2] = d[3] = hi;
  swap16(d[2], d[3]);
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
  u32x4 vw[AHEAD][COLS], vx[AHEAD][GROUPS][Inputs<F32>::PIECES];
  uint32_t vs[AHEAD][COLS];
  const auto ask = [&](int s, uint32_t line) {
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
      vw[s][n] = weight[n].load(line, g);
      vs[s][n] = weight[n].scale(line, g);
    }
#pragma unroll
    for (int m = 0; m < GROUPS; ++m) x[m].load(line, g, vx[s][m]);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto multiply = [&](int s, uint32_t line) {
    // The codes past the inputs, in the last line.
    const int left = (int)((int64_t)a.p.k - (int64_t)(line * 4 + g) * GROUP);
#pragma unroll
    for (int n = 0; n < COLS; ++n) {
      uint32_t codes[4] = {vw[s][n][0], vw[s][n][1], vw[s][n][2], vw[s][n][3]};
      if (line + 1 >= lines) {
#pragma unroll
        for (int t = 0; t < 4; ++t) codes[t] = first_codes(codes[t], left - 8 * t);
      }
      uint32_t scales[4];
      transpose(codes);
      broadcast(vs[s][n], scales);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float scale = scale_of(scales[t]);
        if constexpr (F32) {
          const f32x2 v[4] = {widen_f32<0>(codes[t], scale), widen_f32<1>(codes[t], scale), widen_f32<2>(codes[t], scale),
                              widen_f32<3>(codes[t], scale)};
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int m = 0; m < GROUPS; ++m) {
              const uint32_t u = vx[s][m][2 * t + i / 4][i % 4];
              acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i / 2][i % 2], as_float(u), acc[m][n], 0, 0, 0);
            }
        } else {
          const bf16x8 v = __builtin_bit_cast(bf16x8, widen8(codes[t], scale));
#pragma unroll
          for (int m = 0; m < GROUPS; ++m)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, vx[s][m][t]), acc[m][n], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // Lines w, w + WAVES, ... of the rows (past the rows' end: zeros).
#pragma unroll
  for (int s = 0; s < AHEAD; ++s) ask(s, w + WAVES * s);
  for (uint32_t l0 = w; l0 < lines; l0 += WAVES * AHEAD) {
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) {
      const uint32_t line = l0 + WAVES * s;
      multiply(s, line);
      ask(s, line + WAVES * AHEAD);
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

constexpr int kRows = 64, kSpan = kQ4Span;  // of x in a tile, and inputs of a step of a tile: 64 bytes of a row's codes

// Copies of a tile's codes into LDS: 16 rows of 64 bytes a wave instruction, 64 rows a wave; 16-byte chunk c of row r lies at
// c ^ (r / 4 % 4), so that sixteen rows' chunks lie in sixteen parts of a 256-byte line.
struct CopyCodes {
  const char* base;
  uint32_t off[4], group;

  __device__ __forceinline__ void init(const uint8_t* codes, int64_t groups, int64_t first, int64_t rows, int lane) {
    base = (const char*)codes + first * groups * 16;
    group = (uint32_t)(lane % 4) ^ (uint32_t)(lane / 16 % 4);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = 16 * q + lane / 4;
      off[q] = first + row < rows ? ((uint32_t)row * (uint32_t)groups + group) * 16 : kNowhere;
    }
  }
  __device__ __forceinline__ void issue(lds_char* dst, int64_t t, uint32_t groups, uint32_t none) const {
    const rsrc_t r = make_rsrc(base + t * 64, kBuffer);
    const uint32_t past = none | ((uint32_t)t * 4 + group < groups ? 0 : kNowhere);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + q * 1024), 16, (int)(off[q] | past), 0,
                                               0, 0);
  }
};

// A tile of 64 rows by 64 WAVES outputs over one range of the sum, for bf16. Both operands go through STAGES LDS stages of 128 inputs
// by direct copies, the weight as codes; a wave has 64 outputs of its own, so that each code is widened once a tile. All stages
// but the one that is multiplied are on their way.
// Bound by the copies: 34 KB a stage of four waves, 0.75 us alone and 0.85 to 1.0 with the products (0.43 of the matrix units)
// where every CU has a workgroup. 512 rows of 4,096 -> 8,192 from a captured graph: 38 to 40 us (860 to 900 TFLOP/s), with GELU and a
// residual 41 to 47 (48 with a profiler); with the weight widened first 19 and 43. Beside 36 us on the machine of these
// comparisons: codes from memory straight to the registers that widen them took 51 us (a lane's 16 bytes lie in another line
// than its neighbours'), two stages of 256 inputs 37, the next stage's first reads before the last products of a stage 39.
template <int WAVES, int STAGES>
__global__ void __launch_bounds__(64 * WAVES, 1) q4_tile_kernel(Q4Args a) {
  constexpr int SUBS = kSpan * 2 / kStageBytes, BN = 64 * WAVES, ROWS_STAGE = kRows * kSpan * 2, STAGE = ROWS_STAGE + BN * 64;
  constexpr int kLoads = SUBS * (kRows / 8 / WAVES) + 4 + 1;  // of a span
  static_assert(SUBS == 2, "a half of the wave reads a part of 64 inputs");
  __shared__ __align__(256) char lds0[STAGE], lds1[STAGE], lds2[STAGE], lds3[STAGES > 3 ? STAGE : 256];
  const auto stage = [&](int s) -> lds_char* {
    return s == 0 ? (lds_char*)lds0 : s == 1 ? (lds_char*)lds1 : s == 2 ? (lds_char*)lds2 : (lds_char*)lds3;
  };
  const ProductArgs& p = a.p;
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
  const Work k = work_of<kRows, BN>(p.e);
  const int64_t stages = (p.k + kStageRows - 1) / kStageRows, spans = (p.k + kSpan - 1) / kSpan, t0 = (int64_t)k.split * p.chunk;
  const int64_t t1 = t0 + p.chunk < spans ? t0 + p.chunk : spans, n0 = k.j0 + 64 * w;
  const uint32_t groups = (uint32_t)a.groups;

  Copy<false, WAVES, kRows / 8 / WAVES> cx;
  cx.init(p.a, p.a_stride, k.i0, p.e.m, p.k, 2, stages - 1, w, lane);
  CopyCodes cw;
  cw.init(a.codes, groups, n0, p.e.n, lane);
  // The four scales of a span of row n0 + lane.
  const rsrc_t rs = make_rsrc(a.scales + n0 * a.scale_row, kBuffer);
  const uint32_t soff = n0 + lane < p.e.n ? (uint32_t)lane * (uint32_t)a.scale_row : kNowhere;
  uint32_t scales[STAGES];
  const auto ask = [&](int s, int64_t t) {
    const uint32_t none = t < t1 ? 0 : kNowhere;
#pragma unroll
    for (int u = 0; u < SUBS; ++u) {
      const int64_t at = t * SUBS + u;
      cx.issue(stage(s) + u * (kRows * kStageBytes), at, at == stages - 1 ? ~0u : 0, at < stages ? none : kNowhere, w);
    }
    cw.issue(stage(s) + ROWS_STAGE + w * 4096, t, groups, none);
    scales[s] = __builtin_amdgcn_raw_buffer_load_b32(rs, (int)((soff + (uint32_t)t * 4) | none), 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // The oldest span asked for has landed, and every wave has read the one before it. The wait counts this wave's loads: kLoads of
  // each span, in the order of ask (whose last line keeps it) and nothing else.
  const auto next_barrier = [&] {
    constexpr int kAhead = kLoads * (STAGES - 2);
    static_assert(kAhead < 64, "the wait's count");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((kAhead & 15) | 0x70 | (kAhead >> 4) << 14);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  uint32_t at[8], wat[2];  // of chunk c of row i of x in a stage; of the codes' chunk 2 h + s of row 64 w + i
#pragma unroll
  for (int c = 0; c < 8; ++c) at[c] = (uint32_t)h * (kRows * kStageBytes) + i * kStageBytes + ((c ^ (i / 2 % 8)) << 4);
#pragma unroll
  for (int s = 0; s < 2; ++s) wat[s] = ROWS_STAGE + w * 4096 + i * 64 + (((2 * h + s) ^ (i / 4 % 4)) << 4);
  f32x16 acc[2][2];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[m][n] = zero16();
  // Eight steps of 16 inputs of each half; the operands of one are read and widened while those of the one before are multiplied.
  const auto multiply = [&](const lds_char* from, uint32_t scale, int64_t t) {
    u32x4 x[2][2], f[2][2], codes[2][2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < 2; ++n) codes[s][n] = row_read(from + n * 2048, wat[s]);
    uint32_t e[2] = {scale, scale};  // of rows i and 32 + i, this half's two groups lowest
    swap32(e[0], e[1]);
#pragma unroll
    for (int n = 0; n < 2; ++n) e[n] >>= 16 * h;
    if (t + 1 >= spans) {  // the codes past the inputs
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int left = (int)(p.k - (t * 4 + 2 * h + s) * GROUP);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) codes[s][n][c] = first_codes(codes[s][n][c], left - 8 * c);
      }
    }
    const auto operands = [&](int step) {
      const int s = step / 4, c = step % 4, set = step % 2;
#pragma unroll
      for (int m = 0; m < 2; ++m) x[set][m] = row_read(from + m * (32 * kStageBytes), at[step]);
#pragma unroll
      for (int n = 0; n < 2; ++n) f[set][n] = widen8(codes[s][n][c], scale_of(e[n] >> 8 * s & 0xff));
    };
    operands(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int step = 0; step < 8; ++step) {
      if (step < 7) operands(step + 1);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[m][n] = mfma_bf16(f[step % 2][n], x[step % 2][m], acc[m][n]);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // the reads, then a product with every three conversions
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) ask(s, t0 + s);
  for (int64_t t = t0; t < t1; t += STAGES) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      if (t + s >= t1) break;
      next_barrier();
      ask((s + STAGES - 1) % STAGES, t + s + STAGES - 1);
      multiply(stage(s), scales[s], t + s);
    }
  }
  Bf16Terms<2, false, false> terms;
  if (bf16_rows<false>(p)) terms.load(p.e, k, (int)(p.e.m - k.i0 < kRows ? p.e.m - k.i0 : kRows), 0, 64 * w, lane);
  wait_vmem();  // no copy outlives the stages
  __syncthreads();
  write_tile<kRows, 2, false, false, false>(p, k, acc, (strip_ptr)(stage(w / 2) + w % 2 * kStripBytes), 0, 64 * w, lane, terms,
                                            MendNothing());
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

// 16, 32 or 64 outputs a workgroup: many where there are workgroups enough, as each reads all rows of x. us with 16, 32 and 64, bf16:
// one row of 4,096 -> 4,096 5.8, 7.6 and 11.9, of 8,192 -> 8,192 14.4, 12.4 and 19.9, of 4,096 -> 16,384 15.7, 13.1 and 12.4; 24 rows of
// 4,096 -> 4,096 11.0, 12.9 and 16.9, of 5,120 -> 8,192 24.3, 16.2 and 20.3, 20 of 1,024 -> 16,384 16.1, 10.9 and 7.4. float32 products
// take their time, so that few lines on their way suffice, and long rows take 16 waves: 24 rows of 1,283 -> 2,051 11.4 with 8
// and 14.6 with 16, of 4,096 -> 4,096 24.1 and 20.6.
hipError_t launch_bf16(const Q4Args& a, hipStream_t stream) {
  const bool few = a.p.e.m <= 16;
  if (a.p.e.n > 48 * 256) return few ? launch<false, 1, 4, 8, 2>(a, stream) : launch<false, 2, 4, 8, 1>(a, stream);
  if (a.p.e.n > 16 * 256) return few ? launch<false, 1, 2, 8, 2>(a, stream) : launch<false, 2, 2, 16, 1>(a, stream);
  if (few) return a.p.k > 16 * LINE ? launch<false, 1, 1, 8, 2>(a, stream) : launch<false, 1, 1, 16, 1>(a, stream);
  return launch<false, 2, 1, 8, 2>(a, stream);
}

hipError_t launch_f32(const Q4Args& a, hipStream_t stream) {
  const bool few = a.p.e.m <= 16;
  if (a.p.e.n > 16 * 256) return few ? launch<true, 1, 2, 16, 1>(a, stream) : launch<true, 2, 2, 16, 1>(a, stream);
  if (few) return launch<true, 1, 1, 8, 1>(a, stream);
  return a.p.k > 16 * LINE ? launch<true, 2, 1, 16, 1>(a, stream) : launch<true, 2, 1, 8, 1>(a, stream);
}

}  // namespace

hipError_t launch_q4_rows(bool f32, const Q4Args& a, hipStream_t stream) {
  return f32 ? launch_f32(a, stream) : launch_bf16(a, stream);
}

hipError_t launch_q4_tiles(int waves, const Q4Args& a, hipStream_t stream) {
  const int64_t tiles = ((a.p.e.m + kRows - 1) / kRows) * ((a.p.e.n + 64 * waves - 1) / (64 * waves));
  const dim3 grid((unsigned)(tiles * a.p.splits));
  if (waves == 4)
    hipLaunchKernelGGL(((q4_tile_kernel<4, 4>)), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(((q4_tile_kernel<2, 3>)), grid, dim3(128), 0, stream, a);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !a.p.part) return e;
  return launch_join(a.p, stream);
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
