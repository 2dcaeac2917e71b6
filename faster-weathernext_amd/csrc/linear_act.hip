// Matrix products with bias, activation and residual in their epilogue, and their gradients (gfx950):
//
//   z = x w^T + b,  out = act(z) + residual;   dz = g act'(z),  gx = dz w,  gw = dz^T x,  gb = sum of dz
//
// One kernel for the three products c[i, j] = sum over k of a(i, k) b(j, k) of bf16 or e4m3 operands: one whose rows
// are contiguous in k ("inner": x, w and dz in the first two) is read from LDS row by row, one whose rows are k
// ("outer": w in gx, dz and x in gw) by transpose reads, and both arrive as the same MFMA operands.
//
// Bound by the matrix units, and for short sums by what is not overlapped with them: 8,192 x 8,192 x 8,192 runs at 1,110 to
// 1,260 TFLOP/s in bf16 and 2,100 in e4m3; 40,962 x 768 -> 3,072 takes 204 us (950), 229 with bias and GELU, 167 in e4m3
// with both, of which the main loop has 160 and 92. One workgroup a CU (its two stages are 128 KB of LDS, its sums half
// of the registers): 8 waves of 128 x 64 outputs, so that a byte of a in LDS is read four times and one of b twice.
#include "linear_act_device.h"

namespace fwn {
namespace {

// ------------------------------------------------------------------------------------------
// Copies of an operand's stages into LDS, 1 KB a wave instruction, a few a wave and stage.
//   inner: 8 rows of 128 bytes; 16-byte chunk c of row r lies at c ^ (r / 2 % 8), so that a chunk of sixteen
//          rows, which a ds_read_b128 serves at once, lies in sixteen different parts of a 256-byte line (4 clocks
//          a read measured, 256 bytes a clock). Whole 128-byte lines: with 64-byte rows each line was fetched
//          twice, the L1 holding less than a stage, and the product ran at two thirds of its rate;
//   outer: 4 rows of k by 128 columns, in the swizzled layout of the transpose reads.
// Rows and columns past the operand, k past the sum and stages past the range are copied as zeros: their
// offsets lie past the buffer's end.
template <bool OUTER, int WAVES, int COUNT>
struct Copy {
  const char* base;  // of the tile
  int64_t step;      // bytes from one stage to the next
  uint32_t off[COUNT], tail[COUNT];  // of this lane's 16 bytes, and kNowhere where they lie past the sum in its last stage

  // Tile from row (or column) `first` of `rows`; `k` elements of `size` bytes in the sum, whose last stage is `last`.
  __device__ __forceinline__ void init(const char* p, int64_t stride, int64_t first, int64_t rows,
                                       int64_t k, int size, int64_t last, int w, int lane) {
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

  // Stage `t` to `dst`; `last` all ones: the sum's last stage; `none` kNowhere: zeros.
  __device__ __forceinline__ void issue(lds_char* dst, int64_t t, uint32_t last, uint32_t none, int w) const {
    const rsrc_t r = make_rsrc(base + t * step, kBuffer);
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

constexpr int threads_of(int bm) { return 2 * bm; }

// How a product is formed. The e4m3 matrix instructions do not add in float32: they take eight products at a time as
// multiples of 2^-13 of the largest one's power of two, cut off, and only the sums of eight are added in float32. Random sums
// are off by 1.4e-5 of the rows' norms (RMS; float32's order of magnitude is 1e-8), no sum by more than 2^-10 of its
// products' magnitudes. That is a hundredth of a bf16 output's own rounding, and these have kE4m3 for its rate; float32
// outputs are formed of the codes widened to bf16, exactly, and added in float32. us with kE4m3 and kWidened: 40,962 x 768 ->
// 3,072 182 and 240 (bf16 outputs; float32 ones 220 and 255), 8,192 x 8,192 -> 8,192 440 and 726.
enum class Form { kBf16, kE4m3, kWidened };

// One BM x BN tile of c over one range of the sum. A wave has 32 MI x 64 of the tile.
template <bool OA, bool OB, Form FORM, int BM, int BN>
__global__ void __launch_bounds__((threads_of(BM)), 2) product_kernel(ProductArgs g) {
  constexpr bool E4M3 = FORM == Form::kE4m3, CODES = FORM != Form::kBf16;
  constexpr int WAVES = (threads_of(BM)) / 64, NI = 2, WN = BN / 64, WM = WAVES / WN, MI = BM / WM / 32;
  constexpr int STAGE = (BM + BN) * kStageBytes;
  constexpr int CA = BM / 8 / WAVES, CB = BN / 8 / WAVES;  // copies a wave and operand
  static_assert(CA * WAVES * 8 == BM && CB * WAVES * 8 == BN && WM * MI * 32 == BM, "whole copies and blocks");
  static_assert((!OA || BM % 128 == 0) && (!OB || BN % 128 == 0), "outer operands lie in 128 columns");
  static_assert(!OA || WAVES * 32 == BM, "a wave's column sums");
  // One array a stage: the compiler waits for the copies into the array that a read names, and for those alone.
  __shared__ __align__(256) char lds0[STAGE], lds1[STAGE];
  lds_char *const s0 = (lds_char*)lds0, *const s1 = (lds_char*)lds1;
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Work k = work_of<BM, BN>(g.e);
  const int size = CODES ? 1 : 2, per_stage = kStageBytes / size;
  const int64_t stages = (g.k + per_stage - 1) / per_stage, t0 = (int64_t)k.split * g.chunk;
  const int64_t t1 = t0 + g.chunk < stages ? t0 + g.chunk : stages;
  const int steps = (int)(t1 - t0);

  Copy<OA, WAVES, CA> ca;
  Copy<OB, WAVES, CB> cb;
  ca.init(g.a, g.a_stride, k.i0, g.e.m, g.k, size, stages - 1, w, lane);
  cb.init(g.b, g.b_stride, k.j0, g.e.n, g.k, size, stages - 1, w, lane);
  int64_t at = t0;  // the stage copied next
  const auto copy = [&](lds_char* stage) {
    const uint32_t none = at < t1 ? 0 : kNowhere, last = at == stages - 1 ? ~0u : 0;
    ca.issue(stage, at, last, none, w);
    cb.issue(stage + BM * kStageBytes, at, last, none, w);
    ++at;
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
    if constexpr (CODES) {  // a quarter is 32 codes: eight of this lane's sixteen at a time
#pragma unroll
      for (int h = 0; h < 4; h += 2) {
        u32x4 b[NI];
#pragma unroll
        for (int n = 0; n < NI; ++n) b[n] = widen(fb[set][n][h], fb[set][n][h + 1]);
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const u32x4 a = widen(fa[set][m][h], fa[set][m][h + 1]);
#pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = mfma_bf16(b[n], a, acc[m][n]);
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] = mfma_bf16(fb[set][n], fa[set][m], acc[m][n]);
    }
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
        acc[m][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(join(fb[set][n], fb[set + 1][n]),
                                                                    join(fa[set][m], fa[set + 1][m]), acc[m][n], 0, 0, 0,
                                                                    0x7f7f7f7f, 0, 0x7f7f7f7f);
  };
  // Column sums of a, in the workgroups of the first column tile: wave w takes 32 columns.
  const bool sums = OA && (g.sums || g.sums_out) && k.j0 == 0;
  float sum = 0.f;
  Reads<OA, 1> rs;
  rs.init(0, 32 * w, lane);
  const auto add = [&](const lds_char* stage) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u32x4 v = rs.read(stage, 0, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t u = v[i];
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
  Bf16Terms<MI, OB, CODES> terms;
  if (bf16_rows<OB>(g)) terms.load(g.e, k, (int)(g.e.m - k.i0 < BM ? g.e.m - k.i0 : BM), wm, wn, lane);
  wait_vmem();  // no copy outlives the stages
  __syncthreads();

  if constexpr (OA) {
    if (sums) {
      sum += __shfl_xor(sum, 32);
      const int64_t row = k.i0 + 32 * w + lane;
      if (lane < 32 && row < g.e.m) {
        if (g.sums_out)
          store_one(g.sums_out, row, g.e.dtype, sum);
        else
          g.sums[(int64_t)k.split * g.e.m + row] = sum;
      }
    }
  }
  constexpr int PER = WAVES / 2;  // waves whose strips share a stage's array
  write_tile<BM, MI, OB, FORM == Form::kWidened, CODES>(g, k, acc, (strip_ptr)((w < PER ? s0 : s1) + (w % PER) * kStripBytes), wm, wn,
                                              lane, terms, MendNothing());
}

template <bool PLAIN, bool F32, int N>
__global__ void __launch_bounds__(256) join_kernel(ProductArgs g) {
  join<PLAIN, F32, N>(g, MendNothing());
}

template <bool OA, bool OB, Form FORM, int TILE>
hipError_t launch_tile(const ProductArgs& g, hipStream_t stream) {
  const int64_t tiles = ((g.e.m + TILE - 1) / TILE) * ((g.e.n + TILE - 1) / TILE);
  hipLaunchKernelGGL((product_kernel<OA, OB, FORM, TILE, TILE>), dim3((unsigned)(tiles * g.splits)), dim3(threads_of(TILE)), 0,
                     stream, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !g.part) return e;
  if (g.e.vec)
    hipLaunchKernelGGL((join_kernel<OB, FORM == Form::kWidened, 8>), join_grid(g), dim3(256), 0, stream, g);
  else
    hipLaunchKernelGGL((join_kernel<OB, FORM == Form::kWidened, 1>), join_grid(g), dim3(256), 0, stream, g);
  return hipGetLastError();
}

template <bool OA, bool OB, Form FORM>
hipError_t launch_operands(int tile, const ProductArgs& g, hipStream_t stream) {
  return tile == 256 ? launch_tile<OA, OB, FORM, 256>(g, stream) : launch_tile<OA, OB, FORM, 128>(g, stream);
}

}  // namespace

hipError_t launch_product(Operands how, int32_t op, int tile, const ProductArgs& a, hipStream_t stream) {
  if (op == kOpF32) return launch_product_f32(how, tile, a, stream);
  if (op == kOpE4m3)
    return a.e.dtype == FWN_F32 ? launch_operands<false, false, Form::kWidened>(tile, a, stream)
                                : launch_operands<false, false, Form::kE4m3>(tile, a, stream);
  if (how == Operands::kInnerInner) return launch_operands<false, false, Form::kBf16>(tile, a, stream);
  if (how == Operands::kInnerOuter) return launch_operands<false, true, Form::kBf16>(tile, a, stream);
  return launch_operands<true, true, Form::kBf16>(tile, a, stream);
}

}  // namespace fwn
