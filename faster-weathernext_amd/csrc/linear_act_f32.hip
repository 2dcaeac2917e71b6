// The linear layers' products of float32 operands (gfx950), at float32's precision on the bf16 matrix units.
//
// A value times 2^16 is the exact sum of three bf16 parts: it rounded, what is left rounded, and the rest. The second is at
// most 2^-8 of the value and the third 2^-17, of either sign. Of the nine products of parts the six largest are formed and
// accumulated in float32, small ones first; the three left out are together within 2^-24 (1 + 2^-9) of the product, as its
// rounding to float32 would be, and without a direction. (Parts cut off rather than rounded took as long, lost up to 2^-21
// of a product and always towards zero.) The factor puts the last bits of the least float32 numbers, 2^-149, at bf16's own,
// 2^-133: without it what lies below is lost, 1e-4 of values of 1e-37. Sums carry 2^32, which the epilogue takes back; where
// that or the factor leaves float32's range (sums from 2^96 on, operands from 2^111), outputs come out infinite or NaN and
// are formed anew of the whole values, as those that an infinity feeds. Six bf16 MFMAs do what eight times as many clocks
// of float32 MFMAs do. The parts are formed on the way from memory to LDS, so an operand of any strides and alignment is
// read where it lies, once a tile.
//
// A workgroup is 4 waves on a 128 x 128 tile, a wave 64 x 64: per 16 k it reads 12 KB of LDS for 24 MFMAs. One
// stage of 32 k is 48 KB of parts, so that two or three workgroups share a CU: while one splits and writes its next
// stage, loaded a stage ahead into registers, the others multiply. A stage takes 2.0 us alone on a CU and 1.1 among
// others (4,096 x 4,096 -> 4,096: 200 to 205 TFLOP/s). Where such tiles are too few, an inner a is taken in tiles of 64 x 128, of 1.1 us a
// stage alone and 0.66 among others, us with 128 rows and with 64: 1,000 x 512 -> 512 22 and 17, 2,562 x 515 -> 1,027 43
// and 36, 130 x 1,024 -> 1,024 16 and 13; 10,242 x 768 -> 3,072 260 and 286. Two stages in LDS (a stage split between the products
// of the one before) were slower where tiles fill the chip: 337.
#include "linear_act_device.h"

namespace fwn {
namespace {

constexpr int TILE = 128, STEP = 32;

// Two values as bf16, by one instruction.
__device__ __forceinline__ uint32_t two_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}

// One operand's stages: ROWS rows of 32 k ("inner") or 32 rows of k of 128 columns ("outer"), 4 FOURS values a thread.
// In LDS a part is ROWS rows of 64 bytes or 32 of 256, 16-byte chunks swizzled as for the bf16 kernels.
template <bool OUTER, int ROWS>
struct Operand {
  static constexpr int FOURS = ROWS / 32, PLANE = ROWS * STEP * 2, BYTES = 3 * PLANE;
  static_assert(!OUTER || ROWS == 128, "outer operands have 128 columns");
  const char* base;
  int64_t step;      // bytes from one stage to the next
  uint32_t off[FOURS];   // of this thread's fours of values
  uint32_t lds[FOURS];
  int first_k[FOURS];    // k of a four in the stage
  int limit;         // outer: columns of the fours inside the operand
  bool whole;        // fours do not end inside: of the sum (inner), or of the tile's columns (outer)
  uint32_t at[OUTER ? 4 : 2];  // this lane's reads

  __device__ __forceinline__ void init(const char* p, int64_t stride, int64_t first, int64_t rows, int64_t k, int wave_first,
                                       int lane) {
    base = p + (OUTER ? first * 4 : first * stride);
    step = OUTER ? STEP * stride : STEP * 4;
    whole = OUTER ? rows % 4 == 0 || first + ROWS <= rows : k % 4 == 0;
    const int t = (int)threadIdx.x;
    limit = 4;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
      if constexpr (OUTER) {
        const int row = t / 32 + 8 * i, col = t % 32 * 4;
        off[i] = first + col < rows ? (uint32_t)row * (uint32_t)stride + (uint32_t)col * 4 : kNowhere;
        if (rows - first - col < 4) limit = (int)(rows - first - col);
        first_k[i] = row;
        lds[i] = row * 256 + (((col / 8) ^ swz<16>(row)) << 4) + (col % 8) * 2;
      } else {
        const int row = t / 8 + 32 * i, c = t % 8 * 4;
        off[i] = first + row < rows ? (uint32_t)row * (uint32_t)stride + (uint32_t)c * 4 : kNowhere;
        first_k[i] = c;
        lds[i] = row * 64 + (((c / 8) ^ (row / 4 % 4)) << 4) + (c % 8) * 2;
      }
    }
    const int i = lane & 31, g = lane >> 5;
    if constexpr (OUTER) {
      const int G = lane >> 4, u = lane & 15, e = u >> 2, q = u & 3;
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 8 * g + 4 * h + e, chunk = 4 * ((wave_first + 32 * m) >> 5) + 2 * (G & 1) + (q >> 1);
          at[2 * m + h] = r * 256 + ((chunk ^ swz<16>(r)) << 4) + (q & 1) * 8;
        }
    } else {
      const int r = wave_first + i;
#pragma unroll
      for (int c = 0; c < 2; ++c) at[c] = r * 64 + (((2 * c + g) ^ (r / 4 % 4)) << 4);
    }
  }

  // Stage t's values; `left`: k from its first to the sum's end (what lies past it is zeros). Fours need no alignment
  // but their elements'.
  __device__ __forceinline__ void load(int64_t t, int64_t left, u32x4 (&v)[FOURS]) const {
    const rsrc_t r = make_rsrc(base + t * step, kBuffer);
    if (whole || (!OUTER && left >= STEP)) {
#pragma unroll
      for (int i = 0; i < FOURS; ++i) v[i] = bload16(r, off[i] | (first_k[i] < left ? 0 : kNowhere));
    } else {
#pragma unroll
      for (int i = 0; i < FOURS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = OUTER ? e < limit && first_k[i] < left : first_k[i] + e < left;
          v[i][e] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)((off[i] + 4 * e) | (in ? 0 : kNowhere)), 0, 0);
        }
    }
  }

  // Their parts to LDS. An infinity or NaN, or a value that becomes infinite, gives NaN in the middle part, and so in every
  // output that it feeds.
  __device__ __forceinline__ void split(lds_char* to, const u32x4 (&v)[FOURS]) const {
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t u = v[i][e];
        f[e] = as_float(u) * kUp;
      }
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const u32x2 part{two_bf16(f[0], f[1]), two_bf16(f[2], f[3])};
        *(__attribute__((address_space(3))) u32x2*)(to + p * PLANE + lds[i]) = part;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] -= as_float(e % 2 ? part[e / 2] & 0xffff0000u : part[e / 2] << 16);
      }
    }
  }

  // Block m's operand of half c of the stage in the part at `part`.
  __device__ __forceinline__ u32x4 read(const lds_char* part, int m, int c) const {
    if constexpr (OUTER) {
      const u32x2 lo = tr_read(part + c * 4096, at[2 * m]), hi = tr_read(part + c * 4096, at[2 * m + 1]);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    } else {
      return row_read(part + m * 2048, at[c]);
    }
  }
};

// A tile of BM x 128: a wave has BM / 2 x 64 of it.
template <bool OA, bool OB, int BM>
__global__ void __launch_bounds__(256, OA || OB ? 2 : 3) product_f32_kernel(ProductArgs g) {
  typedef Operand<OA, BM> A;
  typedef Operand<OB, TILE> B;
  constexpr int MI = BM / 64;
  __shared__ __align__(256) char lds[A::BYTES + B::BYTES];
  static_assert(sizeof(lds) >= 4 * kStripBytes, "the waves' strips");
  lds_char* const sa = (lds_char*)lds;
  lds_char* const sb = sa + A::BYTES;
  const int lane = (int)threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const Work k = work_of<BM, TILE>(g.e);
  const int64_t stages = (g.k + STEP - 1) / STEP, t0 = (int64_t)k.split * g.chunk;
  const int64_t t1 = t0 + g.chunk < stages ? t0 + g.chunk : stages;
  const int wm = w / 2 * (BM / 2), wn = w % 2 * 64;
  A a;
  B b;
  a.init(g.a, g.a_stride, k.i0, g.e.m, g.k, wm, lane);
  b.init(g.b, g.b_stride, k.j0, g.e.n, g.k, wn, lane);
  f32x16 acc[MI][2];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[m][n] = zero16();
  u32x4 va[A::FOURS], vb[B::FOURS];
  if (t0 < t1) {
    a.load(t0, g.k - t0 * STEP, va);
    b.load(t0, g.k - t0 * STEP, vb);
  }
  for (int64_t t = t0; t < t1; ++t) {
    lds_barrier();  // every wave has read the last stage
    a.split(sa, va);
    b.split(sb, vb);
    if (t + 1 < t1) {
      a.load(t + 1, g.k - (t + 1) * STEP, va);
      b.load(t + 1, g.k - (t + 1) * STEP, vb);
    }
    lds_barrier();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u32x4 fa[3][MI], fb[3][2];
#pragma unroll
      for (int p = 2; p >= 0; --p) {
#pragma unroll
        for (int m = 0; m < MI; ++m) fa[p][m] = a.read(sa + p * A::PLANE, m, c);
#pragma unroll
        for (int n = 0; n < 2; ++n) fb[p][n] = b.read(sb + p * B::PLANE, n, c);
      }
      constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
      for (int i = 0; i < 6; ++i)
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n) acc[m][n] = mfma_bf16(fb[pb[i]][n], fa[pa[i]][m], acc[m][n]);
    }
  }
  __syncthreads();
  write_tile<BM, MI, OB, 1, false>(g, k, acc, (strip_ptr)(sa + w * kStripBytes), wm, wn, lane, {},
                                    MendParts<OA, OB>{g});
}

template <bool OA, bool OB, int N>
__global__ void __launch_bounds__(256) join_f32_kernel(ProductArgs g) {
  join<OB, true, N>(g, MendParts<OA, OB>{g});
}

template <bool OA, bool OB, int BM = TILE>
hipError_t launch(const ProductArgs& g, hipStream_t stream) {
  const int64_t tiles = ((g.e.m + BM - 1) / BM) * ((g.e.n + TILE - 1) / TILE);
  hipLaunchKernelGGL((product_f32_kernel<OA, OB, BM>), dim3((unsigned)(tiles * g.splits)), dim3(256), 0, stream, g);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !g.part) return e;
  if (g.e.vec)
    hipLaunchKernelGGL((join_f32_kernel<OA, OB, 8>), join_grid(g), dim3(256), 0, stream, g);
  else
    hipLaunchKernelGGL((join_f32_kernel<OA, OB, 1>), join_grid(g), dim3(256), 0, stream, g);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_product_f32(Operands how, int tile, const ProductArgs& g, hipStream_t stream) {
  if (how == Operands::kInnerInner) return tile == 64 ? launch<false, false, 64>(g, stream) : launch<false, false>(g, stream);
  if (how == Operands::kInnerOuter) return tile == 64 ? launch<false, true, 64>(g, stream) : launch<false, true>(g, stream);
  return launch<true, true>(g, stream);
}

}  // namespace fwn
