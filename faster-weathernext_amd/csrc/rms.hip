// Root-mean-square norm of rows, with the residual's addition in front, its output in the tensors' dtype
// or in e4m3 with one scale a row, and its backward pass (gfx950).
//
//   s = rnd(x + y),  r = 1 / sqrt(mean(s^2) + eps),  v = s r w;  out = rnd(v)
//   8 bits: scale = max(max|v| / 448, 2^-126), q = e4m3(v (1 / scale)), from v before any rounding
//   gx = g_sum + r (h - s r^2 mean(h s)),  h = g_out w;   gw = sum over the rows of g_out s r
//
// Streaming passes bound by HBM: a row is held in registers from its only load to its outputs, so each
// byte moves once, and the backward recomputes r from s rather than reading it. TPR threads share a row,
// each with VPT vectors of E elements (16 bytes). Vectors need no alignment but their elements' (the compiler makes
// one 16-byte access of them all the same); where a row ends inside a vector (TAIL) that one goes by elements.
// With x + y, 40,962 x 768 bf16: forward 49 us (5.1 TB/s), in 8 bits 44 to 50, backward 44 and 4 for the weight's sums (5.6);
// 10,242 x 1,283 float32: 44 (4.8) and 47; 8,192 x 4,096 float32: 91 (5.9) and 96.
#include "rms_kernels.h"

#include "fwn_attn.h"
#include "linear_act.h"
#include "rms_device.h"

namespace fwn {
namespace {

typedef uint32_t u8x4_any __attribute__((ext_vector_type(1), aligned(1)));
typedef uint32_t u8x8_any __attribute__((ext_vector_type(2), aligned(1)));

template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
    const uint32_t u = __shfl_xor(v, o);
    v = u > v ? u : v;
  }
  if constexpr (TPR > 64) {
    const int wave = (int)threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = as_float(v);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) {
      const uint32_t u = as_bits(red[w]);
      v = u > v ? u : v;
    }
  }
  return v;
}

// E codes of f * inv at p, inv = 1 / scale rounded: within 2^-23 of the quotient, which decides codes only where it is that near
// the middle of two (0.05% of bf16 rows' codes, whose quotients often are middles; either is as near there). |f * inv| is at
// most 448 (1 + 2^-22), which rounds to 448: no clamp, which would turn NaN into a number.
template <int E, bool TAIL>
__device__ __forceinline__ void store_q8(uint8_t* p, int left, const float (&f)[E], float inv) {
  if (TAIL && left < E) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) p[e] = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[e] * inv, 0.f, 0, false);
    return;
  }
  uint32_t d[E / 4];
#pragma unroll
  for (int k = 0; k < E / 4; ++k) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k] * inv, f[4 * k + 1] * inv, 0, false);
    d[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2] * inv, f[4 * k + 3] * inv, lo, true);
  }
  if constexpr (E == 8)
    *(u8x8_any*)p = u8x8_any{d[0], d[1]};
  else
    *(u8x4_any*)p = u8x4_any{d[0]};
}

template <typename T, int TPR, int VPT, bool Q8, bool NT, bool TAIL>
__global__ void __launch_bounds__(kThreads<TPR>) rms_kernel(RmsArgs a) {
  constexpr int E = 16 / sizeof(T), RPW = kThreads<TPR> / TPR;  // rows of a workgroup
  __shared__ float red[16];
  const int t = (int)threadIdx.x % TPR;
  const float inv_c = 1.f / (float)a.channels;
  for (int64_t row0 = (int64_t)blockIdx.x * RPW; row0 < a.rows; row0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = row0 + (int)threadIdx.x / TPR;
    const bool ok = row < a.rows;
    const T* x = (const T*)a.x + row * a.x_stride;
    float f[VPT][E], w[VPT][E];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] = 0.f;
      if (ok && c < a.channels) load<T, E, true, TAIL>(x + c, a.channels - c, f[k]);
    }
    if (a.y) {
      const T* y = (const T*)a.y + row * a.y_stride;
      float g[VPT][E];
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (ok && c < a.channels) load<T, E, true, TAIL>(y + c, a.channels - c, g[k]);
      }
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (!ok || c >= a.channels) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) f[k][e] += g[k][e];
        round_to<T>(f[k]);
        store<T, E, NT, TAIL>((T*)a.sum + row * a.channels + c, a.channels - c, f[k]);
      }
    }
    float r = 1.f;
    if (a.norm) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (a.weight && c < a.channels) load_weight<T, E, TAIL>(a.weight, a.weight_f32, c, a.channels - c, w[k]);
      }
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) sq = fmaf(f[k][e], f[k][e], sq);
      r = 1.f / sqrtf(row_sum<TPR>(sq, red) * inv_c + a.eps);
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (c >= a.channels) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) f[k][e] = f[k][e] * r * (a.weight ? w[k][e] : 1.f);
      }
    }
    if constexpr (Q8) {
      // The largest magnitude by its bits: a NaN's are above infinity's.
      uint32_t most = 0;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t u = as_bits(f[k][e]) & 0x7fffffffu;
          most = u > most ? u : most;
        }
      const float top = as_float(row_max<TPR>(most, red));
      const float least = 0x1p-126f, s = top / 448.f, scale = s < least ? least : s, inv = 1.f / scale;
      if (!ok) continue;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (c < a.channels) store_q8<E, TAIL>(a.q + row * a.channels + c, a.channels - c, f[k], inv);
      }
      if (t == 0) a.scale[row] = scale;
    } else {
      if (!ok) continue;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (c < a.channels) store<T, E, NT, TAIL>((T*)a.out + row * a.channels + c, a.channels - c, f[k]);
      }
    }
  }
}

// gw's sums stay in each thread's registers over all rows of its workgroup, are added over the rows that
// the workgroup holds at once and go out as one partial row a workgroup, in a fixed order.
template <typename T, int TPR, int VPT, bool NT, bool TAIL>
__global__ void __launch_bounds__(kThreads<TPR>) rms_bwd_kernel(RmsBwdArgs a) {
  constexpr int E = 16 / sizeof(T), RPW = kThreads<TPR> / TPR;
  __shared__ float red[32];
  __shared__ float sums[RPW > 1 ? TPR * VPT * E : 1];
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.channels;
  float w[VPT][E], gw[VPT][E];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = (t + TPR * k) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) gw[k][e] = 0.f, w[k][e] = 1.f;
    if (a.weight && c < a.channels) load_weight<T, E, TAIL>(a.weight, a.weight_f32, c, a.channels - c, w[k]);
  }
  for (int64_t row0 = (int64_t)blockIdx.x * RPW; row0 < a.rows; row0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = row0 + own;
    const bool ok = row < a.rows;
    const int64_t at = row * a.channels;
    float f[VPT][E], g[VPT][E], gs[VPT][E];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] = g[k][e] = gs[k][e] = 0.f;
      if (!ok || c >= a.channels) continue;
      load<T, E, true, TAIL>((const T*)a.s + at + c, a.channels - c, f[k]);
      load<T, E, true, TAIL>((const T*)a.g_out + at + c, a.channels - c, g[k]);
      if (a.g_sum) load<T, E, true, TAIL>((const T*)a.g_sum + at + c, a.channels - c, gs[k]);
    }
    float sq = 0.f, hs = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sq = fmaf(f[k][e], f[k][e], sq);
        hs = fmaf(g[k][e] * w[k][e], f[k][e], hs);
      }
    row_sums<TPR>(sq, hs, red);
    const float r = 1.f / sqrtf(sq * inv_c + a.eps), c2 = hs * inv_c * r * r;
    if (!ok) continue;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      if (c >= a.channels) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        o[e] = fmaf(r, g[k][e] * w[k][e] - f[k][e] * c2, gs[k][e]);
        gw[k][e] = fmaf(g[k][e], f[k][e] * r, gw[k][e]);
      }
      store<T, E, NT, TAIL>((T*)a.gx + at + c, a.channels - c, o);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * a.channels;
  if constexpr (RPW == 1) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (t + TPR * k) * E + e;
        if (c < a.channels) part[c] = gw[k][e];
      }
  } else {
    for (int g = 0; g < RPW; ++g) {
      if (own == g) {
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float* p = sums + (t + TPR * k) * E + e;
            *p = g == 0 ? gw[k][e] : *p + gw[k][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.channels; c += kThreads<TPR>) part[c] = sums[c];
  }
}

template <typename T, bool NT, bool TAIL>
struct Forward {
  const RmsArgs& a;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    constexpr int RPW = kThreads<TPR> / TPR;
    const int64_t blocks = (a.rows + RPW - 1) / RPW;
    const dim3 grid((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)), block(kThreads<TPR>);
    if (a.q)
      hipLaunchKernelGGL((rms_kernel<T, TPR, VPT, true, NT, TAIL>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((rms_kernel<T, TPR, VPT, false, NT, TAIL>), grid, block, 0, stream, a);
    return hipGetLastError();
  }
};

template <typename T, bool NT, bool TAIL>
struct Backward {
  const RmsBwdArgs& a;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, VPT, NT, TAIL>), dim3((unsigned)a.blocks), dim3(kThreads<TPR>), 0, stream, a);
    return hipGetLastError();
  }
};

template <template <typename, bool, bool> class Pass, typename T, typename Args>
hipError_t launch_as(const Args& a, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int n = (a.channels + E - 1) / E;
  if (a.channels % E)
    return a.stream ? choose<E>(n, Pass<T, true, true>{a, stream}) : choose<E>(n, Pass<T, false, true>{a, stream});
  return a.stream ? choose<E>(n, Pass<T, true, false>{a, stream}) : choose<E>(n, Pass<T, false, false>{a, stream});
}

}  // namespace

hipError_t launch_rms(int dtype, const RmsArgs& args, hipStream_t stream) {
  RmsArgs a = args;
  const uint64_t bytes = (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2);
  a.stream = (a.y ? bytes : 0) + (a.q ? (uint64_t)a.rows * a.channels : bytes) >= kStreamBytes;
  return dtype == FWN_F32 ? launch_as<Forward, float>(a, stream) : launch_as<Forward, uint16_t>(a, stream);
}

// Each workgroup writes a partial row, so it has 8 rows at least (32 where rows share waves), and there
// are at most four workgroups a CU. 10,242 x 1,283 float32 with 8 rows 51 us, with 16 59; 4,096 x 8,192 bf16 with 8 rows
// 66, with 4 82.
int32_t rms_bwd_blocks(int64_t rows, int32_t channels) {
  const int64_t least = channels <= 256 ? 32 : 8;
  const int64_t want = (rows + least - 1) / least;
  return (int32_t)(want < 1 ? 1 : want < 1024 ? want : 1024);
}

hipError_t launch_rms_bwd(int dtype, const RmsBwdArgs& args, hipStream_t stream) {
  RmsBwdArgs a = args;
  a.stream = (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  const hipError_t rc = dtype == FWN_F32 ? launch_as<Backward, float>(a, stream) : launch_as<Backward, uint16_t>(a, stream);
  if (rc != hipSuccess || !a.part) return rc;
  return launch_column_sums(a.part, a.blocks, a.channels, a.gw, a.weight_f32 ? FWN_F32 : dtype, stream);
}

}  // namespace fwn
