// Root-mean-square norm of rows, with the residual's addition in front, its output in the tensors' dtype
// or in e4m3 with one scale a row, and its backward pass (gfx950).
//
//   s = rnd(x + y),  r = 1 / sqrt(mean(s^2) + eps),  v = s r w;  out = rnd(v)
//   8 bits: scale = max(max|v| / 448, 2^-126), q = e4m3(v / scale), from v before any rounding
//   gx = g_sum + r (h - s r^2 mean(h s)),  h = g_out w;   gw = sum over the rows of g_out s r
//
// Streaming passes bound by HBM: a row is held in registers from its only load to its outputs, so each
// byte moves once, and the backward recomputes r from s rather than reading it. TPR threads share a row,
// each with VPT vectors of E elements (16 bytes; E = 1 for rows that are not whole aligned vectors).
#include "rms_kernels.h"

#include "fwn_attn.h"

namespace fwn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int64_t kMostBlocks = 1 << 20;           // of a forward launch; more rows are looped over
constexpr uint64_t kStreamBytes = 256ull << 20;  // bytes written from which stores are non-temporal (rows.hip)

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ uint32_t bf16_bits(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// E elements of T (float, or uint16_t: bfloat16 bits) at p as floats.
template <typename T, int E, bool NT>
__device__ __forceinline__ void load(const T* p, float (&f)[E]) {
  if constexpr (E == 1) {
    const T v = NT ? __builtin_nontemporal_load(p) : *p;
    if constexpr (sizeof(T) == 4) {
      f[0] = v;
    } else {
      f[0] = as_float((uint32_t)v << 16);
    }
  } else {
    const u32x4 v = NT ? __builtin_nontemporal_load((const u32x4*)p) : *(const u32x4*)p;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t u = v[k];
      if constexpr (sizeof(T) == 4) {
        f[k] = as_float(u);
      } else {
        f[2 * k] = as_float(u << 16);
        f[2 * k + 1] = as_float(u & 0xffff0000u);
      }
    }
  }
}

template <typename T, int E, bool NT>
__device__ __forceinline__ void store(T* p, const float (&f)[E]) {
  if constexpr (E == 1) {
    T v;
    if constexpr (sizeof(T) == 4) {
      v = f[0];
    } else {
      v = (T)bf16_bits(f[0]);
    }
    if constexpr (NT)
      __builtin_nontemporal_store(v, p);
    else
      *p = v;
  } else {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = as_bits(f[k]);
      } else {
        v[k] = bf16_bits(f[2 * k]) | bf16_bits(f[2 * k + 1]) << 16;
      }
    }
    if constexpr (NT)
      __builtin_nontemporal_store(v, (u32x4*)p);
    else
      *(u32x4*)p = v;
  }
}

// The values as their dtype holds them.
template <typename T, int E>
__device__ __forceinline__ void round_to(float (&f)[E]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = as_float(bf16_bits(f[e]) << 16);
  }
}

// E weights from channel c, of T or of float.
template <typename T, int E>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int64_t c, float (&f)[E]) {
  if (sizeof(T) == 4 || !f32) {
    load<T, E, false>((const T*)w + c, f);
  } else if constexpr (E == 1) {
    f[0] = ((const float*)w)[c];
  } else {
#pragma unroll
    for (int h = 0; h < E; h += 4) {
      const u32x4 v = *(const u32x4*)((const float*)w + c + h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t u = v[k];
        f[h + k] = as_float(u);
      }
    }
  }
}

// Sum and maximum over the TPR threads of a row, by every one of them; fixed order.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (TPR > 64) {
    const int wave = (int)threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) v += red[w];
  }
  return v;
}

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

// E codes of f * inv at p. |f * inv| is at most 448 (1 + 2^-22), which rounds to 448: no clamp, which
// would turn NaN into a number.
template <int E>
__device__ __forceinline__ void store_q8(uint8_t* p, const float (&f)[E], float inv) {
  if constexpr (E == 1) {
    *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, 0.f, 0, false);
  } else {
    uint32_t d[E / 4];
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k] * inv, f[4 * k + 1] * inv, 0, false);
      d[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[4 * k + 2] * inv, f[4 * k + 3] * inv, lo, true);
    }
    if constexpr (E == 8)
      *(u32x2*)p = u32x2{d[0], d[1]};
    else
      *(uint32_t*)p = d[0];
  }
}

template <int TPR>
constexpr int kThreads = TPR < 256 ? 256 : TPR;

template <typename T, int E, int TPR, int VPT, bool Q8, bool NT>
__global__ void __launch_bounds__(kThreads<TPR>) rms_kernel(RmsArgs a) {
  constexpr int RPW = kThreads<TPR> / TPR;  // rows of a workgroup
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
      if (ok && c < a.channels) load<T, E, true>(x + c, f[k]);
    }
    if (a.y) {
      const T* y = (const T*)a.y + row * a.y_stride;
      float g[VPT][E];
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (ok && c < a.channels) load<T, E, true>(y + c, g[k]);
      }
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (!ok || c >= a.channels) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) f[k][e] += g[k][e];
        round_to<T>(f[k]);
        store<T, E, NT>((T*)a.sum + row * a.channels + c, f[k]);
      }
    }
    float r = 1.f;
    if (a.norm) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (a.weight && c < a.channels) load_weight<T, E>(a.weight, a.weight_f32, c, w[k]);
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
        if (c < a.channels) store_q8<E>(a.q + row * a.channels + c, f[k], inv);
      }
      if (t == 0) a.scale[row] = scale;
    } else {
      if (!ok) continue;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        if (c < a.channels) store<T, E, NT>((T*)a.out + row * a.channels + c, f[k]);
      }
    }
  }
}

// gw's sums stay in each thread's registers over all rows of its workgroup, are added over the rows that
// the workgroup holds at once and go out as one partial row a workgroup, in a fixed order.
template <typename T, int E, int TPR, int VPT, bool NT>
__global__ void __launch_bounds__(kThreads<TPR>) rms_bwd_kernel(RmsBwdArgs a) {
  constexpr int RPW = kThreads<TPR> / TPR;
  __shared__ float red[16];
  __shared__ float sums[RPW > 1 ? TPR * VPT * E : 1];
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.channels;
  float w[VPT][E], gw[VPT][E];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = (t + TPR * k) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) gw[k][e] = 0.f, w[k][e] = 1.f;
    if (a.weight && c < a.channels) load_weight<T, E>(a.weight, a.weight_f32, c, w[k]);
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
      load<T, E, true>((const T*)a.s + at + c, f[k]);
      load<T, E, true>((const T*)a.g_out + at + c, g[k]);
      if (a.g_sum) load<T, E, true>((const T*)a.g_sum + at + c, gs[k]);
    }
    float sq = 0.f, hs = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        sq = fmaf(f[k][e], f[k][e], sq);
        hs = fmaf(g[k][e] * w[k][e], f[k][e], hs);
      }
    const float r = 1.f / sqrtf(row_sum<TPR>(sq, red) * inv_c + a.eps);
    const float c2 = row_sum<TPR>(hs, red) * inv_c * r * r;
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
      store<T, E, NT>((T*)a.gx + at + c, o);
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

constexpr int kGroups = 16;  // shares of the partial rows that a workgroup adds in parallel

// gw from the partial rows: 64 channels a workgroup.
__global__ void __launch_bounds__(64 * kGroups) rms_sums_kernel(RmsBwdArgs a, bool bf16) {
  __shared__ float red[kGroups][64];
  const int lane = threadIdx.x & 63, grp = (int)threadIdx.x >> 6;
  const int c = (int)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (c < a.channels) {
#pragma unroll 8
    for (int b = grp; b < a.blocks; b += kGroups) s += a.part[(int64_t)b * a.channels + c];
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp != 0 || c >= a.channels) return;
#pragma unroll
  for (int g = 1; g < kGroups; ++g) s += red[g][lane];
  if (bf16)
    ((uint16_t*)a.gw)[c] = (uint16_t)bf16_bits(s);
  else
    ((float*)a.gw)[c] = s;
}

// Calls f with the instance of (threads a row, vectors a thread) for `n` vectors of E elements.
template <int E, typename F>
hipError_t choose(int n, F&& f) {
  // Rows of few vectors share a wave; long ones take as many waves as keep a thread's vectors few.
  if (n <= 16) return f.template operator()<16, 1>();
  if (n <= 32) return f.template operator()<16, 2>();
  if (n <= 64) return f.template operator()<64, 1>();
  if (n <= 128) return f.template operator()<64, 2>();
  if (n <= 256) return f.template operator()<64, 4>();
  if (n <= 512) return f.template operator()<256, 2>();
  if (n <= 1024) return f.template operator()<256, 4>();
  if (n <= 2048) return f.template operator()<1024, 2>();
  if constexpr (E <= 4) {
    if (n <= 4096) return f.template operator()<1024, 4>();
  }
  if constexpr (E == 1) {
    if (n <= 16384) return f.template operator()<1024, 16>();
  }
  return hipErrorInvalidValue;
}

template <typename T, int E>
struct Forward {
  const RmsArgs& a;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    constexpr int RPW = kThreads<TPR> / TPR;
    const int64_t blocks = (a.rows + RPW - 1) / RPW;
    const dim3 grid((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)), block(kThreads<TPR>);
    if (a.q && a.stream)
      hipLaunchKernelGGL((rms_kernel<T, E, TPR, VPT, true, true>), grid, block, 0, stream, a);
    else if (a.q)
      hipLaunchKernelGGL((rms_kernel<T, E, TPR, VPT, true, false>), grid, block, 0, stream, a);
    else if (a.stream)
      hipLaunchKernelGGL((rms_kernel<T, E, TPR, VPT, false, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((rms_kernel<T, E, TPR, VPT, false, false>), grid, block, 0, stream, a);
    return hipGetLastError();
  }
};

template <typename T, int E>
struct Backward {
  const RmsBwdArgs& a;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    const dim3 grid((unsigned)a.blocks), block(kThreads<TPR>);
    if (a.stream)
      hipLaunchKernelGGL((rms_bwd_kernel<T, E, TPR, VPT, true>), grid, block, 0, stream, a);
    else
      hipLaunchKernelGGL((rms_bwd_kernel<T, E, TPR, VPT, false>), grid, block, 0, stream, a);
    return hipGetLastError();
  }
};

bool aligned(const void* p, uintptr_t to = 16) { return ((uintptr_t)p & (to - 1)) == 0; }

}  // namespace

hipError_t launch_rms(int dtype, const RmsArgs& args, hipStream_t stream) {
  RmsArgs a = args;
  const int size = dtype == FWN_F32 ? 4 : 2, e = 16 / size;
  const uint64_t bytes = (uint64_t)a.rows * a.channels * size;
  a.stream = (a.y ? bytes : 0) + (a.q ? (uint64_t)a.rows * a.channels : bytes) >= kStreamBytes;
  const bool vec = a.channels % e == 0 && a.x_stride % e == 0 && a.y_stride % e == 0 && aligned(a.x) && aligned(a.y) &&
                   aligned(a.weight) && aligned(a.sum) && aligned(a.out) && aligned(a.q, e);
  const int n = vec ? a.channels / e : a.channels;
  if (dtype == FWN_F32)
    return vec ? choose<4>(n, Forward<float, 4>{a, stream}) : choose<1>(n, Forward<float, 1>{a, stream});
  return vec ? choose<8>(n, Forward<uint16_t, 8>{a, stream}) : choose<1>(n, Forward<uint16_t, 1>{a, stream});
}

// Four rows at least to each of a workgroup's places and about four workgroups a CU.
int32_t rms_bwd_blocks(int64_t rows, int32_t channels) {
  const int64_t at_once = channels <= 256 ? 16 : channels <= 2048 ? 4 : 1;
  const int64_t want = (rows + 4 * at_once - 1) / (4 * at_once);
  return (int32_t)(want < 1 ? 1 : want < 1024 ? want : 1024);
}

hipError_t launch_rms_bwd(int dtype, const RmsBwdArgs& args, hipStream_t stream) {
  RmsBwdArgs a = args;
  const int size = dtype == FWN_F32 ? 4 : 2, e = 16 / size;
  a.stream = (uint64_t)a.rows * a.channels * size >= kStreamBytes;
  const bool vec = a.channels % e == 0 && aligned(a.s) && aligned(a.weight) && aligned(a.g_out) && aligned(a.g_sum) &&
                   aligned(a.gx);
  const int n = vec ? a.channels / e : a.channels;
  hipError_t rc;
  if (dtype == FWN_F32)
    rc = vec ? choose<4>(n, Backward<float, 4>{a, stream}) : choose<1>(n, Backward<float, 1>{a, stream});
  else
    rc = vec ? choose<8>(n, Backward<uint16_t, 8>{a, stream}) : choose<1>(n, Backward<uint16_t, 1>{a, stream});
  if (rc != hipSuccess || !a.part) return rc;
  hipLaunchKernelGGL(rms_sums_kernel, dim3((unsigned)(a.channels + 63) / 64), dim3(64 * kGroups), 0, stream, a,
                     dtype == FWN_BF16 && !a.weight_f32);
  return hipGetLastError();
}

}  // namespace fwn
