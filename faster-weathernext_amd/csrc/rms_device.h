// Device-side building blocks of the passes over rows that hold a row in registers (gfx950): vectors of 16 bytes at any
// alignment of their elements, sums over the threads of a row, and the choice of threads and vectors by the row's length.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace fwn {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
// The same at any address of a row.
typedef uint32_t f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t bf16x8_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
struct Any {
  typedef bf16x8_any type;
};
template <>
struct Any<float> {
  typedef f32x4_any type;
};

constexpr int64_t kMostBlocks = 1 << 20;           // of a forward launch; more rows are looped over
constexpr uint64_t kStreamBytes = 256ull << 20;  // bytes written from which stores are non-temporal (rows.hip)

__device__ __forceinline__ float as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t as_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ __forceinline__ uint32_t bf16_bits(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

template <typename T>
__device__ __forceinline__ float load_one(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *p;
  } else {
    return as_float((uint32_t)*p << 16);
  }
}

template <typename T>
__device__ __forceinline__ void store_one(T* p, float v) {
  if constexpr (sizeof(T) == 4) {
    *p = v;
  } else {
    *p = (T)bf16_bits(v);
  }
}

// The E elements of T (float, or uint16_t: bfloat16 bits) at p, as they lie there.
template <typename T, bool NT>
__device__ __forceinline__ u32x4 load_raw(const T* p) {
  typedef typename Any<T>::type vec;
  return NT ? __builtin_nontemporal_load((const vec*)p) : *(const vec*)p;
}

// The same as floats.
template <typename T, int E>
__device__ __forceinline__ void unpack(const u32x4& v, float (&f)[E]) {
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

// The E elements at p as floats; with TAIL those of the first `left`, and zeros.
template <typename T, int E, bool NT, bool TAIL>
__device__ __forceinline__ void load(const T* p, int left, float (&f)[E]) {
  if (TAIL && left < E) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < left ? load_one(p + e) : 0.f;
    return;
  }
  unpack<T>(load_raw<T, NT>(p), f);
}

template <typename T, int E, bool NT, bool TAIL>
__device__ __forceinline__ void store(T* p, int left, const float (&f)[E]) {
  if (TAIL && left < E) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) store_one(p + e, f[e]);
    return;
  }
  typedef typename Any<T>::type vec;
  vec v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) {
      v[k] = as_bits(f[k]);
    } else {
      v[k] = bf16_bits(f[2 * k]) | bf16_bits(f[2 * k + 1]) << 16;
    }
  }
  if constexpr (NT)
    __builtin_nontemporal_store(v, (vec*)p);
  else
    *(vec*)p = v;
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
template <typename T, int E, bool TAIL>
__device__ __forceinline__ void load_weight(const void* w, bool f32, int64_t c, int left, float (&f)[E]) {
  if (sizeof(T) == 4 || !f32) {
    load<T, E, false, TAIL>((const T*)w + c, left, f);
  } else if (TAIL && left < E) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < left ? ((const float*)w)[c + e] : 0.f;
  } else {
#pragma unroll
    for (int h = 0; h < E; h += 4) {
      const u32x4 v = *(const f32x4_any*)((const float*)w + c + h);
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

// Two sums at once.
template <int TPR>
__device__ __forceinline__ void row_sums(float& u, float& v, float* red) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
    u += __shfl_xor(u, o);
    v += __shfl_xor(v, o);
  }
  if constexpr (TPR > 64) {
    const int wave = (int)threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red[2 * wave] = u;
      red[2 * wave + 1] = v;
    }
    __syncthreads();
    u = red[0];
    v = red[1];
#pragma unroll
    for (int w = 1; w < TPR / 64; ++w) {
      u += red[2 * w];
      v += red[2 * w + 1];
    }
  }
}

template <int TPR>
constexpr int kThreads = TPR < 256 ? 256 : TPR;

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
  if constexpr (E == 4) {
    if (n <= 4096) return f.template operator()<1024, 4>();
  }
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace fwn
