// The root-mean-square norms after a block and before the next one, with the block's gate, the residual's scale and dropout between
// them, forward and backward (gfx950). For the residual x and the block's output y:
//
//   r1 = 1 / sqrt(mean(y^2) + eps),  b = gate y r1 w_post;   s = rnd(scale x + drop(b))
//   r2 = 1 / sqrt(mean(s^2) + eps),  out = rnd(s r2 w_pre)
//
//   a = g_out w_pre,  ds = g_sum + r2 (a - s r2^2 mean(a s)),  gx = scale ds,  db = drop(ds)
//   c = db gate w_post,  gy = r1 (c - y r1^2 mean(c y))
//   g_pre = sum of g_out s r2,  g_post = sum of db gate y r1,  g_gate = sum over the gate's rows of db y r1 w_post
//
// Streaming passes bound by HBM: a row is held in registers from its only load to its outputs, and the backward forms
// both r and what is dropped anew from s, y and the counter. TPR threads share a row, each with VPT vectors of E elements.
// 40,962 x 768 bf16: forward 55 to 57 us (4.4 to 4.6 TB/s), with a gate for each member and dropout 64; backward with both 87 and 6 for the sums
// (without dropout 81: the generator's multiplications run at a quarter of the other instructions' rate). 5,124 x 4,096 bf16 with a
// gate an element: 45 and 69 (4.7 and 4.9 TB/s). 20,480 x 768 float32: 48 and 75 (5.3, 5.0).
#include "dropout_device.h"

#include "fwn_attn.h"
#include "linear_act.h"

namespace fwn {
namespace {

// Sums over the TPR threads of a row, by every one of them; fixed order. Within 16 lanes by rotations, beyond by swaps of rows and
// halves of the wave, none of which takes a trip through LDS as __shfl_xor does (40,968 x 768 bf16 with dropout, backward: 97 us, with
// __shfl_xor 103; forward of 40,962 x 768 57 and 60).
template <int ROTATE>
__device__ __forceinline__ float rotated(float v) {
  return as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)as_bits(v), 0x120 + ROTATE, 0xf, 0xf, false));
}
template <int TPR>
__device__ __forceinline__ float wave_sum(float v) {
  v += rotated<8>(v);
  v += rotated<4>(v);
  v += rotated<2>(v);
  v += rotated<1>(v);
  if constexpr (TPR >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(as_bits(v), as_bits(v), false, false);
    const uint32_t a = r[0], b = r[1];
    v = as_float(a) + as_float(b);
  }
  if constexpr (TPR >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(as_bits(v), as_bits(v), false, false);
    const uint32_t a = r[0], b = r[1];
    v = as_float(a) + as_float(b);
  }
  return v;
}
template <int TPR, int N>
__device__ __forceinline__ void all_sums(float (&v)[N], float* red) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum<TPR>(v[i]);
  if constexpr (TPR > 64) {
    constexpr int WAVES = TPR / 64;
    const int wave = (int)threadIdx.x >> 6, first = wave / WAVES * WAVES;  // of the row
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[N * wave + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = red[N * first + i];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) v[i] += red[N * (first + w) + i];
    }
  }
}

// A gate's row of a row: 32-bit division, rows being fewer than 2^32.
__device__ __forceinline__ int64_t gate_row(int64_t row, int64_t gate_rows, int64_t rows) {
  return gate_rows == 1 ? row : gate_rows >= rows ? 0 : (int64_t)((uint32_t)row / (uint32_t)gate_rows);
}

// Stored past the caches where they could not hold it.
template <typename T, int E, bool TAIL>
__device__ __forceinline__ void put(bool stream, T* p, int left, const float (&f)[E]) {
  if (stream)
    store<T, E, true, TAIL>(p, left, f);
  else
    store<T, E, false, TAIL>(p, left, f);
}

// A vector of a row of `channels` with `left` of them from p on, as it lies in memory. With TAIL the row's last vector is read from
// E elements before the row's end, and fit moves it to its place, with zeros behind: loads of single elements, and any
// load whose values are changed before the branches of the two meet, are waited for one by one (24,512 x 1,283 bf16, forward and
// backward: 119 and 193 us so, 82 and 152 without).
template <typename T, int E, bool TAIL, bool NT = true>
__device__ __forceinline__ u32x4 ask(const T* p, int left, int channels) {
  if constexpr (TAIL) {
    if (channels < E) {  // no row to read before it
      uint32_t d[E];
#pragma unroll
      for (int e = 0; e < E; ++e) d[e] = e < left ? as_bits(load_one(p + e)) : 0u;
      u32x4 v = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) v[e * (int)sizeof(T) / 4] |= (sizeof(T) == 4 ? d[e] : d[e] >> 16) << 8 * (e * (int)sizeof(T) % 4);
      return v;
    }
    return load_raw<T, NT>(left < E ? p + (left - E) : p);
  }
  return load_raw<T, NT>(p);
}
template <typename T, int E, bool TAIL>
__device__ __forceinline__ u32x4 fit(const u32x4& v, int left, int channels) {
  if constexpr (TAIL) {
    if (channels < E || !__any(left < E)) return v;
    const int bytes = (E - channels % E) * (int)sizeof(T);
    u32x4 u = v;
    if (bytes & 8) u = u32x4{u[2], u[3], 0, 0};
    if (bytes & 4) u = u32x4{u[1], u[2], u[3], 0};
    if (bytes & 2) u = u32x4{u[0] >> 16 | u[1] << 16, u[1] >> 16 | u[2] << 16, u[2] >> 16 | u[3] << 16, u[3] >> 16};
    return left < E ? u : v;
  }
  return v;
}

// f times the E weights from channel c of row `row` of w (of T, or of float); NULL: as it is.
template <typename T, int E, bool TAIL>
__device__ __forceinline__ void times(const void* w, bool f32, int64_t row, int c, int channels, float (&f)[E]) {
  if (!w) return;
  float g[E];
  if (sizeof(T) == 4 || !f32)
    unpack<T>(fit<T, E, TAIL>(ask<T, E, TAIL, false>((const T*)w + row + c, channels - c, channels), channels - c, channels), g);
  else
    load_weight<T, E, TAIL>(w, true, row + c, channels - c, g);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] *= g[e];
}

template <typename T, int TPR, int VPT, bool TAIL>
__global__ void __launch_bounds__(kThreads<TPR>) sandwich_kernel(SandwichArgs a) {
  constexpr int E = 16 / sizeof(T), RPW = kThreads<TPR> / TPR;  // rows of a workgroup
  __shared__ float red[16];
  const int t = (int)threadIdx.x % TPR;
  const float inv_c = 1.f / (float)a.channels;
  const Draw draw(a.draw);
  for (int64_t row0 = (int64_t)blockIdx.x * RPW; row0 < a.rows; row0 += (int64_t)gridDim.x * RPW) {
    const int64_t row = row0 + (int)threadIdx.x / TPR;
    const bool ok = row < a.rows;
    const T* const x = (const T*)a.x + row * a.x_stride;
    const T* const y = (const T*)a.y + row * a.y_stride;
    u32x4 vx[VPT], vy[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      vx[k] = vy[k] = u32x4{0, 0, 0, 0};
      if (!ok || c >= a.channels) continue;
      vy[k] = ask<T, E, TAIL>(y + c, a.channels - c, a.channels);
      vx[k] = ask<T, E, TAIL>(x + c, a.channels - c, a.channels);
    }
    float f[VPT][E], b[VPT][E];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int left = a.channels - (t + TPR * k) * E;
      unpack<T>(fit<T, E, TAIL>(vy[k], left, a.channels), b[k]);
      unpack<T>(fit<T, E, TAIL>(vx[k], left, a.channels), f[k]);
    }
    float r = 1.f;
    if (a.post_norm) {
      float sq[1] = {0.f};
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) sq[0] = fmaf(b[k][e], b[k][e], sq[0]);
      all_sums<TPR>(sq, red);
      r = 1.f / sqrtf(sq[0] * inv_c + a.eps);
    }
    const int64_t gate_at = a.gate && ok ? gate_row(row, a.gate_rows, a.rows) * a.channels : 0;
    float sq[1] = {0.f};
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      if (!ok || c >= a.channels) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) b[k][e] *= r;
      times<T, E, TAIL>(a.gate, a.gate_f32, gate_at, c, a.channels, b[k]);
      times<T, E, TAIL>(a.post_weight, a.post_f32, 0, c, a.channels, b[k]);
      if (a.drop) draw.template apply<E>((uint32_t)row, (uint32_t)c, b[k]);
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] = fmaf(a.scale, f[k][e], b[k][e]);
      round_to<T>(f[k]);
      put<T, E, TAIL>(a.stream, (T*)a.sum + row * a.channels + c, a.channels - c, f[k]);
      if (TAIL && a.channels - c < E) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e >= a.channels - c) f[k][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) sq[0] = fmaf(f[k][e], f[k][e], sq[0]);
    }
    all_sums<TPR>(sq, red);
    r = 1.f / sqrtf(sq[0] * inv_c + a.eps);
    if (!ok) continue;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      if (c >= a.channels) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] *= r;
      times<T, E, TAIL>(a.pre_weight, a.pre_f32, 0, c, a.channels, f[k]);
      put<T, E, TAIL>(a.stream, (T*)a.out + row * a.channels + c, a.channels - c, f[k]);
    }
  }
}

// Adds the sums that the workgroup's threads hold over the rows that it holds at once, in a fixed order, and hands them out: a
// thread's own vectors where the workgroup has one row, else a channel a thread. give(channel, channels left, values).
template <int TPR, int VPT, int E, typename Give>
__device__ __forceinline__ void over_rows(const float (&v)[VPT][E], float* sums, int channels, const Give& give) {
  constexpr int RPW = kThreads<TPR> / TPR;
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  if constexpr (RPW == 1) {
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      float f[E];
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = v[k][e];
      if (c < channels) give(c, channels - c, f);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
    __syncthreads();
    for (int g = 0; g < RPW; ++g) {
      if (own == g) {
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float* p = sums + (t + TPR * k) * E + e;
            *p = g == 0 ? v[k][e] : *p + v[k][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < channels; c += kThreads<TPR>) {
      float f[1] = {sums[c]};
      give(c, channels - c, f);
    }
  }
}

__device__ __forceinline__ float weight_at(const void* w, bool f32, int64_t i) {
  return f32 ? ((const float*)w)[i] : load_one((const uint16_t*)w + i);
}
__device__ __forceinline__ void put_weight(void* w, bool f32, int64_t i, float v) {
  if (f32)
    ((float*)w)[i] = v;
  else
    store_one((uint16_t*)w + i, v);
}

// The first `left` of N sums.
template <int N>
__device__ __forceinline__ void put_sums(float* p, int left, const float (&f)[N]) {
  if constexpr (N % 4 == 0) {
    if (left >= N) {
#pragma unroll
      for (int h = 0; h < N; h += 4) *(f32x4_any*)(p + h) = f32x4_any{as_bits(f[h]), as_bits(f[h + 1]), as_bits(f[h + 2]), as_bits(f[h + 3])};
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < left) p[e] = f[e];
}

// E weights from channel c times v; NULL: v.
template <typename T, int E, bool TAIL>
__device__ __forceinline__ void weights(const void* w, bool f32, int64_t row, int c, int channels, float v, float (&f)[E]) {
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = v;
  times<T, E, TAIL>(w, f32, row, c, channels, f);
}

// Waves a SIMD that the backward's registers leave room for.
template <typename T, int TPR, int VPT>
constexpr int kWaves = TPR == 1024 ? 4 : 16 / (int)sizeof(T) * VPT <= 8 ? 4 : 16 / (int)sizeof(T) * VPT <= 16 ? 3 : 2;

// EACH: the gate is of x's shape. Else the rows go by groups that share a row of the gate (one group without a gate), whose
// sum of db y r1 is both the gate's gradient but for post_weight and the group's share of post_weight's but for the gate: one sum in
// registers, beside pre_weight's. What dropout multiplies by is part of the weights, not of db.
template <typename T, int TPR, int VPT, bool EACH, bool TAIL>
__global__ void __launch_bounds__(kThreads<TPR>) __attribute__((amdgpu_waves_per_eu(kWaves<T, TPR, VPT>))) sandwich_bwd_kernel(SandwichBwdArgs a, SandwichGrid grid) {
  constexpr int E = 16 / sizeof(T), RPW = kThreads<TPR> / TPR;
  __shared__ float red[32];
  __shared__ float sums[RPW > 1 ? TPR * VPT * E : 1];
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.channels;
  const Draw draw(a.draw);
  const float keep = a.drop ? draw.keep : 1.f;
  float g_pre[VPT][E], q[VPT][E], pre[VPT][E], w[VPT][E];
#pragma unroll
  for (int k = 0; k < VPT; ++k) {
    const int c = (t + TPR * k) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) g_pre[k][e] = q[k][e] = pre[k][e] = w[k][e] = 0.f;
    if (c >= a.channels) continue;
    weights<T, E, TAIL>(a.pre_weight, a.pre_f32, 0, c, a.channels, 1.f, pre[k]);
    if (EACH) weights<T, E, TAIL>(a.post_weight, a.post_f32, 0, c, a.channels, keep, w[k]);
  }
  float* const part_pre = a.part + (int64_t)blockIdx.x * a.channels;
  float* const part_post = part_pre + (a.g_pre ? (int64_t)grid.blocks * a.channels : 0);
  float* const part_gate = part_post + (a.g_post ? (int64_t)grid.blocks * a.channels : 0);
  const int64_t first = (int64_t)((int)blockIdx.x / grid.per) * grid.of_block;
  const int sub = (int)blockIdx.x % grid.per;
  for (int64_t group = first; group < first + grid.of_block && group < grid.groups; ++group) {
    if constexpr (!EACH) {
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) q[k][e] = 0.f;
        if (c >= a.channels) continue;
        weights<T, E, TAIL>(a.post_weight, a.post_f32, 0, c, a.channels, keep, w[k]);
        times<T, E, TAIL>(a.gate, a.gate_f32, group * a.channels, c, a.channels, w[k]);
      }
    }
    const int64_t begin = group * grid.group_rows, end = begin + grid.group_rows;
    for (int64_t row0 = begin + sub * RPW; row0 < end; row0 += grid.per * RPW) {
      const int64_t row = row0 + own;
      const bool ok = row < end;
      const int64_t at = row * a.channels;
      u32x4 vs[VPT], vy[VPT], vo[VPT], vg[VPT];  // s, y, g_out and g_sum as they lie in memory
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E;
        vs[k] = vy[k] = vo[k] = vg[k] = u32x4{0, 0, 0, 0};
        if (!ok || c >= a.channels) continue;
        const int left = a.channels - c;
        vs[k] = ask<T, E, TAIL>((const T*)a.s + at + c, left, a.channels);
        if (a.g_out) vo[k] = ask<T, E, TAIL>((const T*)a.g_out + at + c, left, a.channels);
        if (a.g_sum) vg[k] = ask<T, E, TAIL>((const T*)a.g_sum + at + c, left, a.channels);
        vy[k] = ask<T, E, TAIL>((const T*)a.y + row * a.y_stride + c, left, a.channels);
      }
      if constexpr (TAIL) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          const int left = a.channels - (t + TPR * k) * E;
          vs[k] = fit<T, E, TAIL>(vs[k], left, a.channels);
          vo[k] = fit<T, E, TAIL>(vo[k], left, a.channels);
          vg[k] = fit<T, E, TAIL>(vg[k], left, a.channels);
          vy[k] = fit<T, E, TAIL>(vy[k], left, a.channels);
        }
      }
      float r2 = 0.f, k2 = 0.f;
      if (a.g_out) {
        float m[2] = {0.f, 0.f};  // s^2, and a s
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          float s[E], h[E];
          unpack<T>(vs[k], s);
          unpack<T>(vo[k], h);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            m[0] = fmaf(s[e], s[e], m[0]);
            m[1] = fmaf(h[e] * pre[k][e], s[e], m[1]);
          }
        }
        all_sums<TPR>(m, red);
        r2 = 1.f / sqrtf(m[0] * inv_c + a.eps);
        k2 = m[1] * inv_c * r2 * r2;
      }
      float db[VPT][E], m[2] = {0.f, 0.f};  // y^2, and c y
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E, left = a.channels - c;
#pragma unroll
        for (int e = 0; e < E; ++e) db[k][e] = 0.f;
        if (!ok || left <= 0) continue;
        unpack<T>(vg[k], db[k]);
        if (a.g_out) {
          float s[E], h[E];
          unpack<T>(vs[k], s);
          unpack<T>(vo[k], h);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            g_pre[k][e] = fmaf(h[e], s[e] * r2, g_pre[k][e]);
            db[k][e] = fmaf(r2, fmaf(-k2, s[e], h[e] * pre[k][e]), db[k][e]);
          }
        }
        if (a.gx) {
          float o[E];
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = a.scale * db[k][e];
          put<T, E, TAIL>(a.stream, (T*)a.gx + at + c, left, o);
        }
        if (a.drop) draw.template select<E>((uint32_t)row, (uint32_t)c, db[k]);
        float y[E], g[E];
        unpack<T>(vy[k], y);
        if constexpr (EACH) {
#pragma unroll
          for (int e = 0; e < E; ++e) g[e] = w[k][e];
          times<T, E, TAIL>(a.gate, a.gate_f32, at, c, a.channels, g);
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          m[0] = fmaf(y[e], y[e], m[0]);
          m[1] = fmaf(db[k][e] * (EACH ? g[e] : w[k][e]), y[e], m[1]);
        }
      }
      float r1 = 1.f, k1 = 0.f;
      if (a.post_norm) {
        all_sums<TPR>(m, red);
        r1 = 1.f / sqrtf(m[0] * inv_c + a.eps);
        k1 = m[1] * inv_c * r1 * r1;
      }
      if (!ok) continue;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E, left = a.channels - c;
        if (left <= 0) continue;
        float y[E], o[E];
        unpack<T>(vy[k], y);
        if constexpr (EACH) {
          // The gate's gradient, and db times the gate in place of db.
          float g[E];
          weights<T, E, TAIL>(a.gate, a.gate_f32, at, c, a.channels, 1.f, g);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            o[e] = db[k][e] * w[k][e] * (y[e] * r1);
            db[k][e] *= g[e];
          }
          if (a.g_gate) {
            if (sizeof(T) == 4 || !a.gate_f32) {
              put<T, E, TAIL>(a.stream, (T*)a.g_gate + at + c, left, o);
            } else {
#pragma unroll
              for (int e = 0; e < E; ++e)
                if (!TAIL || e < left) ((float*)a.g_gate)[at + c + e] = o[e];
            }
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          q[k][e] = fmaf(db[k][e], y[e] * r1, q[k][e]);
          o[e] = db[k][e] * w[k][e];
          if (a.post_norm) o[e] = r1 * fmaf(-k1, y[e], o[e]);
        }
        if (a.gy) put<T, E, TAIL>(a.stream, (T*)a.gy + at + c, left, o);
      }
    }
    if (!EACH && (a.g_post || a.g_gate)) {
      over_rows<TPR>(q, sums, a.channels, [&](int c, int left, auto& v) {
        constexpr int N = sizeof(v) / sizeof(float);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= keep;
        if (a.g_gate && grid.per > 1) put_sums<N>(part_gate + c, left, v);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (e >= left) break;
          if (a.g_gate && grid.per == 1)
            put_weight(a.g_gate, a.gate_f32, group * a.channels + c + e,
                       a.post_weight ? v[e] * weight_at(a.post_weight, a.post_f32, c + e) : v[e]);
          if (a.gate) v[e] *= weight_at(a.gate, a.gate_f32, group * a.channels + c + e);
          if (a.g_post && group > first) v[e] += part_post[c + e];
        }
        if (a.g_post) put_sums<N>(part_post + c, left, v);
      });
    }
  }
  if (a.g_pre) over_rows<TPR>(g_pre, sums, a.channels, [&](int c, int left, auto& v) { put_sums<sizeof(v) / 4>(part_pre + c, left, v); });
  if (a.g_post && (EACH || first >= grid.groups))
    over_rows<TPR>(q, sums, a.channels, [&](int c, int left, auto& v) {
#pragma unroll
      for (int e = 0; e < (int)(sizeof(v) / 4); ++e) v[e] *= keep;
      put_sums<sizeof(v) / 4>(part_post + c, left, v);
    });
}

constexpr int kSumCols = 16, kShares = 64;  // columns of a workgroup, and shares of the rows that it adds in parallel

// The partial sums of the workgroups, in a fixed order: of pre_weight, of post_weight, and of each group's gate (times
// post_weight), as many of the three as are wanted, one after the other in blockIdx.y.
__global__ void __launch_bounds__(kSumCols * kShares) sandwich_sums_kernel(SandwichBwdArgs a, SandwichGrid grid) {
  __shared__ float red[kShares][kSumCols];
  const int lane = (int)threadIdx.x % kSumCols, share = (int)threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lane;
  int what = (int)blockIdx.y;
  const float* part = a.part;
  int32_t count = grid.blocks;
  void* out = nullptr;
  bool f32 = false;
  if (a.g_pre) {
    if (what == 0) out = a.g_pre, f32 = a.pre_f32;
    --what;
    if (!out) part += (int64_t)grid.blocks * a.channels;
  }
  if (!out && a.g_post) {
    if (what == 0) out = a.g_post, f32 = a.post_f32;
    --what;
    if (!out) part += (int64_t)grid.blocks * a.channels;
  }
  float weight = 1.f;
  if (!out) {  // group `what`
    out = a.g_gate, f32 = a.gate_f32;
    count = grid.per;
    part += (int64_t)what * grid.per * a.channels;
    if (a.post_weight && c < a.channels) weight = weight_at(a.post_weight, a.post_f32, c);
  } else {
    what = 0;
  }
  float s = 0.f;
  if (c < a.channels) {
#pragma unroll 8
    for (int b = share; b < count; b += kShares) s += part[(int64_t)b * a.channels + c];
  }
  red[share][lane] = s;
  __syncthreads();
  if (share < 8) {
#pragma unroll
    for (int k = 8; k < kShares; k += 8) s += red[share + k][lane];
  }
  __syncthreads();
  if (share < 8) red[share][lane] = s;
  __syncthreads();
  if (share != 0 || c >= a.channels) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) s += red[k][lane];
  put_weight(out, f32, (int64_t)what * a.channels + c, s * weight);
}

// The instance of the backward pass for `n` vectors of E elements: few vectors a thread, as each costs 50 registers. us with one and
// with two vectors a thread: 40,968 x 768 bf16 97 and 115, 2,562 x 1,283 float32 29 and 41, 4,096 x 8,192 bf16 99 and 140,
// 4,096 x 4,096 float32 87 and 111.
template <int E, typename F>
hipError_t choose_bwd(int n, F&& f) {
  if (n <= 16) return f.template operator()<16, 1>();
  if (n <= 32) return f.template operator()<32, 1>();
  if (n <= 64) return f.template operator()<64, 1>();
  if (n <= 128) return f.template operator()<128, 1>();
  if (n <= 256) return f.template operator()<256, 1>();
  if (n <= 512) return f.template operator()<512, 1>();
  if (n <= 1024) return f.template operator()<1024, 1>();
  if (n <= 2048) return f.template operator()<1024, 2>();
  if constexpr (E == 4) {
    if (n <= 4096) return f.template operator()<1024, 4>();
  }
  return hipErrorInvalidValue;
}

// Of the forward pass, which needs fewer: long rows with two vectors a thread have fewer waves to wait for at their sums. us with one
// and with two: 5,124 x 4,096 bf16 44.6 and 43, 4,096 x 8,192 bf16 81 and 66, 2,562 x 1,283 float32 19 and 16.5; 40,962 x 768 bf16 57.5
// and 59, 15,000 x 2,048 47 and 50.
template <int E, typename F>
hipError_t choose_fwd(int n, F&& f) {
  if (n <= 16) return f.template operator()<16, 1>();
  if (n <= 32) return f.template operator()<32, 1>();
  if (n <= 64) return f.template operator()<64, 1>();
  if (n <= 128) return f.template operator()<128, 1>();
  if (n <= 256) return f.template operator()<256, 1>();
  if (n <= 512) return f.template operator()<256, 2>();
  if (n <= 1024) return f.template operator()<512, 2>();
  if (n <= 2048) return f.template operator()<1024, 2>();
  if constexpr (E == 4) {
    if (n <= 4096) return f.template operator()<1024, 4>();
  }
  return hipErrorInvalidValue;
}

template <typename T, bool TAIL>
struct Forward {
  const SandwichArgs& a;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    constexpr int RPW = kThreads<TPR> / TPR;
    const int64_t blocks = (a.rows + RPW - 1) / RPW;
    hipLaunchKernelGGL((sandwich_kernel<T, TPR, VPT, TAIL>), dim3((unsigned)(blocks < kMostBlocks ? blocks : kMostBlocks)),
                       dim3(kThreads<TPR>), 0, stream, a);
    return hipGetLastError();
  }
};

template <typename T, bool EACH, bool TAIL>
struct Backward {
  const SandwichBwdArgs& a;
  const SandwichGrid& grid;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    hipLaunchKernelGGL((sandwich_bwd_kernel<T, TPR, VPT, EACH, TAIL>), dim3((unsigned)grid.blocks), dim3(kThreads<TPR>), 0, stream, a,
                       grid);
    return hipGetLastError();
  }
};

template <typename T>
hipError_t forward_as(const SandwichArgs& a, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int n = (a.channels + E - 1) / E;
  return a.channels % E ? choose_fwd<E>(n, Forward<T, true>{a, stream}) : choose_fwd<E>(n, Forward<T, false>{a, stream});
}

template <typename T, bool EACH>
hipError_t backward_as(const SandwichBwdArgs& a, const SandwichGrid& grid, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int n = (a.channels + E - 1) / E;
  return a.channels % E ? choose_bwd<E>(n, Backward<T, EACH, true>{a, grid, stream})
                        : choose_bwd<E>(n, Backward<T, EACH, false>{a, grid, stream});
}

}  // namespace

hipError_t launch_sandwich(int dtype, const SandwichArgs& args, hipStream_t stream) {
  SandwichArgs a = args;
  a.stream = 2 * (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  return dtype == FWN_F32 ? forward_as<float>(a, stream) : forward_as<uint16_t>(a, stream);
}

// As many workgroups as the chip holds at once, 1,024 threads a CU, with four rows each at least (32 where rows share waves), as
// each leaves its partial sums. Backward pass and sums with that many and with 1,024 of any size: 5,124 x 4,096 bf16 71 and 7 us,
// 78 and 12; 4,096 x 8,192 99 and 10, 127 and 31.
constexpr int64_t kCus = 256;
SandwichGrid sandwich_grid(int64_t rows, int64_t gate_rows, int32_t channels, int32_t dtype) {
  SandwichGrid g;
  const int n = (channels * (dtype == FWN_F32 ? 4 : 2) + 15) / 16, threads = n <= 256 ? 256 : n <= 512 ? 512 : 1024;
  const int64_t most = kCus * 1024 / threads, least = n <= 32 ? 32 : 4;
  g.group_rows = gate_rows > 1 ? gate_rows : rows;
  g.groups = g.group_rows > 0 ? rows / g.group_rows : 0;
  const int64_t want = (g.group_rows + least - 1) / least, room = g.groups < most ? most / (g.groups > 0 ? g.groups : 1) : 1;
  g.per = (int32_t)(want < 1 ? 1 : want < room ? want : room);
  g.of_block = (int32_t)(g.per > 1 ? 1 : (g.groups + most - 1) / most);
  if (g.of_block < 1) g.of_block = 1;
  g.blocks = (int32_t)(g.per > 1 ? g.groups * g.per : (g.groups + g.of_block - 1) / g.of_block);
  if (g.blocks < 1) g.blocks = 1;
  g.parts = 2 + (gate_rows > 1 && g.per > 1);
  return g;
}

hipError_t launch_sandwich_bwd(int dtype, const SandwichBwdArgs& args, hipStream_t stream) {
  SandwichBwdArgs a = args;
  a.stream = 2 * (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  const bool each = a.gate && a.gate_rows == 1;
  SandwichGrid grid = sandwich_grid(a.rows, a.gate ? a.gate_rows : a.rows, a.channels, dtype);
  const bool gates = a.g_gate && !each && grid.per > 1;
  grid.parts = (a.g_pre != nullptr) + (a.g_post != nullptr) + gates;
  hipError_t rc;
  if (dtype == FWN_F32)
    rc = each ? backward_as<float, true>(a, grid, stream) : backward_as<float, false>(a, grid, stream);
  else
    rc = each ? backward_as<uint16_t, true>(a, grid, stream) : backward_as<uint16_t, false>(a, grid, stream);
  if (rc != hipSuccess || grid.parts == 0) return rc;
  const unsigned roles = (unsigned)((a.g_pre != nullptr) + (a.g_post != nullptr) + (gates ? grid.groups : 0));
  hipLaunchKernelGGL(sandwich_sums_kernel, dim3((unsigned)((a.channels + kSumCols - 1) / kSumCols), roles),
                     dim3(kSumCols * kShares), 0, stream, a, grid);
  return hipGetLastError();
}

}  // namespace fwn
