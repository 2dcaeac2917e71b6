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
#include "dropout_device.h"

#include "fwn_attn.h"
#include "linear_act.h"

namespace fwn {
namespace {

template <typename T>
struct Bits {
  typedef uint16_t type;
};
template <>
struct Bits<float> {
  typedef uint32_t type;
};

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

template <typename T, int E, bool TAIL>
__device__ __forceinline__ void times(const void* w, bool f32, int64_t at, int left, float (&f)[E]) {
  if (!w) return;
  float g[E];
  load_weight<T, E, TAIL>(w, f32, at, left, g);
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
    float f[VPT][E], b[VPT][E];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] = b[k][e] = 0.f;
      if (!ok || c >= a.channels) continue;
      load<T, E, true, TAIL>(y + c, a.channels - c, b[k]);
      load<T, E, true, TAIL>(x + c, a.channels - c, f[k]);
    }
    float r = 1.f;
    if (a.post_norm) {
      float sq = 0.f;
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) sq = fmaf(b[k][e], b[k][e], sq);
      r = 1.f / sqrtf(row_sum<TPR>(sq, red) * inv_c + a.eps);
    }
    const int64_t gate_at = a.gate && ok ? gate_row(row, a.gate_rows, a.rows) * a.channels : 0;
    float sq = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      if (!ok || c >= a.channels) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) b[k][e] *= r;
      times<T, E, TAIL>(a.gate, a.gate_f32, gate_at + c, a.channels - c, b[k]);
      times<T, E, TAIL>(a.post_weight, a.post_f32, c, a.channels - c, b[k]);
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
      for (int e = 0; e < E; ++e) sq = fmaf(f[k][e], f[k][e], sq);
    }
    r = 1.f / sqrtf(row_sum<TPR>(sq, red) * inv_c + a.eps);
    if (!ok) continue;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
      const int c = (t + TPR * k) * E;
      if (c >= a.channels) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) f[k][e] *= r;
      times<T, E, TAIL>(a.pre_weight, a.pre_f32, c, a.channels - c, f[k]);
      put<T, E, TAIL>(a.stream, (T*)a.out + row * a.channels + c, a.channels - c, f[k]);
    }
  }
}

// Adds the sums that the workgroup's threads hold over the rows that it holds at once, in a fixed order, and hands
// each to its channel's thread: give(channel, value).
template <int TPR, int VPT, int E, typename Give>
__device__ __forceinline__ void over_rows(const float (&v)[VPT][E], float* sums, int channels, const Give& give) {
  constexpr int RPW = kThreads<TPR> / TPR;
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  if constexpr (RPW == 1) {
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (t + TPR * k) * E + e;
        if (c < channels) give(c, v[k][e]);
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
    for (int c = threadIdx.x; c < channels; c += kThreads<TPR>) give(c, sums[c]);
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

// A vector as it lies in memory; with TAIL its first `left` elements, and zeros.
template <typename T, int E, bool TAIL>
__device__ __forceinline__ u32x4 take(const T* p, int left) {
  if (TAIL && left < E) {
    u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) v[e * (int)sizeof(T) / 4] |= (uint32_t)((const typename Bits<T>::type*)p)[e] << 8 * (e * (int)sizeof(T) % 4);
    return v;
  }
  return load_raw<T, true>(p);
}

// SUMS: the gate's gradient is summed over rows. The sums of a workgroup's rows stay in its threads' registers; those of
// the gate are handed on at the end of each group of rows.
template <typename T, int TPR, int VPT, bool SUMS, bool TAIL>
__global__ void __launch_bounds__(kThreads<TPR>) sandwich_bwd_kernel(SandwichBwdArgs a, SandwichGrid grid) {
  constexpr int E = 16 / sizeof(T), RPW = kThreads<TPR> / TPR;
  __shared__ float red[32];
  __shared__ float sums[RPW > 1 ? TPR * VPT * E : 1];
  const int t = (int)threadIdx.x % TPR, own = (int)threadIdx.x / TPR;
  const float inv_c = 1.f / (float)a.channels;
  const Draw draw(a.draw);
  float g_pre[VPT][E], g_post[VPT][E], g_gate[SUMS ? VPT : 1][E];
#pragma unroll
  for (int k = 0; k < VPT; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) g_pre[k][e] = g_post[k][e] = 0.f;
  const int64_t first = (int64_t)((int)blockIdx.x / grid.per) * grid.of_block;
  const int sub = (int)blockIdx.x % grid.per;
  for (int64_t group = first; group < first + grid.of_block && group < grid.groups; ++group) {
    if constexpr (SUMS) {
#pragma unroll
      for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) g_gate[k][e] = 0.f;
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
        vs[k] = take<T, E, TAIL>((const T*)a.s + at + c, left);
        if (a.g_out) vo[k] = take<T, E, TAIL>((const T*)a.g_out + at + c, left);
        if (a.g_sum) vg[k] = take<T, E, TAIL>((const T*)a.g_sum + at + c, left);
        vy[k] = take<T, E, TAIL>((const T*)a.y + row * a.y_stride + c, left);
      }
      float r2 = 0.f, k2 = 0.f;
      if (a.g_out) {
        float sq = 0.f, as = 0.f;  // of s^2, and of a s
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
          const int c = (t + TPR * k) * E;
          float s[E], h[E];
          unpack<T>(vs[k], s);
          unpack<T>(vo[k], h);
          if (ok && c < a.channels) times<T, E, TAIL>(a.pre_weight, a.pre_f32, c, a.channels - c, h);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            sq = fmaf(s[e], s[e], sq);
            as = fmaf(h[e], s[e], as);
          }
        }
        row_sums<TPR>(sq, as, red);
        r2 = 1.f / sqrtf(sq * inv_c + a.eps);
        k2 = as * inv_c * r2 * r2;
      }
      const int64_t gate_at = a.gate && ok ? gate_row(row, a.gate_rows, a.rows) * a.channels : 0;
      float db[VPT][E], yy = 0.f, cy = 0.f;  // of y^2, and of c y
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E, left = a.channels - c;
#pragma unroll
        for (int e = 0; e < E; ++e) db[k][e] = 0.f;
        if (!ok || left <= 0) continue;
        float ds[E];
        unpack<T>(vg[k], ds);
        if (a.g_out) {
          float s[E], h[E];
          unpack<T>(vs[k], s);
          unpack<T>(vo[k], h);
#pragma unroll
          for (int e = 0; e < E; ++e) g_pre[k][e] = fmaf(h[e], s[e] * r2, g_pre[k][e]);
          times<T, E, TAIL>(a.pre_weight, a.pre_f32, c, left, h);
#pragma unroll
          for (int e = 0; e < E; ++e) ds[e] = fmaf(r2, h[e] - s[e] * k2, ds[e]);
        }
        if (a.gx) {
          float o[E];
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = a.scale * ds[e];
          put<T, E, TAIL>(a.stream, (T*)a.gx + at + c, left, o);
        }
        if (a.drop) draw.template apply<E>((uint32_t)row, (uint32_t)c, ds);
#pragma unroll
        for (int e = 0; e < E; ++e) db[k][e] = ds[e];
        if (!a.post_norm) continue;
        float y[E];
        unpack<T>(vy[k], y);
        times<T, E, TAIL>(a.gate, a.gate_f32, gate_at + c, left, ds);
        times<T, E, TAIL>(a.post_weight, a.post_f32, c, left, ds);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          yy = fmaf(y[e], y[e], yy);
          cy = fmaf(ds[e], y[e], cy);
        }
      }
      float r1 = 1.f, k1 = 0.f;
      if (a.post_norm) {
        row_sums<TPR>(yy, cy, red);
        r1 = 1.f / sqrtf(yy * inv_c + a.eps);
        k1 = cy * inv_c * r1 * r1;
      }
      if (!ok) continue;
#pragma unroll
      for (int k = 0; k < VPT; ++k) {
        const int c = (t + TPR * k) * E, left = a.channels - c;
        if (left <= 0) continue;
        float unit[E], d[E], o[E];
        unpack<T>(vy[k], unit);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o[e] = unit[e] * k1;
          unit[e] *= r1;
          d[e] = db[k][e];
        }
        times<T, E, TAIL>(a.gate, a.gate_f32, gate_at + c, left, d);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          g_post[k][e] = fmaf(d[e], unit[e], g_post[k][e]);
          if constexpr (SUMS) g_gate[k][e] = fmaf(db[k][e], unit[e], g_gate[k][e]);
        }
        if (a.gy) {
          times<T, E, TAIL>(a.post_weight, a.post_f32, c, left, d);
          if (a.post_norm) {
#pragma unroll
            for (int e = 0; e < E; ++e) d[e] = r1 * (d[e] - o[e]);
          }
          put<T, E, TAIL>(a.stream, (T*)a.gy + at + c, left, d);
        }
        if (!SUMS && a.g_gate) {
#pragma unroll
          for (int e = 0; e < E; ++e) unit[e] *= db[k][e];
          times<T, E, TAIL>(a.post_weight, a.post_f32, c, left, unit);
          if (sizeof(T) == 4 || !a.gate_f32) {
            put<T, E, TAIL>(a.stream, (T*)a.g_gate + at + c, left, unit);
          } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (!TAIL || e < left) ((float*)a.g_gate)[at + c + e] = unit[e];
          }
        }
      }
    }
    if constexpr (SUMS) {
      float* const part = a.part + ((int64_t)(grid.parts - 1) * grid.blocks + blockIdx.x) * a.channels;
      over_rows<TPR>(g_gate, sums, a.channels, [&](int c, float v) {
        if (grid.per > 1)
          part[c] = v;
        else
          put_weight(a.g_gate, a.gate_f32, group * a.channels + c, a.post_weight ? v * weight_at(a.post_weight, a.post_f32, c) : v);
      });
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.channels;
  if (a.g_pre) {
    over_rows<TPR>(g_pre, sums, a.channels, [&](int c, float v) { part[c] = v; });
    part += (int64_t)grid.blocks * a.channels;
  }
  if (a.g_post) over_rows<TPR>(g_post, sums, a.channels, [&](int c, float v) { part[c] = v; });
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

template <typename T, bool SUMS, bool TAIL>
struct Backward {
  const SandwichBwdArgs& a;
  const SandwichGrid& grid;
  hipStream_t stream;
  template <int TPR, int VPT>
  hipError_t operator()() const {
    hipLaunchKernelGGL((sandwich_bwd_kernel<T, TPR, VPT, SUMS, TAIL>), dim3((unsigned)grid.blocks), dim3(kThreads<TPR>), 0, stream, a,
                       grid);
    return hipGetLastError();
  }
};

template <typename T>
hipError_t forward_as(const SandwichArgs& a, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int n = (a.channels + E - 1) / E;
  return a.channels % E ? choose<E>(n, Forward<T, true>{a, stream}) : choose<E>(n, Forward<T, false>{a, stream});
}

template <typename T, bool SUMS>
hipError_t backward_as(const SandwichBwdArgs& a, const SandwichGrid& grid, hipStream_t stream) {
  constexpr int E = 16 / sizeof(T);
  const int n = (a.channels + E - 1) / E;
  return a.channels % E ? choose<E>(n, Backward<T, SUMS, true>{a, grid, stream})
                        : choose<E>(n, Backward<T, SUMS, false>{a, grid, stream});
}

bool gate_sums(const SandwichBwdArgs& a) { return a.g_gate && a.gate_rows > 1; }

}  // namespace

hipError_t launch_sandwich(int dtype, const SandwichArgs& args, hipStream_t stream) {
  SandwichArgs a = args;
  a.stream = 2 * (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  return dtype == FWN_F32 ? forward_as<float>(a, stream) : forward_as<uint16_t>(a, stream);
}

// At most 1,024 workgroups, four a CU, with eight rows each at least (32 where rows share waves), as each leaves its partial sums.
SandwichGrid sandwich_grid(int64_t rows, int64_t gate_rows, int32_t channels, bool sums) {
  SandwichGrid g;
  constexpr int64_t most = 1024;
  const int64_t least = channels <= 256 ? 32 : 8;
  g.group_rows = sums ? gate_rows : rows;
  g.groups = g.group_rows > 0 ? rows / g.group_rows : 0;
  const int64_t want = (g.group_rows + least - 1) / least, room = g.groups < most ? most / (g.groups > 0 ? g.groups : 1) : 1;
  g.per = (int32_t)(want < 1 ? 1 : want < room ? want : room);
  g.of_block = (int32_t)(g.per > 1 ? 1 : (g.groups + most - 1) / most);
  if (g.of_block < 1) g.of_block = 1;
  g.blocks = (int32_t)(g.per > 1 ? g.groups * g.per : (g.groups + g.of_block - 1) / g.of_block);
  if (g.blocks < 1) g.blocks = 1;
  g.parts = 2 + (sums && g.per > 1);
  return g;
}

hipError_t launch_sandwich_bwd(int dtype, const SandwichBwdArgs& args, hipStream_t stream) {
  SandwichBwdArgs a = args;
  a.stream = 2 * (uint64_t)a.rows * a.channels * (dtype == FWN_F32 ? 4 : 2) >= kStreamBytes;
  const bool sums = gate_sums(a);
  SandwichGrid grid = sandwich_grid(a.rows, a.gate_rows, a.channels, sums);
  const bool gates = sums && grid.per > 1;
  grid.parts = (a.g_pre != nullptr) + (a.g_post != nullptr) + gates;
  hipError_t rc;
  if (dtype == FWN_F32)
    rc = sums ? backward_as<float, true>(a, grid, stream) : backward_as<float, false>(a, grid, stream);
  else
    rc = sums ? backward_as<uint16_t, true>(a, grid, stream) : backward_as<uint16_t, false>(a, grid, stream);
  if (rc != hipSuccess || grid.parts == 0) return rc;
  const unsigned roles = (unsigned)((a.g_pre != nullptr) + (a.g_post != nullptr) + (gates ? grid.groups : 0));
  hipLaunchKernelGGL(sandwich_sums_kernel, dim3((unsigned)((a.channels + kSumCols - 1) / kSumCols), roles),
                     dim3(kSumCols * kShares), 0, stream, a, grid);
  return hipGetLastError();
}

}  // namespace fwn
