// Copies of a product's operands into LDS, stage by stage (gfx950).
#pragma once

#include "linear_act_device.h"

namespace fwn {
namespace {

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

// This wave's copies have landed and its LDS reads have returned, and so have every other wave's.
__device__ __forceinline__ void stage_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace
}  // namespace fwn
