// Dropout's random numbers (gfx950): which of a row's channels are kept, from a counter and nothing stored.
#pragma once

#include "dropout.h"
#include "rms_device.h"

namespace fwn {
namespace {

// One instruction where the compiler makes two of ^ (40,968 x 768 bf16, backward of the norms around a block with dropout: 87 us, with ^ 96).
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
  return (uint32_t)__builtin_amdgcn_bitop3_b32((int)a, (int)b, (int)c, 0x96);
}

// The state of a launch: of its arguments, or as the GPU's memory holds it when the kernel runs.
struct Draw {
  uint32_t key[2], offset[2];
  uint32_t border;
  float keep;

  __device__ __forceinline__ explicit Draw(const DropoutArgs& d) : border(d.border), keep(d.keep) {
    const uint64_t seed = d.state ? d.state[0] : d.seed, at = d.state ? d.state[1] : d.offset;
    key[0] = (uint32_t)seed;
    key[1] = (uint32_t)(seed >> 32);
    offset[0] = (uint32_t)at;
    offset[1] = (uint32_t)(at >> 32);
  }

  // Philox-4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) of the counter (eight,
  // row, offset): 4 words whose 8 halves belong to the channels 8 eight .. 8 eight + 7 of the row, the low half first.
  // Sixteen bits a channel rather than 32: p is taken to the nearest 2^-16, for half of the rounds. A block of ten rounds is
  // 20 multiplications of 32 x 32 bits, a quarter of the other instructions' rate each.
  __device__ __forceinline__ void block(uint32_t row, uint32_t eight, uint32_t (&c)[4]) const {
    uint32_t k0 = key[0], k1 = key[1];
    c[0] = eight, c[1] = row, c[2] = offset[0], c[3] = offset[1];
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const uint64_t a = (uint64_t)c[0] * 0xD2511F53u, b = (uint64_t)c[2] * 0xCD9E8D57u;
      c[0] = xor3((uint32_t)(b >> 32), c[1], k0);
      c[1] = (uint32_t)b;
      c[2] = xor3((uint32_t)(a >> 32), c[3], k1);
      c[3] = (uint32_t)a;
      k0 += 0x9E3779B9u;
      k1 += 0xBB67AE85u;
    }
  }

  // f of the channels col .. col + E - 1 (a vector of the row: col is a multiple of E): itself, or zero whatever it was.
  template <int E>
  __device__ __forceinline__ void select(uint32_t row, uint32_t col, float (&f)[E]) const {
    uint32_t c[4];
    block(row, col / 8, c);
    // A vector of four has one half of the words, chosen by value (an index that varies would put them into memory).
    const uint32_t w[4] = {E == 4 && (col & 4) ? c[2] : c[0], E == 4 && (col & 4) ? c[3] : c[1], c[2], c[3]};
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      f[e] = (w[e / 2] & 0xffffu) >= border ? f[e] : 0.f;
      f[e + 1] = (w[e / 2] >> 16) >= border ? f[e + 1] : 0.f;
    }
  }

  // The same times `keep`.
  template <int E>
  __device__ __forceinline__ void apply(uint32_t row, uint32_t col, float (&f)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= keep;
    select(row, col, f);
  }
};

}  // namespace
}  // namespace fwn
