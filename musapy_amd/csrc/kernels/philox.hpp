// philox.hpp -- counter-based random numbers: Philox4x32-10.
//
// The generator is the published one (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds over a 128-bit counter, each multiplying two of its words by
// constants into 64 bits and mixing the halves with the other two and a key that grows by a constant
// a round.  Any counter can be evaluated by itself, so a dropout mask is formed where it is needed,
// in the forward pass and again in the backward one, and never stored.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mpy {

struct PhiloxKey {
  uint32_t k0, k1;  // seed low, high
  uint32_t c2, c3;  // offset low, high
};
inline PhiloxKey philox_key(uint64_t seed, uint64_t offset) {
  return PhiloxKey{uint32_t(seed), uint32_t(seed >> 32), uint32_t(offset), uint32_t(offset >> 32)};
}

__device__ inline uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) { return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96); }

// The four words of the counter (c0, c1, c2, c3).  The 64-bit products are one v_mad_u64_u32 each,
// and the mixing one three-operand v_bitop3 each; the keys are the same for all lanes and stay in
// scalar registers.
__device__ inline void philox(const PhiloxKey& key, uint32_t c0, uint32_t c1, uint32_t (&w)[4]) {
  uint32_t c2 = key.c2, c3 = key.c3, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p = uint64_t(c0) * 0xD2511F53u, q = uint64_t(c2) * 0xCD9E8D57u;
    c0 = xor3(uint32_t(q >> 32), c1, k0);
    c1 = uint32_t(q);
    c2 = xor3(uint32_t(p >> 32), c3, k1);
    c3 = uint32_t(p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0;
  w[1] = c1;
  w[2] = c2;
  w[3] = c3;
}

// The eight 16-bit numbers of columns 8 c8 .. 8 c8 + 7 of a row, as a bit mask of those to keep: 16
// bits an element halve the generator's work, and hold a drop rate to 2^-17.
__device__ inline uint32_t philox_keep8(const PhiloxKey& key, uint32_t c8, uint32_t row, uint32_t threshold) {
  uint32_t w[4];
  philox(key, c8, row, w);
  uint32_t keep = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    keep |= uint32_t((w[i] & 0xffffu) >= threshold) << (2 * i);
    keep |= uint32_t((w[i] >> 16) >= threshold) << (2 * i + 1);
  }
  return keep;
}

inline float dropout_scale(uint32_t threshold) {
  return threshold >= 65536u ? 0.0f : float(65536.0 / double(65536u - threshold));
}

}  // namespace mpy
