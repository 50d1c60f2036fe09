// vocab.hpp -- what the kernels over a vocabulary share: token numbers, runtime dtypes, sums over a
// workgroup.
#pragma once

#include "kcommon.hpp"
#include "pack.hpp"

namespace mpy {

// Token numbers as a caller holds them, 32 or 64 bits wide.
struct Ids {
  const void* at;
  int wide;
};

// A number as it was loaded, and the number: `none` where it is outside [0, none).  What is loaded under a branch and used
// there is waited for there, with every load in front of it; so loads that are to be under way together come first, their uses after.
struct RawId {
  uint32_t low, high;
};
__device__ inline RawId id_load(const Ids& ids, uint64_t i) {
  RawId r;
  if (ids.wide) {
    const uint2 v = static_cast<const uint2*>(ids.at)[i];
    r.low = v.x;
    r.high = v.y;
  } else {
    r.low = static_cast<const uint32_t*>(ids.at)[i];
    r.high = 0;
  }
  return r;
}
__device__ inline uint32_t id_of(const RawId& r, uint32_t none) { return r.high == 0 && r.low < none ? r.low : none; }
__device__ inline uint32_t id_at(const Ids& ids, uint64_t i, uint32_t none) { return id_of(id_load(ids, i), none); }

inline bool vocab_float(int dtype) {
  return dtype == MUSAPY_DT_F32 || dtype == MUSAPY_DT_BF16 || dtype == MUSAPY_DT_F16;
}
inline bool vocab_id(int dtype) { return dtype == MUSAPY_DT_I32 || dtype == MUSAPY_DT_I64; }
inline Ids vocab_ids(const void* at, int dtype) { return Ids{at, dtype == MUSAPY_DT_I64}; }

// Rows and columns are numbered in 31 bits.
constexpr uint64_t kVocabLimit = uint64_t(1) << 31;

inline int vocab_bad(int code = 6) {
  g_wrapper_error = code;
  return -1;
}

// Calls fn with a value of the element type.
template <class F>
inline void vocab_type(int dtype, F&& fn) {
  if (dtype == MUSAPY_DT_F32) fn(float(0));
  else if (dtype == MUSAPY_DT_BF16) fn(bf16(0));
  else fn(f16(0));
}

// The same for elements of a runtime dtype.
__device__ inline uint32_t float_load(const void* at, int dtype, uint64_t i) {
  uint32_t bits;
  if (dtype == MUSAPY_DT_F32) bits = static_cast<const uint32_t*>(at)[i];
  else bits = static_cast<const uint16_t*>(at)[i];
  return bits;
}
__device__ inline float float_of(uint32_t bits, int dtype) {
  if (dtype == MUSAPY_DT_F32) return __builtin_bit_cast(float, bits);
  if (dtype == MUSAPY_DT_BF16) return __builtin_bit_cast(float, bits << 16);
  return float(__builtin_bit_cast(f16, uint16_t(bits)));
}
__device__ inline float float_at(const void* at, int dtype, uint64_t i) { return float_of(float_load(at, dtype, i), dtype); }

__device__ inline uint32_t wave_uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }

__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}
__device__ inline float wave_max(float v) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, kWave));
  return v;
}

}  // namespace mpy
