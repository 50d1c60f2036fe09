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

// The number, or `none` where it is outside [0, none).
__device__ inline uint32_t id_at(const Ids& ids, uint64_t i, uint32_t none) {
  if (ids.wide) {
    const uint64_t v = static_cast<const uint64_t*>(ids.at)[i];
    return v < none ? uint32_t(v) : none;
  }
  const uint32_t v = static_cast<const uint32_t*>(ids.at)[i];
  return v < none ? v : none;
}

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

__device__ inline float float_at(const void* at, int dtype, uint64_t i) {
  if (dtype == MUSAPY_DT_F32) return static_cast<const float*>(at)[i];
  if (dtype == MUSAPY_DT_BF16) return float(static_cast<const bf16*>(at)[i]);
  return float(static_cast<const f16*>(at)[i]);
}

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
