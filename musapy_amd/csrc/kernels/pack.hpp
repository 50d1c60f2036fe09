// pack.hpp -- f32, f16 and bf16 vectors as they lie in memory.
//
// Elements that are loaded well before they are used stay packed in 32-bit words and become f32 one by
// one.  (As arrays of 16-bit elements the compiler gives each a register of its own wherever a vector
// comes from two branches, a full load and one of the last elements of a row.)
#pragma once

#include "kcommon.hpp"

namespace mpy {

using bf16 = __bf16;
using f16 = _Float16;

template <class T, int N>
struct Pack {
  static constexpr int kWords = N * int(sizeof(T)) / 4;
  uint32_t w[kWords];
};

template <class T>
__device__ inline uint32_t pack_bits(T v) {
  if constexpr (sizeof(T) == 4) return __builtin_bit_cast(uint32_t, v);
  else return __builtin_bit_cast(uint16_t, v);
}

template <class T, int N>
__device__ inline float pack_get(const Pack<T, N>& p, int e) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, p.w[e]);
  } else if constexpr (std::is_same_v<T, bf16>) {
    return __builtin_bit_cast(float, e % 2 ? p.w[e / 2] & 0xffff0000u : p.w[e / 2] << 16);
  } else {
    return float(__builtin_bit_cast(f16, uint16_t(p.w[e / 2] >> (16 * (e % 2)))));
  }
}

template <class T, int N>
__device__ inline Pack<T, N> pack_all(T v) {
  const uint32_t b = pack_bits(v);
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < p.kWords; ++i) p.w[i] = sizeof(T) == 4 ? b : b | b << 16;
  return p;
}

// N elements from any element address; of fewer than N, `none` in the place of the rest.
template <bool NT, int N, class T>
__device__ inline Pack<T, N> pack_load(const T* at, int n, T none) {
  Pack<T, N> p;
  if (n == N) {
    const Vec<T, N> v = vload_el<T, N, NT>(at);
    __builtin_memcpy(&p, &v, sizeof(p));
    return p;
  }
#pragma unroll
  for (int i = 0; i < p.kWords; ++i) p.w[i] = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const uint32_t b = pack_bits(e < n ? at[e] : none);
    if constexpr (sizeof(T) == 4) p.w[e] = b;
    else p.w[e / 2] |= b << (16 * (e % 2));
  }
  return p;
}

// Of elements that were loaded from `by` elements in front of their place: those from there on, then
// zeros.  The last elements of a row are loaded so, as N in one piece that ends with the row: one by
// one, under a branch, each operand's loads were waited for before the next one's were issued.
template <class T, int N>
__device__ inline void pack_shift(Pack<T, N>& p, int by) {
  if (by == 0) return;
  auto words = [&](int k) {
#pragma unroll
    for (int i = 0; i < p.kWords; ++i) p.w[i] = i + k < p.kWords ? p.w[i + k < p.kWords ? i + k : 0] : 0;
  };
  if constexpr (sizeof(T) == 2) {
    if (by & 1)
#pragma unroll
      for (int i = 0; i < p.kWords; ++i)
        p.w[i] = p.w[i] >> 16 | (i + 1 < p.kWords ? p.w[i + 1 < p.kWords ? i + 1 : 0] << 16 : 0);
    by /= 2;
  }
  if (by & 1) words(1);
  if (by & 2) words(2);
  if constexpr (Pack<T, N>::kWords > 4)
    if (by & 4) words(4);
}

// The first n of N elements, rounded to T, to any element address.
template <bool NT, class T, int N>
__device__ inline void pack_store(T* at, int n, const float (&x)[N]) {
  if (n == N) {
    Vec<T, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = T(x[e]);
    vstore_el<NT, T, N>(at, v);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) at[e] = T(x[e]);
  }
}

// Hides where a value comes from, so that what was computed from it before is formed again instead of
// being kept in registers.
template <class T, int N>
__device__ inline void pack_opaque(Pack<T, N>& p) {
#pragma unroll
  for (int i = 0; i < p.kWords; ++i) asm volatile("" : "+v"(p.w[i]));
}

// s = sigmoid(g) and 1 - s, each with a small relative error: both from exp(-|g|) <= 1, so neither
// is a difference of near numbers.  The hardware's exp2 and reciprocal are within 1 ulp.
__device__ inline void sigmoid_pair(float g, float& s, float& rest) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float er = e * r;
  s = g >= 0.0f ? r : er;      // a NaN gate: both are NaN
  rest = g >= 0.0f ? er : r;
}

}  // namespace mpy
