// gated_scan.hpp -- the gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis, and its
// gradient: what the forward (gated_scan.hip) and backward (gated_scan_grad.hip) kernels share.
//
// Gradient: with c[t] what flows into h[t-1],
//   G[t] = dh[t] + c[t+1],  c[t] = a[t] G[t],  c[T] = dlast,
// which is the same recurrence run over reversed time, with (a[t], a[t] dh[t]) for (a, b).
#pragma once

#include "kcommon.hpp"

namespace mpy {

using bf16 = __bf16;
using f16 = _Float16;

constexpr int kGsBlock = 256;

// Operands, and their places in the strides.  kGsState is first / last / dlast: x's shape without
// the scanned axis.
enum GsOperand { kGsX, kGsGate, kGsReset, kGsOut, kGsState, kGsH, kGsDh, kGsDgate, kGsOps };

struct GsArgs {
  RowIndexer<kGsOps> ix;     // the rows: coalesced non-axis dims but the innermost
  int64_t ts[kGsOps];        // strides along the scanned axis
  int64_t ls[kGsOps];        // strides along the lanes (the innermost non-axis dim)
  uint64_t T;                // steps
  uint32_t D;                // lanes of a row
  uint32_t nv;               // vectors of a row: ceil(D / V)
  uint32_t nvec;             // vectors in all
  FastDiv nvdiv;             // divides a vector's number by nv
  const void* x;
  const void* gate;
  const uint8_t* reset;
  const void* h;
  const void* dh;
  const float* first;        // carried in: first (forward), dlast (gradient)
  const float* h_first;      // gradient: the forward's first
  void* out;
  void* dgate;
  float* last;               // carried out
  bool dgate_f32;            // dgate is stored as f32 whatever the gate's type
  int part_lanes;            // lanes that share one dgate partial sum: log2 of the vectors; < 0: no sums
};

// s = sigmoid(g) and 1 - s, each with a small relative error: both from exp(-|g|) <= 1, so neither
// is a difference of near numbers.  The hardware's exp2 and reciprocal are within 1 ulp.
__device__ inline void gs_sigmoid(float g, float& s, float& rest) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float er = e * r;
  s = g >= 0.0f ? r : er;      // a NaN gate: both are NaN
  rest = g >= 0.0f ? er : r;
}

// V consecutive lanes as f32: from a vector, from one shared element (lane stride 0), or element by
// element (the last lanes of a row).
template <class T, int V>
__device__ inline void gs_load(const T* p, int64_t ls, int nl, float (&o)[V]) {
  if constexpr (V == 1) {
    o[0] = float(*p);
  } else if (ls == 0) {
    const float e = float(*p);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = e;
  } else if (nl == V) {
    const Vec<T, V> w = vload_el<T, V, false>(p);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = float(w.v[v]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = v < nl ? float(p[v]) : 0.0f;
  }
}
template <class T, int V>
__device__ inline void gs_store(T* p, int nl, const float (&x)[V]) {
  if (nl == V) {
    Vec<T, V> w;
#pragma unroll
    for (int v = 0; v < V; ++v) w.v[v] = T(x[v]);
    vstore_el<false, T, V>(p, w);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nl) p[v] = T(x[v]);
  }
}

// ---- host side ----------------------------------------------------------------------------------
struct GsPlan {
  GsArgs a;
  uint64_t rows;  // rows of D lanes
  bool lanes;     // the lanes are unit-stride (gate: or shared), resets shared by the lanes
};

// Checks and normalises a call; false with the wrapper error set when an argument is out of range.
// Empty calls (no lanes) come back with rows or D equal to 0.
bool gs_plan(const musapy_gated_scan_args* p, bool grad, GsPlan& out);
// Splits the lanes into vectors of V.
void gs_vectors(GsPlan& pl, int V);

inline int gs_vector(int dtype) { return dtype == MUSAPY_DT_F32 ? 4 : 8; }  // 16 bytes of x

// The largest power of two of vectors, up to 8, that divides a row of vectors: neighbouring
// threads that sum a shared gate's gradient before it is stored.
inline int gs_part_shift(uint64_t D, int V) {
  const uint64_t nv = (D + V - 1) / V;
  int s = 0;
  while (s < 3 && nv % (uint64_t(2) << s) == 0) ++s;
  return s;
}

// Calls fn(TX{}, TG{}) with the element types of x and the gate.
template <class Fn>
inline void gs_types(int dtype, int gate_dtype, Fn&& fn) {
  if (dtype == MUSAPY_DT_F32) return fn(float{}, float{});
  if (dtype == MUSAPY_DT_BF16) {
    if (gate_dtype == MUSAPY_DT_F32) return fn(bf16{}, float{});
    return fn(bf16{}, bf16{});
  }
  if (gate_dtype == MUSAPY_DT_F32) return fn(f16{}, float{});
  return fn(f16{}, f16{});
}

}  // namespace mpy
