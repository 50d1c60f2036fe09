// gated_scan_grad.hip -- the gated scan's gradient kernels, for gfx950.
#include "gated_scan.hpp"

namespace mpy {

// One thread per V lanes, from the last step to the first; V = 1 takes any strides.
template <class TX, class TG, bool BLEND, int V>
__global__ __launch_bounds__(kGsBlock) void k_gs_grad_walk(GsArgs p) {
  const uint64_t q = uint64_t(blockIdx.x) * kGsBlock + threadIdx.x;
  // threads past the last vector stay for the sums between neighbours
  const bool on = q < p.nvec;
  const uint32_t row = fd_div(p.nvdiv, on ? uint32_t(q) : 0);
  const uint32_t vec = on ? uint32_t(q) - row * p.nv : 0;
  const uint32_t col = vec * V;
  const int nl = !on ? 0 : p.D - col < uint32_t(V) ? int(p.D - col) : V;
  int64_t off[kGsOps];
  row_offsets<kGsOps>(p.ix, row, off);
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
  float c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = p.first && v < nl ? p.first[off[kGsState] + v] : 0.0f;
  for (uint64_t k = 0; k < p.T; ++k) {
    const int64_t t = int64_t(p.T - 1 - k);
    float dh[V], g[V], hb[V], x[V], dg[V], dx[V];
#pragma unroll
    for (int v = 0; v < V; ++v) dh[v] = g[v] = hb[v] = x[v] = 0.0f;
    bool cut = false;
    if (on) {
      gs_load<TX, V>(static_cast<const TX*>(p.dh) + off[kGsDh] + t * p.ts[kGsDh], p.ls[kGsDh], nl, dh);
      gs_load<TG, V>(static_cast<const TG*>(p.gate) + off[kGsGate] + t * p.ts[kGsGate], p.ls[kGsGate], nl, g);
      if constexpr (BLEND)
        gs_load<TX, V>(static_cast<const TX*>(p.x) + off[kGsX] + t * p.ts[kGsX], p.ls[kGsX], nl, x);
      cut = p.reset && p.reset[off[kGsReset] + t * p.ts[kGsReset]];
      if (!cut) {
        if (t > 0)
          gs_load<TX, V>(static_cast<const TX*>(p.h) + off[kGsH] + (t - 1) * p.ts[kGsH], p.ls[kGsH], nl, hb);
        else if (p.h_first)
#pragma unroll
          for (int v = 0; v < V; ++v) hb[v] = v < nl ? p.h_first[off[kGsState] + v] : 0.0f;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float G = dh[v] + c[v];
      if constexpr (BLEND) {
        float s, rest;
        gs_sigmoid(g[v], s, rest);
        dx[v] = rest * G;
        dg[v] = G * (hb[v] - x[v]) * (s * rest);
        c[v] = cut ? 0.0f : s * G;
      } else {
        dx[v] = G;
        dg[v] = cut ? 0.0f : G * hb[v];
        c[v] = cut ? 0.0f : g[v] * G;
      }
    }
    if (on) gs_store<TX, V>(static_cast<TX*>(p.out) + off[kGsOut] + t * p.ts[kGsOut], nl, dx);
    if (p.part_lanes >= 0) {
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) sum += v < nl ? dg[v] : 0.0f;
      for (int m = 1; m < (1 << p.part_lanes); m <<= 1) sum += __shfl_xor(sum, m, kWave);
      if (on && (vec & ((1u << p.part_lanes) - 1)) == 0)
        static_cast<float*>(p.dgate)[off[kGsDgate] + t * p.ts[kGsDgate] + (vec >> p.part_lanes)] = sum;
    } else if (on) {
      const int64_t at = off[kGsDgate] + t * p.ts[kGsDgate];
      if (p.dgate_f32) gs_store<float, V>(static_cast<float*>(p.dgate) + at, nl, dg);
      else gs_store<TG, V>(static_cast<TG*>(p.dgate) + at, nl, dg);
    }
  }
  if (p.last) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nl) p.last[off[kGsState] + v] = c[v];
  }
}

}  // namespace mpy

using namespace mpy;

extern "C" {

int musapy_gated_scan_grad_v1(const musapy_gated_scan_args* p, void* scratch, size_t scratch_bytes, void* workspace,
                              size_t workspace_bytes, hipStream_t st) {
  GsPlan pl;
  if (!gs_plan(p, true, pl)) return -1;
  if (pl.rows == 0 || pl.a.D == 0) return 0;
  const int V = pl.lanes ? gs_vector(p->dtype) : 1;
  gs_vectors(pl, V);
  const unsigned grid = unsigned((uint64_t(pl.a.nvec) + kGsBlock - 1) / kGsBlock);
  gs_types(p->dtype, p->gate_dtype, [&](auto tx, auto tg) {
    using TX = decltype(tx);
    using TG = decltype(tg);
    constexpr int kV = 16 / int(sizeof(TX));
    if (p->kind == MUSAPY_SCAN_BLEND) {
      if (V == 1) k_gs_grad_walk<TX, TG, true, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_grad_walk<TX, TG, true, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    } else {
      if (V == 1) k_gs_grad_walk<TX, TG, false, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_grad_walk<TX, TG, false, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    }
  });
  return 0;
}

}  // extern "C"
