// gated_scan.hip -- the gated scan's forward kernels and the planning of both directions, for gfx950.
#include "gated_scan.hpp"

namespace mpy {

// One thread per V lanes, one step after the other; V = 1 takes any strides.
template <class TX, class TG, bool BLEND, int V>
__global__ __launch_bounds__(kGsBlock) void k_gs_walk(GsArgs p) {
  const uint64_t q = uint64_t(blockIdx.x) * kGsBlock + threadIdx.x;
  if (q >= p.nvec) return;
  const uint32_t row = fd_div(p.nvdiv, uint32_t(q));
  const uint32_t col = (uint32_t(q) - row * p.nv) * V;
  const int nl = p.D - col < uint32_t(V) ? int(p.D - col) : V;
  int64_t off[kGsOps];
  row_offsets<kGsOps>(p.ix, row, off);
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
  const TX* x = static_cast<const TX*>(p.x) + off[kGsX];
  const TG* gate = static_cast<const TG*>(p.gate) + off[kGsGate];
  const uint8_t* reset = p.reset ? p.reset + off[kGsReset] : nullptr;
  TX* out = static_cast<TX*>(p.out) + off[kGsOut];
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = p.first && v < nl ? p.first[off[kGsState] + v] : 0.0f;
  for (uint64_t t = 0; t < p.T; ++t) {
    float b[V], g[V];
    gs_load<TX, V>(x, p.ls[kGsX], nl, b);
    gs_load<TG, V>(gate, p.ls[kGsGate], nl, g);
    const bool cut = reset && *reset;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = g[v], in = b[v];
      if constexpr (BLEND) {
        float rest;
        gs_sigmoid(g[v], a, rest);
        in = rest * b[v];
      }
      h[v] = cut ? in : __builtin_fmaf(a, h[v], in);
    }
    gs_store<TX, V>(out, nl, h);
    x += p.ts[kGsX];
    gate += p.ts[kGsGate];
    out += p.ts[kGsOut];
    if (reset) reset += p.ts[kGsReset];
  }
  if (p.last) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nl) p.last[off[kGsState] + v] = h[v];
  }
}

// ---- planning -------------------------------------------------------------------------------------
namespace {
bool gs_bad() {
  g_wrapper_error = 6;
  return false;
}
bool gs_dtype(int d) { return d == MUSAPY_DT_F32 || d == MUSAPY_DT_F16 || d == MUSAPY_DT_BF16; }
}  // namespace

bool gs_plan(const musapy_gated_scan_args* p, bool grad, GsPlan& out) {
  if (p == nullptr) return gs_bad();
  if (p->ndim < 1 || p->ndim > kMaxDims || p->axis < 0 || p->axis >= p->ndim) {
    g_wrapper_error = 3;
    return false;
  }
  const bool blend = p->kind == MUSAPY_SCAN_BLEND;
  if ((!blend && p->kind != MUSAPY_SCAN_DECAY) || !gs_dtype(p->dtype) ||
      (p->gate_dtype != p->dtype && p->gate_dtype != MUSAPY_DT_F32) || p->shape == nullptr || p->gate_strides == nullptr ||
      (p->reset != nullptr && p->reset_strides == nullptr))
    return gs_bad();
  const bool reads_x = !grad || blend;
  if (reads_x && p->x_strides == nullptr) return gs_bad();
  if (grad && (p->h_strides == nullptr || p->dh_strides == nullptr ||
               (p->dgate_dtype != p->gate_dtype && p->dgate_dtype != MUSAPY_DT_F32)))
    return gs_bad();
  uint64_t numel = 1;
  for (int i = 0; i < p->ndim; ++i) {
    if (p->shape[i] >= (uint64_t(1) << 32)) return gs_bad();
    numel *= p->shape[i];
  }
  if (numel > 0 && (p->gate == nullptr || p->out == nullptr || (reads_x && p->x == nullptr) ||
                    (grad && (p->h == nullptr || p->dh == nullptr || p->dgate == nullptr))))
    return gs_bad();

  out = GsPlan{};
  GsArgs& a = out.a;
  const int nd = p->ndim, axis = p->axis;
  const bool parts = grad && p->parts != 0;
  if (parts && (axis == nd - 1 || p->gate_strides[nd - 1] != 0 || p->dgate_dtype != MUSAPY_DT_F32)) return gs_bad();
  // strides of every operand in every dim
  int64_t st[kGsOps][kMaxDims];
  int64_t full = 1, lane = 1, dg = 1;
  for (int i = nd - 1; i >= 0; --i) {
    st[kGsX][i] = reads_x ? p->x_strides[i] : 0;
    st[kGsGate][i] = p->gate_strides[i];
    st[kGsReset][i] = p->reset ? p->reset_strides[i] : 0;
    st[kGsH][i] = grad ? p->h_strides[i] : 0;
    st[kGsDh][i] = grad ? p->dh_strides[i] : 0;
    st[kGsOut][i] = full;
    full *= int64_t(p->shape[i]);
    st[kGsState][i] = i == axis ? 0 : lane;
    if (i != axis) lane *= int64_t(p->shape[i]);
    if (parts && i == nd - 1) {
      st[kGsDgate][i] = 0;
      dg *= int64_t(p->parts);
    } else {
      st[kGsDgate][i] = dg;
      dg *= int64_t(p->shape[i]);
    }
  }
  // non-axis dims, innermost first, merged where every operand walks two of them as one
  uint64_t size[kMaxDims];
  int64_t cst[kGsOps][kMaxDims];
  int n = 0;
  for (int i = nd - 1; i >= 0; --i) {
    // the dim that shared gates are summed over stays one of its own, whatever its size
    const bool keep = parts && i == nd - 1;
    if (i == axis || (p->shape[i] == 1 && !keep)) continue;
    if (n > 0 && !(parts && n == 1)) {
      bool merge = true;
      for (int o = 0; o < kGsOps; ++o) merge = merge && st[o][i] == cst[o][n - 1] * int64_t(size[n - 1]);
      if (merge && size[n - 1] * p->shape[i] < (uint64_t(1) << 32)) {
        size[n - 1] *= p->shape[i];
        continue;
      }
    }
    size[n] = p->shape[i];
    for (int o = 0; o < kGsOps; ++o) cst[o][n] = st[o][i];
    ++n;
  }
  if (n == 0) {
    size[0] = 1;
    for (int o = 0; o < kGsOps; ++o) cst[o][0] = 1;
    n = 1;
  }
  a.T = p->shape[axis];
  a.D = uint32_t(size[0]);
  out.rows = 1;
  a.ix.nd = n - 1;
  for (int i = 1; i < n; ++i) {
    out.rows *= size[i];
    a.ix.div[i - 1] = make_fastdiv(uint32_t(size[i] ? size[i] : 1));
    for (int o = 0; o < kGsOps; ++o) a.ix.stride[o][i - 1] = cst[o][i];
  }
  for (int o = 0; o < kGsOps; ++o) {
    a.ls[o] = cst[o][0];
    a.ts[o] = st[o][axis];
  }
  if (uint64_t(lane) >= (uint64_t(1) << 32)) return gs_bad();  // lanes are numbered in 32 bits
  auto unit = [&](int o) { return a.ls[o] == 1 || a.D == 1; };
  out.lanes = (!reads_x || unit(kGsX)) && unit(kGsOut) && unit(kGsState) && (unit(kGsGate) || a.ls[kGsGate] == 0) &&
              (p->reset == nullptr || a.ls[kGsReset] == 0 || a.D == 1) && (!grad || (unit(kGsH) && unit(kGsDh)));
  a.x = p->x;
  a.gate = p->gate;
  a.reset = p->reset;
  a.h = p->h;
  a.dh = p->dh;
  a.first = grad ? p->dlast : p->first;
  a.h_first = p->first;
  a.out = p->out;
  a.dgate = p->dgate;
  a.last = p->last;
  a.dgate_f32 = grad && p->dgate_dtype == MUSAPY_DT_F32;
  a.part_lanes = -1;
  if (parts) {
    const int V = gs_vector(p->dtype);
    if (!out.lanes || a.D != p->shape[nd - 1]) return gs_bad();
    a.part_lanes = gs_part_shift(a.D, V);
    if (p->parts != ((a.D + V - 1) / V) >> a.part_lanes) return gs_bad();
  }
  return true;
}

void gs_vectors(GsPlan& pl, int V) {
  pl.a.nv = (pl.a.D + uint32_t(V) - 1) / uint32_t(V);
  pl.a.nvec = uint32_t(pl.rows) * pl.a.nv;
  pl.a.nvdiv = make_fastdiv(pl.a.nv ? pl.a.nv : 1);
}

}  // namespace mpy

using namespace mpy;

extern "C" {

size_t musapy_gated_scan_scratch_v1(const musapy_gated_scan_args* p, int grad) { return 0; }

size_t musapy_gated_scan_parts_v1(const musapy_gated_scan_args* p) {
  if (p == nullptr || p->shape == nullptr || p->gate_strides == nullptr || p->ndim < 2 || p->ndim > kMaxDims ||
      p->axis == p->ndim - 1 || p->gate_strides[p->ndim - 1] != 0 || !gs_dtype(p->dtype))
    return 0;
  // sums over the lanes are formed where every other operand has unit-stride lanes
  const int i = p->ndim - 1;
  auto unit = [&](const ssize_t* s) { return s != nullptr && (s[i] == 1 || p->shape[i] == 1); };
  if ((p->kind == MUSAPY_SCAN_BLEND && !unit(p->x_strides)) || !unit(p->h_strides) || !unit(p->dh_strides) ||
      (p->reset && (p->reset_strides == nullptr || (p->reset_strides[i] != 0 && p->shape[i] != 1))))
    return 0;
  const int V = gs_vector(p->dtype);
  return ((p->shape[i] + V - 1) / V) >> gs_part_shift(p->shape[i], V);
}

int musapy_gated_scan_v1(const musapy_gated_scan_args* p, void* scratch, size_t scratch_bytes, void* workspace,
                         size_t workspace_bytes, hipStream_t st) {
  GsPlan pl;
  if (!gs_plan(p, false, pl)) return -1;
  if (pl.rows == 0 || pl.a.D == 0) return 0;
  const int V = pl.lanes ? gs_vector(p->dtype) : 1;
  gs_vectors(pl, V);
  const unsigned grid = unsigned((uint64_t(pl.a.nvec) + kGsBlock - 1) / kGsBlock);
  gs_types(p->dtype, p->gate_dtype, [&](auto tx, auto tg) {
    using TX = decltype(tx);
    using TG = decltype(tg);
    constexpr int kV = 16 / int(sizeof(TX));
    if (p->kind == MUSAPY_SCAN_BLEND) {
      if (V == 1) k_gs_walk<TX, TG, true, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_walk<TX, TG, true, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    } else {
      if (V == 1) k_gs_walk<TX, TG, false, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_walk<TX, TG, false, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    }
  });
  return 0;
}

}  // extern "C"
