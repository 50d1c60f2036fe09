// gated_scan.hip -- the gated scan's forward kernels and the planning of both directions, for gfx950.
#include "gated_scan_rows.hpp"

namespace mpy {

// One thread per V lanes, in batches of steps: two lanes, so that short scans have threads enough
// (16 steps of (64, 8192) lanes bf16 14.4 us, with eight lanes a thread 30.2); V = 1 takes any strides.  A
// batch's loads are issued before the stores of the one in front, which they would else wait behind.
template <class TX, class TG, bool BLEND, int V>
__global__ __launch_bounds__(kGsBlock) void k_gs_walk(GsArgs p) {
  const uint64_t q = uint64_t(blockIdx.x) * kGsBlock + threadIdx.x;
  if (q >= p.nvec) return;
  const uint32_t row = fd_div(p.nvdiv, uint32_t(q));
  const uint32_t col = (uint32_t(q) - row * p.nv) * V;
  const int nl = p.D - col < uint32_t(V) ? int(p.D - col) : V;
  int64_t off[kGsOps];
  gs_row_offsets(p.ix, row, off);
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
  const TX* x = static_cast<const TX*>(p.x) + off[kGsX];
  const TG* gate = static_cast<const TG*>(p.gate) + off[kGsGate];
  const uint8_t* reset = p.reset ? p.reset + off[kGsReset] : nullptr;
  TX* out = static_cast<TX*>(p.out) + off[kGsOut];
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = p.first && v < nl ? p.first[off[kGsState] + v] : 0.0f;
  GsBatch<TX, V> nb;
  GsBatch<TG, V> ng;
  bool ncuts[kGsBatch];
  auto load = [&](uint64_t t) {
    const int steps = p.T - t < uint64_t(kGsBatch) ? int(p.T - t) : kGsBatch;
    nb.load(x, p.ts[kGsX], p.ls[kGsX], nl, steps);
    ng.load(gate, p.ts[kGsGate], p.ls[kGsGate], nl, steps);
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) ncuts[s] = reset && s < steps && reset[s * p.ts[kGsReset]];
    x += kGsBatch * p.ts[kGsX];
    gate += kGsBatch * p.ts[kGsGate];
    if (reset) reset += kGsBatch * p.ts[kGsReset];
  };
  if (p.T > 0) load(0);
  for (uint64_t t = 0; t < p.T; t += kGsBatch) {
    const int steps = p.T - t < uint64_t(kGsBatch) ? int(p.T - t) : kGsBatch;
    const GsBatch<TX, V> b = nb;
    const GsBatch<TG, V> g = ng;
    bool cuts[kGsBatch];
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) cuts[s] = ncuts[s];
    if (t + kGsBatch < p.T) load(t + kGsBatch);
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) {
      if (s >= steps) break;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = g.get(s, v), in = b.get(s, v);
        if constexpr (BLEND) {
          float rest;
          sigmoid_pair(a, a, rest);
          in = rest * in;
        }
        h[v] = cuts[s] ? in : __builtin_fmaf(a, h[v], in);
      }
      pack_store<false>(out + s * p.ts[kGsOut], nl, h);
    }
    out += kGsBatch * p.ts[kGsOut];
  }
  if (p.last) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nl) p.last[off[kGsState] + v] = h[v];
  }
}

// One tile (gated_scan.hpp) a workgroup; SPLIT: several tiles to a chain.  Bound by HBM as rows in pieces of
// 128 bytes use it: (8, 2048, 4096) bf16 blend 93 us with the clearing of its words, 4.3 TB/s, where a plain copy in
// that order takes 88 us (of 512-byte pieces 65 to 69: tiles of wider pieces were not tried); (65536, 2048) bf16
// decay with f32 gates 233 us, 4.6 TB/s.
template <class TX, class TG, bool BLEND, bool RESET, bool SPLIT, bool NT>
__global__ __launch_bounds__(kGsBlock) __attribute__((amdgpu_waves_per_eu(4))) void k_gs_tiles(GsArgs p, GsSplit sp) {
  constexpr int V = 16 / int(sizeof(TX));
  constexpr int S = kGsS;
  constexpr uint32_t kSteps = kGsTileSteps;
  using F = GsFactor<BLEND>;
  __shared__ GsTile<V, F> sm;
  uint32_t chain, tile;
  if (!gs_take<SPLIT>(sp, sm.ticket, chain, tile)) return;
  const GsPlace<V> at(p, chain);
  const uint64_t t0 = uint64_t(tile) * kSteps + threadIdx.x / kGsLt * S;  // the thread's first step
  const bool full = GsPlace<V>::whole(p, chain) && (uint64_t(tile) + 1) * kSteps <= p.T;
  const int steps = full ? S : at.nl == 0 || t0 >= p.T ? 0 : p.T - t0 < uint64_t(S) ? int(p.T - t0) : S;
  const TX* x = static_cast<const TX*>(p.x) + at.off[kGsX] + int64_t(t0) * p.ts[kGsX];
  const TG* gate = static_cast<const TG*>(p.gate) + at.off[kGsGate] + int64_t(t0) * p.ts[kGsGate];
  TX* out = static_cast<TX*>(p.out) + at.off[kGsOut] + int64_t(t0) * p.ts[kGsOut];

  Pack<TX, V> wx[S];
  Pack<TG, V> wg[S];
  uint32_t cuts = 0;
  auto load = [&](auto FULL) {
    constexpr bool F = decltype(FULL)::value;
    // steps and lanes that are not there leave the state alone: x = 0 and a factor of 1
    gs_load_steps<F, NT>(wx, x, p.ts[kGsX], 1, at.nl, steps, TX(0.0f));
    gs_load_steps<F, NT>(wg, gate, p.ts[kGsGate], p.ls[kGsGate], at.nl, steps, TG(BLEND ? __builtin_inff() : 1.0f));
    if constexpr (RESET) {
      const uint8_t* reset = p.reset + at.off[kGsReset] + int64_t(t0) * p.ts[kGsReset];
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (F || s < steps) cuts |= uint32_t(reset[s * p.ts[kGsReset]] != 0) << s;
    }
  };
  if (full) load(std::true_type{});
  else load(std::false_type{});

  float P = 0.0f;
  if (p.first && at.state_on) P = p.first[at.state];
  // blend: kept for the results, decay: formed again from the packed words
  float a[BLEND ? S : 1][V], b[BLEND ? S : 1][V], H[V], c[V];
  F A[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = gs_one<F>();
    H[v] = 0.0f;
  }
  auto step = [&](int s, int v, float h) {
    const bool cut = RESET && ((cuts >> s) & 1);
    const float as = BLEND ? a[BLEND ? s : 0][v] : pack_get(wg[s], v), bs = BLEND ? b[BLEND ? s : 0][v] : pack_get(wx[s], v);
    return cut ? bs : __builtin_fmaf(as, h, bs);
  };
#pragma unroll
  for (int s = 0; s < S; ++s) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float as = pack_get(wg[s], v);
      if constexpr (BLEND) {
        float rest;
        sigmoid_pair(as, as, rest);
        a[s][v] = as;
        b[s][v] = pack_get(wx[s], v) * rest;
      }
      H[v] = step(s, v, H[v]);
      if constexpr (BLEND) A[v] = RESET && ((cuts >> s) & 1) ? gs_none<F>() : A[v] * as;
    }
  }

  if constexpr (!BLEND) gs_run_lanes(A, wg, RESET && cuts);
  gs_tile_state<V, SPLIT, F>(sm, A, H, c, P, sp, chain, tile);

  if constexpr (!BLEND) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      pack_opaque(wx[s]);
      pack_opaque(wg[s]);
    }
  }
  auto finish = [&](auto FULL) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (!decltype(FULL)::value && s >= steps) continue;
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = step(s, v, c[v]);
      pack_store<NT>(out + s * p.ts[kGsOut], decltype(FULL)::value ? V : at.nl, c);
    }
  };
  if (full) finish(std::true_type{});
  else finish(std::false_type{});
  if (tile + 1 == sp.tiles && p.last && at.state_on) p.last[at.state] = P;
}

// Rows of unit-stride steps (gated_scan_rows.hpp): (4, 1500, 5001) f32 77.0 us, 4.7 TB/s, on rows that start
// off cache lines.
template <class TX, class TG, bool BLEND, bool RESET, int GW, bool SPLIT, bool NT>
__global__ __launch_bounds__(kGsBlock) void k_gs_rows(GsArgs p, GsSplit sp) {
  using F = GsFactor<BLEND>;
  __shared__ GsRowTile<F> sm;
  uint32_t chain, tile;
  int64_t off[kGsOps];
  if (!gs_row_take<GW, SPLIT>(p, sp, sm.ticket, chain, tile, off)) return;
  constexpr uint32_t kSteps = GW * kGsRun;
  uint64_t t = uint64_t(tile) * kSteps + threadIdx.x % GW * kGsRun;  // the thread's first step
  auto left = [&](uint64_t at) { return at >= p.T ? 0 : p.T - at < uint64_t(kGsRun) ? int(p.T - at) : kGsRun; };
  Pack<TX, kGsRun> nx;
  Pack<TG, kGsRun> ng;
  uint32_t ncuts = 0;
  auto load = [&](uint64_t at) {
    const int n = left(at);
    nx = gs_load_run<false, NT>(static_cast<const TX*>(p.x) + off[kGsX] + int64_t(at), 1, n, TX(0.0f));
    ng = gs_load_run<false, NT>(static_cast<const TG*>(p.gate) + off[kGsGate] + int64_t(at) * p.ts[kGsGate], p.ts[kGsGate], n,
                                TG(BLEND ? __builtin_inff() : 1.0f));
    if constexpr (RESET)
      ncuts = gs_load_cuts<false>(p.reset + off[kGsReset] + int64_t(at) * p.ts[kGsReset], p.ts[kGsReset], n);
  };
  load(t);
  float P = p.first ? p.first[off[kGsState]] : 0.0f;
  int half = 0;
  for (;;) {
    float a[kGsRun], b[kGsRun], H = 0.0f;
    F A = gs_one<F>();
    const uint32_t cuts = ncuts;
#pragma unroll
    for (int e = 0; e < kGsRun; ++e) {
      a[e] = pack_get(ng, e);
      b[e] = pack_get(nx, e);
      if constexpr (BLEND) {
        float rest;
        sigmoid_pair(a[e], a[e], rest);
        b[e] *= rest;
      }
      const bool cut = RESET && ((cuts >> e) & 1);
      H = cut ? b[e] : __builtin_fmaf(a[e], H, b[e]);
      if constexpr (BLEND) A = cut ? gs_none<F>() : A * a[e];
    }
    if constexpr (!BLEND) {
      bool plain = true;
      A = gs_run(a, plain);
      if (!plain) A = gs_run_stepwise(a);
      if (RESET && cuts) A = gs_none<F>();
    }
    if (!SPLIT && tile + 1 < sp.tiles) load(t + kSteps);
    float c = gs_row_state<GW, SPLIT, F>(sm, half, A, H, P, sp, chain, tile);
    float h[kGsRun];
#pragma unroll
    for (int e = 0; e < kGsRun; ++e) {
      c = RESET && ((cuts >> e) & 1) ? b[e] : __builtin_fmaf(a[e], c, b[e]);
      h[e] = c;
    }
    const int n = left(t);
    if (n > 0) gs_store_run<false, NT>(static_cast<TX*>(p.out) + off[kGsOut] + int64_t(t), n, h);
    if (tile + 1 >= sp.tiles) {
      if (p.last && threadIdx.x % GW == 0) p.last[off[kGsState]] = P;
      break;
    }
    if (SPLIT) break;
    ++tile;
    t += kSteps;
  }
}

__global__ void k_gs_clear(uint64_t* w, uint64_t n) {
  for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += uint64_t(gridDim.x) * blockDim.x) w[i] = 0;
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
  bool empty = false;
  for (int i = 0; i < p->ndim; ++i) {
    if (p->shape[i] >= (uint64_t(1) << 32)) return gs_bad();
    empty = empty || (i != p->axis && p->shape[i] == 0);
  }
  out = GsPlan{};
  if (empty) return true;  // no lanes
  uint64_t lanes = 1;
  for (int i = 0; i < p->ndim; ++i)  // lanes are numbered in 32 bits
    if (i != p->axis && (lanes *= p->shape[i]) >= (uint64_t(1) << 32)) return gs_bad();
  if (p->shape[p->axis] > (uint64_t(1) << 60) / lanes) return gs_bad();
  if (p->shape[p->axis] > 0 && (p->gate == nullptr || p->out == nullptr || (reads_x && p->x == nullptr) ||
                    (grad && (p->h == nullptr || p->dh == nullptr || p->dgate == nullptr))))
    return gs_bad();

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
  if (n > kGsRowDims + 1) return gs_bad();
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
  auto unit = [&](int o) { return a.ls[o] == 1 || a.D == 1; };
  out.lanes = (!reads_x || unit(kGsX)) && unit(kGsOut) && unit(kGsState) && (unit(kGsGate) || a.ls[kGsGate] == 0) &&
              (p->reset == nullptr || a.ls[kGsReset] == 0 || a.D == 1) && (!grad || (unit(kGsH) && unit(kGsDh)));
  auto run = [&](int o) { return a.ts[o] == 1; };
  out.steps = (!reads_x || run(kGsX)) && run(kGsOut) && (run(kGsGate) || a.ts[kGsGate] == 0) &&
              (p->reset == nullptr || run(kGsReset) || a.ts[kGsReset] == 0) &&
              (!grad || (run(kGsH) && run(kGsDh) && run(kGsDgate) && !parts));
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

namespace {
void gs_vectors(GsPlan& pl, int V) {
  pl.a.nv = (pl.a.D + uint32_t(V) - 1) / uint32_t(V);
  pl.a.nvec = uint32_t(pl.rows) * pl.a.nv;
  pl.a.nvdiv = make_fastdiv(pl.a.nv ? pl.a.nv : 1);
}
}  // namespace

constexpr uint64_t kGsHead = kGsShards * kGsCounterWords;  // words in front of the tiles': the ticket counters

GsRoute gs_route(GsPlan& pl, int dtype) {
  GsRoute r;
  const uint64_t T = pl.a.T;
  auto words = [&](uint64_t lanes) {
    r.group_words = (r.tiles + kGsGroup - 1) / kGsGroup * r.chains * lanes;
    r.words = kGsHead + r.chains * r.tiles * lanes + r.group_words;
  };
  if (pl.steps && T > 1 && (!pl.lanes || pl.a.D == 1)) {
    gs_vectors(pl, 1);
    r.kind = GsRoute::kRows;
    r.group = T <= 8 * kGsRun ? 8 : T <= uint64_t(kWave) * kGsRun ? kWave : kGsBlock;
    r.chains = pl.a.nvec;
    r.tiles = (T + r.group * kGsRun - 1) / (r.group * kGsRun);
    // fewer rows than the GPU holds workgroups at a time: a workgroup to a tile
    if (r.tiles > 1 && r.chains < 1024) words(1);
    if (grid_fits((r.chains + kGsShards) * (r.words ? r.tiles : 1), kGsBlock)) return r;
    r = GsRoute{};
  }
  const int V = gs_vector(dtype);
  // A walk takes about 0.3 us a step (gradient: 0.8), however many lanes run beside each other; a tile's
  // time hardly depends on how many of its 128 steps there are.  bf16, us, walk and tiles: 600 lanes x 4 rows,
  // 8 steps 6.6 and 7.0, 32 steps 11.7 and 7.1; 131072 lanes, 32 steps 14.0 and 17.9, 64 steps 27.8 and 23.5;
  // 262144 lanes, 64 steps 31.4 and 41.3, 128 steps 58.5 and 40.6; 524288 lanes, 512 steps 309 and 353.
  // The gradient's tiles are slower by as much: 2400 lanes, 8 steps 10.2 and 11.2, 16 steps 16.3 and 11.0; 65536
  // lanes, 16 steps 17.1 and 21.2, 32 steps 29.9 and 21.5; 262144 lanes, 64 steps 72 and 97, 128 steps 140 and 111;
  // 524288 lanes, 512 steps 729 and 780.  f32 decay: 16384 lanes, 8 steps 5.7 and 5.7; 65536 lanes, 16 steps 8.0 and
  // 9.1, 32 steps 12.3 and 10.3; 262144 lanes, 64 steps 41.3 and 40.3; 524288 lanes, 512 steps 602 and 780 (gradient
  // 8.6 and 7.2; 13.8 and 13.9, 23.2 and 14.9; 71.1 and 71.3; 1052 and 1022).
  const uint64_t lanes = pl.rows * pl.a.D;
  gs_vectors(pl, V);
  const uint64_t chains = (uint64_t(pl.a.nvec) + kGsLt - 1) / kGsLt, tiles = (T + kGsTileSteps - 1) / kGsTileSteps;
  if (!pl.lanes || T <= 8 + lanes / 4096 || lanes >= 524288 || !grid_fits((chains + kGsShards) * tiles, kGsBlock)) {
    r.V = pl.lanes ? 2 : 1;
    if (pl.a.part_lanes >= 0) {  // the lanes of a sum stay those of whole vectors
      if (pl.a.D % V) r.V = V;
      else pl.a.part_lanes += V == 8 ? 2 : 1;
    }
    gs_vectors(pl, r.V);
    return r;
  }
  r.kind = GsRoute::kTiles;
  r.V = V;
  r.chains = chains;
  r.tiles = tiles;
  if (r.tiles > 1) words(kGsLt * uint64_t(r.V));
  return r;
}

bool gs_split(GsSplit& sp, const GsRoute& r, void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes,
              hipStream_t st) {
  sp.chains = uint32_t(r.chains);
  sp.tiles = uint32_t(r.tiles);
  sp.shards = sp.chains < kGsShards ? sp.chains : kGsShards;
  sp.per_shard = (sp.chains + sp.shards - 1) / sp.shards;
  sp.sdiv = make_fastdiv(sp.shards);
  sp.pdiv = make_fastdiv(sp.per_shard);
  if (r.words == 0) return true;
  WsSplit ws;
  if (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 7) || scratch_bytes < r.words * 8 ||
      !ws_split(workspace, workspace_bytes, ws)) {
    g_wrapper_error = 1;
    return false;
  }
  uint64_t* w = static_cast<uint64_t*>(scratch);
  sp.counters = w;
  sp.groups = w + kGsHead;
  sp.words = sp.groups + r.group_words;
  sp.fault = ws.fault;
  sp.spin_limit = wait_spin_limit();
  const uint64_t blocks = (r.words + 255) / 256;
  k_gs_clear<<<unsigned(blocks < 2048 ? blocks : 2048), 256, 0, st>>>(w, r.words);
  return true;
}

}  // namespace mpy

using namespace mpy;

extern "C" {

size_t musapy_gated_scan_scratch_v1(const musapy_gated_scan_args* p, int grad) {
  GsPlan pl;
  if (!gs_plan(p, grad != 0, pl)) {
    g_wrapper_error = 0;  // the call itself reports it
    return 0;
  }
  if (pl.rows == 0 || pl.a.D == 0) return 0;
  return gs_route(pl, p->dtype).words * 8;
}

int musapy_gated_scan_route_v1(const musapy_gated_scan_args* p, int grad, musapy_gated_scan_route* route) {
  GsPlan pl;
  if (route == nullptr) return gs_bad() ? 0 : -1;
  if (!gs_plan(p, grad != 0, pl)) return -1;
  *route = musapy_gated_scan_route{};
  if (pl.rows == 0 || pl.a.D == 0) return 0;
  const GsRoute r = gs_route(pl, p->dtype);
  route->kind = r.kind == GsRoute::kWalk ? MUSAPY_SCAN_WALK : r.kind == GsRoute::kTiles ? MUSAPY_SCAN_TILES : MUSAPY_SCAN_ROWS;
  route->vector = r.V;
  route->rows = pl.rows;
  route->lanes = pl.a.D;
  route->vectors = pl.a.nv;
  route->chains = r.chains;
  route->tiles = r.tiles;
  route->split = r.words != 0;
  return 0;
}

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
  const GsRoute r = gs_route(pl, p->dtype);
  const int V = r.V;
  if (r.kind != GsRoute::kWalk) {
    GsSplit sp{};
    if (!gs_split(sp, r, scratch, scratch_bytes, workspace, workspace_bytes, st)) return -1;
    const unsigned grid = gs_grid(r, sp);
    const bool nt = gs_stream(pl, r, p->dtype);
    gs_types(p->dtype, p->gate_dtype, [&](auto tx, auto tg) {
      using TX = decltype(tx);
      using TG = decltype(tg);
      gs_flags([&](auto BLEND, auto RESET, auto NT) {
        if (r.kind == GsRoute::kRows)
          gs_row_kernel(r, [&](auto GW, auto SPLIT) {
            k_gs_rows<TX, TG, BLEND.value, RESET.value, GW.value, SPLIT.value, NT.value><<<grid, kGsBlock, 0, st>>>(pl.a, sp);
          });
        else if (r.words)
          k_gs_tiles<TX, TG, BLEND.value, RESET.value, true, NT.value><<<grid, kGsBlock, 0, st>>>(pl.a, sp);
        else
          k_gs_tiles<TX, TG, BLEND.value, RESET.value, false, NT.value><<<grid, kGsBlock, 0, st>>>(pl.a, sp);
      }, p->kind == MUSAPY_SCAN_BLEND, p->reset != nullptr, nt);
    });
    return 0;
  }
  const unsigned grid = unsigned((uint64_t(pl.a.nvec) + kGsBlock - 1) / kGsBlock);
  if (!grid_fits(grid, kGsBlock) || (V != 1 && V != 2)) return gs_bad() ? 0 : -1;  // (the walks that there are)
  gs_types(p->dtype, p->gate_dtype, [&](auto tx, auto tg) {
    using TX = decltype(tx);
    using TG = decltype(tg);
    if (p->kind == MUSAPY_SCAN_BLEND) {
      if (V == 1) k_gs_walk<TX, TG, true, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_walk<TX, TG, true, 2><<<grid, kGsBlock, 0, st>>>(pl.a);
    } else {
      if (V == 1) k_gs_walk<TX, TG, false, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_walk<TX, TG, false, 2><<<grid, kGsBlock, 0, st>>>(pl.a);
    }
  });
  return 0;
}

}  // extern "C"
