// gated_scan_grad.hip -- the gated scan's gradient kernels, for gfx950.
#include "gated_scan_rows.hpp"

namespace mpy {

// One thread per V lanes, from the last step to the first, in batches as the forward's (16 steps of (64, 8192)
// bf16 blend 32 us, 3.3 TB/s; with eight lanes a thread 63).
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
  gs_row_offsets(p.ix, row, off);
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
  float c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = p.first && v < nl ? p.first[off[kGsState] + v] : 0.0f;
  GsBatch<TX, V> nd, nh, nx;
  GsBatch<TG, V> ng;
  bool ncuts[kGsBatch];
  auto load = [&](uint64_t k0) {
    const int64_t t = int64_t(p.T - 1 - k0);
    const int steps = !on ? 0 : p.T - k0 < uint64_t(kGsBatch) ? int(p.T - k0) : kGsBatch;
    nd.load(static_cast<const TX*>(p.dh) + off[kGsDh] + t * p.ts[kGsDh], -p.ts[kGsDh], p.ls[kGsDh], nl, steps);
    ng.load(static_cast<const TG*>(p.gate) + off[kGsGate] + t * p.ts[kGsGate], -p.ts[kGsGate], p.ls[kGsGate], nl, steps);
    if constexpr (BLEND)
      nx.load(static_cast<const TX*>(p.x) + off[kGsX] + t * p.ts[kGsX], -p.ts[kGsX], p.ls[kGsX], nl, steps);
    // (step t = 0 has no h[t-1])
    nh.load(static_cast<const TX*>(p.h) + off[kGsH] + (t - 1) * p.ts[kGsH], -p.ts[kGsH], p.ls[kGsH], nl,
            steps > 0 && k0 + steps == p.T ? steps - 1 : steps);
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s)
      ncuts[s] = p.reset && s < steps && p.reset[off[kGsReset] + (t - s) * p.ts[kGsReset]];
  };
  if (p.T > 0) load(0);
  for (uint64_t k0 = 0; k0 < p.T; k0 += kGsBatch) {
    const int steps = p.T - k0 < uint64_t(kGsBatch) ? int(p.T - k0) : kGsBatch;
    const int64_t tl = int64_t(p.T - 1 - k0);
    const GsBatch<TX, V> bd = nd, bh = nh, bx = nx;
    const GsBatch<TG, V> bg = ng;
    bool cuts[kGsBatch];
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) cuts[s] = ncuts[s];
    if (k0 + kGsBatch < p.T) load(k0 + kGsBatch);
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) {
      if (s >= steps) break;
      const int64_t t = tl - s;
      const bool cut = cuts[s];
      float dg[V], dx[V], dh[V], g[V], x[V], hb[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        dh[v] = bd.get(s, v);
        g[v] = bg.get(s, v);
        if constexpr (BLEND) x[v] = bx.get(s, v);
        hb[v] = bh.get(s, v);
        if (t == 0) hb[v] = p.h_first && v < nl ? p.h_first[off[kGsState] + v] : 0.0f;
        if (cut) hb[v] = 0.0f;
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float G = dh[v] + c[v];
        if constexpr (BLEND) {
          float s, rest;
          sigmoid_pair(g[v], s, rest);
          dx[v] = rest * G;
          dg[v] = G * (hb[v] - x[v]) * (s * rest);
          c[v] = cut ? 0.0f : s * G;
        } else {
          dx[v] = G;
          dg[v] = cut ? 0.0f : G * hb[v];
          c[v] = cut ? 0.0f : g[v] * G;
        }
      }
      if (on) pack_store<false>(static_cast<TX*>(p.out) + off[kGsOut] + t * p.ts[kGsOut], nl, dx);
      if (p.part_lanes >= 0) {
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) sum += v < nl ? dg[v] : 0.0f;
        for (int m = 1; m < (1 << p.part_lanes); m <<= 1) sum += __shfl_xor(sum, m, kWave);
        if (on && (vec & ((1u << p.part_lanes) - 1)) == 0)
          static_cast<float*>(p.dgate)[off[kGsDgate] + t * p.ts[kGsDgate] + (vec >> p.part_lanes)] = sum;
      } else if (on) {
        const int64_t at = off[kGsDgate] + t * p.ts[kGsDgate];
        if (p.dgate_f32) pack_store<false>(static_cast<float*>(p.dgate) + at, nl, dg);
        else pack_store<false>(static_cast<TG*>(p.dgate) + at, nl, dg);
      }
    }
  }
  if (p.last) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v < nl) p.last[off[kGsState] + v] = c[v];
  }
}

// One tile a workgroup, over reversed time: step k is t = T - 1 - k.  What was loaded stays as it was,
// and the factors are formed twice, for the tile's map and for its results: registers are dearer here
// than the second sigmoid.  Bound as the forward's tiles: (8, 2048, 4096) bf16 blend, with the clearing of its
// words, 172 to 203 us, 4.0 to 4.7 TB/s, by where its five arrays lie (the same build, calls and process); (2, 4099, 16, 128)
// f16 with decays shared by a head's channels 45 to 50 us, of which clearing takes 4.9 and the sums over the rest of a
// head 4.6.
template <class TX, class TG, bool BLEND, bool RESET, bool SPLIT, bool NT>
__global__ __launch_bounds__(kGsBlock) __attribute__((amdgpu_waves_per_eu(3))) void k_gs_grad_tiles(GsArgs p, GsSplit sp) {
  constexpr int V = 16 / int(sizeof(TX));
  constexpr int S = kGsS;
  constexpr uint32_t kSteps = kGsTileSteps;
  using F = GsFactor<BLEND>;
  __shared__ GsTile<V, F> sm;
  uint32_t chain, tile;
  if (!gs_take<SPLIT>(sp, sm.ticket, chain, tile)) return;
  const GsPlace<V> at(p, chain);
  const uint64_t k0 = uint64_t(tile) * kSteps + threadIdx.x / kGsLt * S;
  // (t = 0 has no h[t-1], so its tile is not a full one)
  const bool full = GsPlace<V>::whole(p, chain) && (uint64_t(tile) + 1) * kSteps < p.T;
  const int steps = full ? S : at.nl == 0 || k0 >= p.T ? 0 : p.T - k0 < uint64_t(S) ? int(p.T - k0) : S;
  const int64_t t0 = int64_t(p.T) - 1 - int64_t(k0);
  auto from = [&](auto* base, int o, int64_t t) { return base + at.off[o] + t * p.ts[o]; };
  Pack<TX, V> wd[S], wh[S], wx[S];
  Pack<TG, V> wg[S];
  uint32_t cuts = 0;
  auto load = [&](auto FULL) {
    constexpr bool F = decltype(FULL)::value;
    // steps and lanes that are not there pass the flow on: dh = 0 and a factor of 1
    gs_load_steps<F, NT>(wd, from(static_cast<const TX*>(p.dh), kGsDh, t0), -p.ts[kGsDh], 1, at.nl, steps, TX(0.0f));
    gs_load_steps<F, NT>(wg, from(static_cast<const TG*>(p.gate), kGsGate, t0), -p.ts[kGsGate], p.ls[kGsGate], at.nl, steps,
                         TG(BLEND ? __builtin_inff() : 1.0f));
    const int hs = k0 + steps == p.T ? steps - 1 : steps;  // h[-1] is no element of h
    gs_load_steps<F, NT>(wh, from(static_cast<const TX*>(p.h), kGsH, t0 - 1), -p.ts[kGsH], 1, at.nl, hs, TX(0.0f));
    if constexpr (BLEND)
      gs_load_steps<F, NT>(wx, from(static_cast<const TX*>(p.x), kGsX, t0), -p.ts[kGsX], 1, at.nl, steps, TX(0.0f));
    if constexpr (RESET) {
      const uint8_t* r = from(p.reset, kGsReset, t0);
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (F || s < steps) cuts |= uint32_t(r[-s * p.ts[kGsReset]] != 0) << s;
    }
  };
  if (full) load(std::true_type{});
  else load(std::false_type{});
  float P = 0.0f;
  if (p.first && at.state_on) P = p.first[at.state];
  float H[V], c[V];
  F A[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = gs_one<F>();
    H[v] = 0.0f;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const bool cut = RESET && ((cuts >> s) & 1);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = pack_get(wg[s], v), rest;
      if constexpr (BLEND) sigmoid_pair(a, a, rest);
      H[v] = cut ? 0.0f : a * (pack_get(wd[s], v) + H[v]);
      if constexpr (BLEND) A[v] = cut ? gs_none<F>() : A[v] * a;
    }
  }

  if constexpr (!BLEND) gs_run_lanes(A, wg, RESET && cuts);
  gs_tile_state<V, SPLIT, F>(sm, A, H, c, P, sp, chain, tile);

#pragma unroll
  for (int s = 0; s < S; ++s) {
    pack_opaque(wd[s]);
    pack_opaque(wg[s]);
  }
  TX* dx = from(static_cast<TX*>(p.out), kGsOut, t0);
  const int64_t dgate = at.off[kGsDgate] + t0 * p.ts[kGsDgate];
  const uint32_t vec = chain * kGsLt + threadIdx.x % kGsLt;  // parts: rows are whole groups of vectors
  const int parts = p.part_lanes < 0 ? 0 : 1 << p.part_lanes;
  const uint32_t part = parts ? (vec - fd_div(p.nvdiv, vec) * p.nv) >> p.part_lanes : 0;
  auto finish = [&](auto FULL) {
    constexpr bool F = decltype(FULL)::value;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (!F && s >= steps && !parts) continue;
      const bool cut = RESET && ((cuts >> s) & 1);
      float ox[V], og[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = pack_get(wg[s], v), rest = 1.0f;
        if constexpr (BLEND) sigmoid_pair(a, a, rest);
        float hb = pack_get(wh[s], v);
        if (!F && k0 + s + 1 == p.T && p.h_first && v < at.nl) hb = p.h_first[at.off[kGsState] + v];
        if (cut) hb = 0.0f;
        const float G = pack_get(wd[s], v) + c[v];
        if constexpr (BLEND) {
          ox[v] = rest * G;
          og[v] = G * (hb - pack_get(wx[s], v)) * (a * rest);
        } else {
          ox[v] = G;
          og[v] = cut ? 0.0f : G * hb;
        }
        c[v] = cut ? 0.0f : a * G;
      }
      const bool in = F || s < steps;
      if (in) pack_store<NT>(dx - s * p.ts[kGsOut], F ? V : at.nl, ox);
      const int64_t to = dgate - s * p.ts[kGsDgate];
      if (parts) {
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) sum += F || v < at.nl ? og[v] : 0.0f;
        for (int m = 1; m < parts; m <<= 1) sum += __shfl_xor(sum, m, kWave);
        if (in && (vec & uint32_t(parts - 1)) == 0) static_cast<float*>(p.dgate)[to + part] = sum;
      } else if (p.dgate_f32) {
        pack_store<NT>(static_cast<float*>(p.dgate) + to, F ? V : at.nl, og);
      } else {
        pack_store<NT>(static_cast<TG*>(p.dgate) + to, F ? V : at.nl, og);
      }
    }
  };
  if (full) finish(std::true_type{});
  else finish(std::false_type{});
  if (tile + 1 == sp.tiles && p.last && at.state_on) p.last[at.state] = P;
}

// Rows of unit-stride steps (gated_scan_rows.hpp), over reversed time: step k is t = T - 1 - k.  (4, 1500, 5001) f32
// 130 us, 4.6 TB/s.
template <class TX, class TG, bool BLEND, bool RESET, int GW, bool SPLIT, bool NT>
__global__ __launch_bounds__(kGsBlock) void k_gs_grad_rows(GsArgs p, GsSplit sp) {
  using F = GsFactor<BLEND>;
  __shared__ GsRowTile<F> sm;
  uint32_t chain, tile;
  int64_t off[kGsOps];
  if (!gs_row_take<GW, SPLIT>(p, sp, sm.ticket, chain, tile, off)) return;
  constexpr uint32_t kSteps = GW * kGsRun;
  uint64_t k = uint64_t(tile) * kSteps + threadIdx.x % GW * kGsRun;
  auto left = [&](uint64_t at) { return at >= p.T ? 0 : p.T - at < uint64_t(kGsRun) ? int(p.T - at) : kGsRun; };
  Pack<TX, kGsRun> nd, nh, nx;
  Pack<TG, kGsRun> ng;
  uint32_t ncuts = 0;
  auto load = [&](uint64_t at) {
    const int n = left(at);
    const int64_t t = int64_t(p.T) - 1 - int64_t(at);
    nd = gs_load_run<true, NT>(static_cast<const TX*>(p.dh) + off[kGsDh] + t, 1, n, TX(0.0f));
    // (step t = 0 has no h[t-1])
    nh = gs_load_run<true, NT>(static_cast<const TX*>(p.h) + off[kGsH] + t - 1, 1, at + n == p.T ? n - 1 : n, TX(0.0f));
    if constexpr (BLEND) nx = gs_load_run<true, NT>(static_cast<const TX*>(p.x) + off[kGsX] + t, 1, n, TX(0.0f));
    ng = gs_load_run<true, NT>(static_cast<const TG*>(p.gate) + off[kGsGate] + t * p.ts[kGsGate], p.ts[kGsGate], n,
                               TG(BLEND ? __builtin_inff() : 1.0f));
    if constexpr (RESET) ncuts = gs_load_cuts<true>(p.reset + off[kGsReset] + t * p.ts[kGsReset], p.ts[kGsReset], n);
  };
  load(k);
  float P = p.first ? p.first[off[kGsState]] : 0.0f;
  int half = 0;
  for (;;) {
    const uint32_t cuts = ncuts;
    float a[kGsRun], rest[kGsRun], dh[kGsRun], hb[kGsRun], x[kGsRun], H = 0.0f;
    F A = gs_one<F>();
    const int n = left(k);
#pragma unroll
    for (int e = 0; e < kGsRun; ++e) {
      const int j = gs_at<true>(e);
      a[e] = pack_get(ng, j);
      rest[e] = 1.0f;
      dh[e] = pack_get(nd, j);
      hb[e] = pack_get(nh, j);
      if constexpr (BLEND) {
        sigmoid_pair(a[e], a[e], rest[e]);
        x[e] = pack_get(nx, j);
      }
      const bool cut = RESET && ((cuts >> e) & 1);
      H = cut ? 0.0f : a[e] * (dh[e] + H);
      if constexpr (BLEND) A = cut ? gs_none<F>() : A * a[e];
    }
    if constexpr (!BLEND) {
      bool plain = true;
      A = gs_run(a, plain);
      if (!plain) A = gs_run_stepwise(a);
      if (RESET && cuts) A = gs_none<F>();
    }
    if (k + n == p.T && n > 0) {
      const float first = p.h_first ? p.h_first[off[kGsState]] : 0.0f;
#pragma unroll
      for (int e = 0; e < kGsRun; ++e) hb[e] = e == n - 1 ? first : hb[e];
    }
    if (!SPLIT && tile + 1 < sp.tiles) load(k + kSteps);
    float c = gs_row_state<GW, SPLIT, F>(sm, half, A, H, P, sp, chain, tile);
    float ox[kGsRun], og[kGsRun];
#pragma unroll
    for (int e = 0; e < kGsRun; ++e) {
      const bool cut = RESET && ((cuts >> e) & 1);
      const float G = dh[e] + c, h = cut ? 0.0f : hb[e];
      if constexpr (BLEND) {
        ox[e] = rest[e] * G;
        og[e] = G * (h - x[e]) * (a[e] * rest[e]);
      } else {
        ox[e] = G;
        og[e] = cut ? 0.0f : G * h;
      }
      c = cut ? 0.0f : a[e] * G;
    }
    if (n > 0) {
      const int64_t t = int64_t(p.T) - 1 - int64_t(k);
      gs_store_run<true, NT>(static_cast<TX*>(p.out) + off[kGsOut] + t, n, ox);
      if (p.dgate_f32) gs_store_run<true, NT>(static_cast<float*>(p.dgate) + off[kGsDgate] + t, n, og);
      else gs_store_run<true, NT>(static_cast<TG*>(p.dgate) + off[kGsDgate] + t, n, og);
    }
    if (tile + 1 >= sp.tiles) {
      if (p.last && threadIdx.x % GW == 0) p.last[off[kGsState]] = P;
      break;
    }
    if (SPLIT) break;
    ++tile;
    k += kSteps;
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
            k_gs_grad_rows<TX, TG, BLEND.value, RESET.value, GW.value, SPLIT.value, NT.value>
                <<<grid, kGsBlock, 0, st>>>(pl.a, sp);
          });
        else if (r.words)
          k_gs_grad_tiles<TX, TG, BLEND.value, RESET.value, true, NT.value><<<grid, kGsBlock, 0, st>>>(pl.a, sp);
        else
          k_gs_grad_tiles<TX, TG, BLEND.value, RESET.value, false, NT.value><<<grid, kGsBlock, 0, st>>>(pl.a, sp);
      }, p->kind == MUSAPY_SCAN_BLEND, p->reset != nullptr, nt);
    });
    return 0;
  }
  const unsigned grid = unsigned((uint64_t(pl.a.nvec) + kGsBlock - 1) / kGsBlock);
  if (!grid_fits(grid, kGsBlock)) {
    g_wrapper_error = 6;
    return -1;
  }
  gs_types(p->dtype, p->gate_dtype, [&](auto tx, auto tg) {
    using TX = decltype(tx);
    using TG = decltype(tg);
    constexpr int kV = 16 / int(sizeof(TX));
    if (p->kind == MUSAPY_SCAN_BLEND) {
      if (V == 1) k_gs_grad_walk<TX, TG, true, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else if (V == 2) k_gs_grad_walk<TX, TG, true, 2><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_grad_walk<TX, TG, true, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    } else {
      if (V == 1) k_gs_grad_walk<TX, TG, false, 1><<<grid, kGsBlock, 0, st>>>(pl.a);
      else if (V == 2) k_gs_grad_walk<TX, TG, false, 2><<<grid, kGsBlock, 0, st>>>(pl.a);
      else k_gs_grad_walk<TX, TG, false, kV><<<grid, kGsBlock, 0, st>>>(pl.a);
    }
  });
  return 0;
}

}  // extern "C"
