// gated_scan_rows.hpp -- gated scans whose steps are unit-stride: what both directions share.
//
// A thread holds eight consecutive steps of a row, a group of GW threads a tile of 8 GW: eight threads
// for rows of up to 64 steps, a wave for up to 512, a workgroup beyond.  The groups' maps are joined by
// DPP moves in the wave, and across the four waves of a workgroup in LDS.  A workgroup walks the
// tiles of its row with the next one's loads in flight, or, where there are too few rows to fill the
// GPU, each tile has a workgroup of its own and a look-back (gated_scan.hpp).
#pragma once

#include "gated_scan.hpp"

namespace mpy {

constexpr int kGsRun = 8;  // steps of a thread

template <int CTRL, int MASK>
__device__ inline float gs_dpp(float none, float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, MASK, 0xf, false));
}

template <int CTRL, int MASK>
__device__ inline GsWide gs_dpp(GsWide none, GsWide v) {
  return {gs_dpp<CTRL, MASK>(none.m, v.m), __builtin_amdgcn_update_dpp(none.e, v.e, CTRL, MASK, 0xf, false)};
}
// the value of the last lane of the thread's group of GW lanes
template <int GW>
__device__ inline float gs_lane(float v) {
  if constexpr (GW == kWave) return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), kWave - 1));
  else return __shfl(v, GW - 1, GW);
}
template <int GW>
__device__ inline GsWide gs_lane(GsWide v) {
  if constexpr (GW == kWave) return {gs_lane<GW>(v.m), __builtin_amdgcn_readlane(v.e, kWave - 1)};
  else return {__shfl(v.m, GW - 1, GW), __shfl(v.e, GW - 1, GW)};
}

// From each thread's map (A, H) to the one of all threads in front of it in its group (of at most a
// wave), and the whole group's (ta, th).
template <int GW, class F>
__device__ inline void gs_join(F A, float H, F& ea, float& eh, F& ta, float& th) {
  const int l = threadIdx.x % GW;
  auto step = [&](auto ctrl, auto mask, int d) {
    F pa = gs_dpp<ctrl.value, mask.value>(gs_one<F>(), A);
    float ph = gs_dpp<ctrl.value, mask.value>(0.0f, H);
    if (GW < 16 && l < d) {  // a neighbour group's
      pa = gs_one<F>();
      ph = 0.0f;
    }
    H = gs_apply(A, H, ph);
    A = gs_then(A, pa);
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{}, 1);  // row_shr:1, 2, 4, 8
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{}, 2);
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{}, 4);
  if constexpr (GW > 8) {
    step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{}, 8);
    step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{}, 0);  // row_bcast:15
    step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{}, 0);  // row_bcast:31
    ta = gs_lane<GW>(A);
    th = gs_lane<GW>(H);
    ea = gs_dpp<0x138, 0xf>(gs_one<F>(), A);  // wave_shr:1
    eh = gs_dpp<0x138, 0xf>(0.0f, H);
  } else {
    ta = gs_lane<GW>(A);
    th = gs_lane<GW>(H);
    ea = gs_dpp<0x111, 0xf>(gs_one<F>(), A);
    eh = gs_dpp<0x111, 0xf>(0.0f, H);
    if (l == 0) {
      ea = gs_one<F>();
      eh = 0.0f;
    }
  }
}

template <class F>
struct GsRowTile {
  F a[2][kGsBlock / kWave];
  float h[2][kGsBlock / kWave];
  float state;
  uint32_t ticket;
};

// The state in front of each thread, from its steps' map; `P`, the state in front of the tile (of the
// row with SPLIT), becomes the one behind it.  `half` alternates between tiles.
template <int GW, bool SPLIT, class F>
__device__ inline float gs_row_state(GsRowTile<F>& sm, int& half, F A, float H, float& P, const GsSplit& sp, uint32_t chain,
                                     uint32_t tile) {
  F ea, ta;
  float eh, th;
  gs_join<GW < kWave ? GW : kWave>(A, H, ea, eh, ta, th);
  if constexpr (GW <= kWave) {
    const float c = gs_apply(ea, eh, P);
    P = gs_apply(ta, th, P);
    return c;
  } else {
    constexpr int kWaves = kGsBlock / kWave;
    const int wv = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
      sm.a[half][wv] = ta;
      sm.h[half][wv] = th;
    }
    lds_barrier();
    F wa[kWaves];
    float wh[kWaves];
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      wa[i] = sm.a[half][i];
      wh[i] = sm.h[half][i];
    }
    half ^= 1;
    if constexpr (SPLIT) {
      if (threadIdx.x == 0) {
        F A4 = wa[0];
        float H4 = wh[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) {
          H4 = gs_apply(wa[i], wh[i], H4);
          A4 = gs_then(wa[i], A4);
        }
        sm.state = gs_look_back<1, F>(sp, chain, tile, 0, P, A4, H4);
      }
      lds_barrier();
      P = sm.state;
    }
    float c = P;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      if (i == wv) c = P;
      P = gs_apply(wa[i], wh[i], P);
    }
    return gs_apply(ea, eh, c);
  }
}

// Eight steps from step `at` on (BACK: from it backwards; they lie in the pack in memory order, so step
// e of the thread is gs_at<BACK>(e)); of fewer than eight, `none` in the others' place.  ts is 0 where
// one element serves all steps.
template <bool BACK>
__device__ constexpr int gs_at(int e) { return BACK ? kGsRun - 1 - e : e; }
template <bool BACK, bool NT, class T>
__device__ inline Pack<T, kGsRun> gs_load_run(const T* at, int64_t ts, int n, T none) {
  if (n <= 0) return pack_all<T, kGsRun>(none);
  if (ts == 0 && n == kGsRun) return pack_all<T, kGsRun>(*at);
  if (n == kGsRun) return pack_load<NT, kGsRun>(BACK ? at - (kGsRun - 1) : at, kGsRun, none);
  Pack<T, kGsRun> p;
#pragma unroll
  for (int i = 0; i < p.kWords; ++i) p.w[i] = 0;
#pragma unroll
  for (int e = 0; e < kGsRun; ++e) {
    const int j = gs_at<BACK>(e);
    const uint32_t b = pack_bits(e < n ? at[BACK ? -e * ts : e * ts] : none);
    if constexpr (sizeof(T) == 4) p.w[j] = b;
    else p.w[j / 2] |= b << (16 * (j % 2));
  }
  return p;
}
template <bool BACK, bool NT, class T>
__device__ inline void gs_store_run(T* at, int n, const float (&x)[kGsRun]) {
  if (n == kGsRun) {
    float y[kGsRun];
#pragma unroll
    for (int e = 0; e < kGsRun; ++e) y[gs_at<BACK>(e)] = x[e];
    pack_store<NT>(BACK ? at - (kGsRun - 1) : at, kGsRun, y);
  } else {
#pragma unroll
    for (int e = 0; e < kGsRun; ++e)
      if (e < n) at[BACK ? -e : e] = T(x[e]);
  }
}
template <bool BACK>
__device__ inline uint32_t gs_load_cuts(const uint8_t* at, int64_t ts, int n) {
  uint32_t cuts = 0;
#pragma unroll
  for (int e = 0; e < kGsRun; ++e)
    if (e < n) cuts |= uint32_t(at[BACK ? -e * ts : e * ts] != 0) << e;
  return cuts;
}

// The row and tile a thread's group starts with; false where there is none.
template <int GW, bool SPLIT>
__device__ inline bool gs_row_take(const GsArgs& p, const GsSplit& sp, uint32_t& ticket, uint32_t& chain, uint32_t& tile,
                                   int64_t (&off)[kGsOps]) {
  if (!gs_take<SPLIT>(sp, ticket, chain, tile)) return false;
  if constexpr (GW < kGsBlock) {
    chain = blockIdx.x * (kGsBlock / GW) + threadIdx.x / GW;
    if (chain >= p.nvec) return false;  // a whole group: the others go on
  }
  const uint32_t row = fd_div(p.nvdiv, chain), col = chain - row * p.nv;
  gs_row_offsets(p.ix, row, off);
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
  return true;
}

// Calls fn with (GW, SPLIT) of a route.
template <class Fn>
inline void gs_row_kernel(const GsRoute& r, Fn&& fn) {
  using std::integral_constant;
  if (r.group == 8) fn(integral_constant<int, 8>{}, std::false_type{});
  else if (r.group == kWave) fn(integral_constant<int, kWave>{}, std::false_type{});
  else if (r.words == 0) fn(integral_constant<int, kGsBlock>{}, std::false_type{});
  else fn(integral_constant<int, kGsBlock>{}, std::true_type{});
}

}  // namespace mpy
