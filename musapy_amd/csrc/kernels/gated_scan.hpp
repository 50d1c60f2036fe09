// gated_scan.hpp -- the gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis, and its
// gradient: what the forward (gated_scan.hip) and backward (gated_scan_grad.hip) kernels share.
//
// Gradient: with c[t] what flows into h[t-1],
//   G[t] = dh[t] + c[t+1],  c[t] = a[t] G[t],  c[T] = dlast,
// which is the same recurrence run over reversed time, with (a[t], a[t] dh[t]) for (a, b).
#pragma once

#include <tuple>
#include <type_traits>

#include "kcommon.hpp"
#include "pack.hpp"
#include "publish.hpp"

namespace mpy {

constexpr int kGsBlock = 256;
constexpr int kGsBatch = 4;  // steps that a thread of the walks loads at a time

// Operands, and their places in the strides.  kGsState is first / last / dlast: x's shape without
// the scanned axis.
enum GsOperand { kGsX, kGsGate, kGsReset, kGsOut, kGsState, kGsH, kGsDh, kGsDgate, kGsOps };

// The rows: coalesced non-axis dims but the innermost, innermost first.  (Kernel arguments of a few
// hundred bytes: with room for 32 dims they were 2.5 KB.)
constexpr int kGsRowDims = 6;
struct GsRows {
  int nd;
  FastDiv div[kGsRowDims];
  int64_t stride[kGsOps][kGsRowDims];
};
__device__ inline void gs_row_offsets(const GsRows& ix, uint32_t row, int64_t (&off)[kGsOps]) {
#pragma unroll
  for (int o = 0; o < kGsOps; ++o) off[o] = 0;
  for (int i = 0; i < ix.nd; ++i) {
    const uint32_t q = fd_div(ix.div[i], row);
    const uint32_t c = row - q * ix.div[i].d;
    row = q;
#pragma unroll
    for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(c) * ix.stride[o][i];
  }
}

struct GsArgs {
  GsRows ix;
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

// The S steps of a thread as they lie in memory, `p` at the first one.  FULL: all steps and lanes are
// there; else `steps` and `nl` of them, and `none` in the others' place.
template <bool FULL, bool NT, class T, int V, int S>
__device__ inline void gs_load_steps(Pack<T, V> (&w)[S], const T* p, int64_t ts, int64_t ls, int nl, int steps, T none) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const T* at = p + s * ts;
    if (!FULL && s >= steps) w[s] = pack_all<T, V>(none);
    else if (ls == 0) w[s] = pack_all<T, V>(*at);
    else w[s] = pack_load<NT, V>(at, FULL ? V : nl, none);
  }
}

// The steps that a walk loads at a time, zeros past the last.
template <class T, int V>
struct GsBatch {
  Pack<T, V> w[kGsBatch];
  __device__ void load(const T* p, int64_t ts, int64_t ls, int nl, int steps) {
    gs_load_steps<false, false>(w, p, ts, ls, nl, steps, T(0.0f));
  }
  __device__ float get(int s, int v) const { return pack_get(w[s], v); }
};
template <class T>
struct GsBatch<T, 1> {
  T w[kGsBatch];
  __device__ void load(const T* p, int64_t ts, int64_t, int, int steps) {
#pragma unroll
    for (int s = 0; s < kGsBatch; ++s) w[s] = s < steps ? p[s * ts] : T(0.0f);
  }
  __device__ float get(int s, int) const { return float(w[s]); }
};

// ---- tiles of steps -------------------------------------------------------------------------------
// A run of steps maps the state c in front of it to A c + H behind it, and two runs compose to
// (A2 A1, A2 H1 + H2).  A run that holds a reset has A = gs_none(), "the state in front does not matter";
// a state of 0 is not multiplied, so that a product of growing gates that overflowed does not make it NaN.
//
// The type of A.  "blend": f32; its factors are at most 1, so that A is at most 1, and what it loses below 2^-126 is
// lost to the rounding of the state in front.  "decay": a fraction and an exponent, as decays may grow: a product that
// runs through 2^200 and back, on a state that stays in f32's range all the way, has to come back.  (While the states stay
// there, products of any run of steps are between 2^-278 and 2^278.)  (65536, 2048) bf16 takes 233 us so, 239 with factors
// in f64, whose compositions take longer, and 228 with f32 ones that lose the range.
struct GsWide {
  float m;  // 0, or from 0.5 to 1 in size; NaN: gs_none()
  int e;
};
template <bool BLEND>
using GsFactor = std::conditional_t<BLEND, float, GsWide>;

template <class F>
__device__ inline F gs_one();
template <>
__device__ inline float gs_one<float>() { return 1.0f; }
template <>
__device__ inline GsWide gs_one<GsWide>() { return {0.5f, 1}; }
template <class F>  // (a NaN gate gives it too, and has made H NaN already)
__device__ inline F gs_none();
template <>
__device__ inline float gs_none<float>() { return __builtin_nanf(""); }
template <>
__device__ inline GsWide gs_none<GsWide>() { return {__builtin_nanf(""), 0}; }

__device__ inline float gs_apply(float A, float H, float c) {
  return c == 0.0f || A != A ? H : __builtin_fmaf(A, c, H);
}
__device__ inline float gs_apply(GsWide A, float H, float c) {
  return c == 0.0f || A.m != A.m ? H : __builtin_amdgcn_ldexpf(A.m * c, A.e) + H;
}
// The factor of a run and of the one in front of it together.
__device__ inline float gs_then(float A, float front) { return A * front; }
__device__ inline GsWide gs_then(GsWide A, GsWide front) {
  const float p = A.m * front.m;
  return {__builtin_amdgcn_frexp_mantf(p), A.e + front.e + __builtin_amdgcn_frexp_expf(p)};
}
// The factor of N steps in a row, from their gates.  "decay": as one product where those of two neighbours are of a
// size that no product of all of them can leave f32's range or its normal numbers; `plain` becomes false where they
// are not, and the factor is to be formed step by step (which for eight steps takes twice the instructions).
template <int N>
__device__ inline GsWide gs_run(const float (&a)[N], bool& plain) {
  float p[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; ++i) p[i] = a[2 * i] * a[2 * i + 1];
  float all = p[0];
#pragma unroll
  for (int i = 1; i < N / 2; ++i) all *= p[i];
  constexpr float kMost = N == 4 ? 0x1p60f : 0x1p30f;
  float lo = __builtin_fabsf(p[0]), hi = lo;
#pragma unroll
  for (int i = 1; i < N / 2; ++i) {  // (where one is a NaN, so is the product: the factor is gs_none() either way)
    lo = __builtin_fminf(lo, __builtin_fabsf(p[i]));
    hi = __builtin_fmaxf(hi, __builtin_fabsf(p[i]));
  }
  plain = plain && lo >= 1.0f / kMost && hi <= kMost;
  return {__builtin_amdgcn_frexp_mantf(all), __builtin_amdgcn_frexp_expf(all)};
}
template <int N>
__device__ inline GsWide gs_run_stepwise(const float (&a)[N]) {
  GsWide A = gs_one<GsWide>();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float p = a[i] * A.m;
    A = {__builtin_amdgcn_frexp_mantf(p), A.e + __builtin_amdgcn_frexp_expf(p)};
  }
  return A;
}
// ... of the steps of each lane of a thread of the tiles
template <class T, int V, int S>
__device__ inline void gs_run_lanes(GsWide (&A)[V], const Pack<T, V> (&gates)[S], bool cut) {
  auto lane = [&](int v, auto&& run) {
    float a[S];
#pragma unroll
    for (int s = 0; s < S; ++s) a[s] = pack_get(gates[s], v);
    A[v] = run(a);
  };
  bool plain = true;
#pragma unroll
  for (int v = 0; v < V; ++v) lane(v, [&](const float (&a)[S]) { return gs_run(a, plain); });
  if (!plain) {
#pragma unroll
    for (int v = 0; v < V; ++v) lane(v, [&](const float (&a)[S]) { return gs_run_stepwise(a); });
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (cut) A[v] = gs_none<GsWide>();
}

// Tiles of 32 segments of 4 steps by 8 vectors of lanes: 128 bytes of x a step, every cache line one
// tile's.  Thread (segment, vector) holds its segment's steps in registers.
constexpr int kGsLt = 8;
constexpr int kGsS = 4;                                  // steps of a segment
constexpr int kGsTileSteps = kGsBlock / kGsLt * kGsS;    // 128

template <int V, class F>
struct GsTile {
  static constexpr int BS = kGsBlock;
  static constexpr int kSegs = BS / kGsLt;
  static constexpr int kLanes = kGsLt * V;              // 64 or 32
  static constexpr int kParts = BS / kLanes;            // threads that scan one lane's segments
  static constexpr int kPer = kSegs / kParts;           // segments of each
  // element v of thread (segment, vector); the padding puts the v of a vector on banks of their own, so
  // that both the threads' accesses and those lane by lane touch every bank once
  F a[V][BS + kGsLt];
  float h[V][BS + kGsLt];
  F pa[kParts][kLanes];
  float ph[kParts][kLanes], c[kParts][kLanes];
  uint32_t ticket;
};

// Steps split over workgroups.  For each tile of each chain (a group of vectors) and lane, one word
// holds the tile's (A, H); every kGsGroup tiles form a group, whose last tile publishes the group's
// (A, H) too, and later, in the same word, the state behind the group as (none, state), which is the
// map that gives that state whatever lies in front.  A word is 0 until it is published: (+0, +0)
// goes as (-0, +0), which means the same.
constexpr uint32_t kGsGroup = 4;
constexpr int kGsWindow = 8;  // groups whose words the look-back reads at once
struct GsSplit {
  // Tickets: one counter for each shard of chains, a cache line apart.  One counter for all took
  // 14 ns a ticket, the rate of atomics on one address: 239 us of the 16384 tiles of (65536, 2048).
  uint64_t* counters;
  // A shard is a run of neighbouring chains, and blocks go to the XCDs in turn: neighbours, which share
  // cache lines where rows do not start on them, run on one XCD at about the same time.
  uint32_t shards, per_shard;
  FastDiv sdiv, pdiv;
  uint64_t* words;   // [tile][chain][lane]
  uint64_t* groups;  // [group][chain][lane]
  uint32_t* fault;
  uint32_t spin_limit;
  uint32_t chains, tiles;
};
constexpr uint32_t kGsShards = 32;
constexpr uint32_t kGsCounterWords = 16;

// A word's upper half is A in 32 bits: an f32's own, or a sign, ten bits of exponent and 21 of fraction, rounded
// to nearest (2^-22, as much as a few of the tile's roundings).  What is too small for the exponent is as small as it
// can be and what is too large comes back as 2^1000000: the states behind them are 0 and infinite, and infinite behind both.
__device__ inline uint32_t gs_code(float A) { return __float_as_uint(A); }
constexpr uint32_t kGsHuge = 1023u << 21, kGsNone = kGsHuge | 1u, kGsTiny = 1u;
__device__ inline uint32_t gs_code(GsWide A) {
  const uint32_t b = __float_as_uint(A.m), sign = b & 0x80000000u, f = b & 0x7fffffu;
  uint32_t c = (uint32_t(A.e + 511) << 21) + ((f + 1u + ((f >> 2) & 1u)) >> 2);
  c = A.e < -510 ? kGsTiny : A.e > 511 || c > kGsHuge ? kGsHuge : c;
  c = A.m == 0.0f ? 0u : c;
  return A.m != A.m ? kGsNone : c | sign;
}
template <class F>
__device__ inline F gs_decode(uint32_t c);
template <>
__device__ inline float gs_decode<float>(uint32_t c) { return __uint_as_float(c); }
template <>
__device__ inline GsWide gs_decode<GsWide>(uint32_t c) {
  const uint32_t u = c & 0x7fffffffu, f = u >> 21;
  const float m = __uint_as_float((c & 0x80000000u) | 0x3f000000u | (u & 0x1fffffu) << 2);
  return {u == kGsNone ? __builtin_nanf("") : u == 0 ? 0.0f : m, f == 1023 ? 1000000 : int(f) - 511};
}
template <class F>
__device__ inline uint64_t gs_pack(F A, float H) {
  const uint64_t w = (uint64_t(gs_code(A)) << 32) | __float_as_uint(H);
  return w ? w : uint64_t(0x80000000u) << 32;
}
template <class F>
__device__ inline F gs_word_factor(uint64_t w) { return gs_decode<F>(uint32_t(w >> 32)); }
template <class F>
__device__ inline float gs_apply_word(uint64_t w, float c) { return gs_apply(gs_word_factor<F>(w), __uint_as_float(uint32_t(w)), c); }
template <class F>
__device__ inline bool gs_word_is_state(uint64_t w) {
  const uint32_t c = uint32_t(w >> 32);
  return std::is_same_v<F, GsWide> ? c == kGsNone : c << 1 > 0xff000000u;
}

// The state in front of `tile` for one lane, from the group in front's and the tiles of its own
// group that lie between; that group's state from the nearest one published, through the (A, H) of the
// groups between.  Every state is folded front to back over the same runs wherever the
// look-back starts, so results are the same bits run to run.  (ta, th) is the tile's own map; the last
// tile of a group publishes its group's.  A wait makes at most spin_limit polls, then records its
// fault and goes on with 0, so every workgroup exits.
template <int LANES, class F>
__device__ inline float gs_look_back(const GsSplit& sp, uint32_t chain, uint32_t tile, int lane, float first, F ta, float th) {
  const uint32_t group = tile / kGsGroup, in = tile % kGsGroup;
  const uint64_t ws = uint64_t(sp.chains) * LANES;
  uint64_t* const wt = sp.words + (uint64_t(tile) * sp.chains + chain) * LANES + lane;
  uint64_t* const wg = sp.groups + (uint64_t(group) * sp.chains + chain) * LANES + lane;
  const bool follow = tile + 1 < sp.tiles;            // a tile behind waits on this one,
  const bool last = follow && in == kGsGroup - 1;     // or on its group
  if (follow && !last) st_relaxed(wt, gs_pack(ta, th));
  uint32_t spins = 0;
  bool done = false;
  // the tiles of the group in front of this one
  uint64_t w[kGsGroup - 1] = {};
  for (; !done && spins < sp.spin_limit; ++spins) {
    bool ok = true;
#pragma unroll
    for (uint32_t i = 0; i < kGsGroup - 1; ++i) {
      w[i] = i < in ? ld_relaxed(wt - uint64_t(in - i) * ws) : gs_pack(gs_one<F>(), 0.0f);
      ok = ok && w[i] != 0;
    }
    done = __all(ok);
    if (!done) __builtin_amdgcn_s_sleep(1);
  }
  uint64_t mine = 0;
  if (last) {
    F ga = gs_one<F>();
    float gh = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kGsGroup - 1; ++i) {
      gh = gs_apply_word<F>(w[i], gh);
      ga = gs_then(gs_word_factor<F>(w[i]), ga);
    }
    mine = gs_pack(gs_then(ta, ga), gs_apply(ta, th, gh));
    st_relaxed(wg, mine);
  }
  // the state behind the group in front
  float P = first;
  if (group > 0) {
    done = false;
    for (; !done && spins < sp.spin_limit; ++spins) {
      uint64_t m[kGsWindow];
      m[0] = ld_relaxed(wg - ws);
      P = __uint_as_float(uint32_t(m[0]));
      done = __all(gs_word_is_state<F>(m[0]));
      if (done) break;
#pragma unroll
      for (int d = 1; d < kGsWindow; ++d) m[d] = uint32_t(d) < group ? ld_relaxed(wg - uint64_t(d + 1) * ws) : 0;
      // the nearest group whose state all lanes know, with the maps of all between
      int from = 0;
#pragma unroll
      for (int d = 1; d < kGsWindow; ++d) {
        if (from == 0 && !__all(m[d - 1] != 0)) from = kGsWindow;
        if (from == 0 && __all(gs_word_is_state<F>(m[d]))) from = d;
      }
      done = from > 0 && from < kGsWindow;
      P = 0.0f;
#pragma unroll
      for (int d = kGsWindow - 1; d >= 0; --d)
        if (done && d <= from) P = gs_apply_word<F>(m[d], P);
      if (!done) __builtin_amdgcn_s_sleep(1);
    }
  }
  if (!done && (group > 0 || in > 0)) {
    if (lane == 0) atomicOr(sp.fault, kFaultGatedScanWait);
    P = 0.0f;
  }
  if (last) st_relaxed(wg, gs_pack(gs_none<F>(), gs_apply_word<F>(mine, P)));
#pragma unroll
  for (uint32_t i = 0; i < kGsGroup - 1; ++i)
    if (i < in) P = gs_apply_word<F>(w[i], P);
  return P;
}

// From each thread's segment (A, H) to the state c in front of it.  `P` (thread l: the tile's lane l)
// is the state in front of the first tile; it becomes the one behind this tile.
template <int V, bool SPLIT, class F>
__device__ inline void gs_tile_state(GsTile<V, F>& sm, const F (&A)[V], const float (&H)[V], float (&c)[V], float& P,
                                     const GsSplit& sp, uint32_t chain, uint32_t tile) {
  using G = GsTile<V, F>;
  const int tid = threadIdx.x, lt = tid % kGsLt, seg = tid / kGsLt;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    sm.a[v][tid] = A[v];
    sm.h[v][tid] = H[v];
  }
  lds_barrier();
  // lane l of the tile: element l / 8 of vector l % 8
  const int lane = tid % G::kLanes, part = tid / G::kLanes;
  F* const la = &sm.a[lane / kGsLt][part * G::kPer * kGsLt + lane % kGsLt];
  float* const lh = &sm.h[lane / kGsLt][part * G::kPer * kGsLt + lane % kGsLt];
  F a[G::kPer];
  float h[G::kPer];
#pragma unroll
  for (int i = 0; i < G::kPer; ++i) {
    a[i] = la[i * kGsLt];
    h[i] = lh[i * kGsLt];
  }
  F pa = gs_one<F>();
  float ph = 0.0f;
#pragma unroll
  for (int i = 0; i < G::kPer; ++i) {
    la[i * kGsLt] = pa;
    lh[i * kGsLt] = ph;
    ph = gs_apply(a[i], h[i], ph);
    pa = gs_then(a[i], pa);
  }
  sm.pa[part][lane] = pa;
  sm.ph[part][lane] = ph;
  lds_barrier();
  if (tid < kWave) {  // (of 32 lanes, the wave's other half follows)
    F xa[G::kParts];
    float xh[G::kParts];
#pragma unroll
    for (int i = 0; i < G::kParts; ++i) {
      xa[i] = sm.pa[i][lane];
      xh[i] = sm.ph[i][lane];
    }
    F ta = xa[0];
    float th = xh[0];
#pragma unroll
    for (int i = 1; i < G::kParts; ++i) {
      th = gs_apply(xa[i], xh[i], th);
      ta = gs_then(xa[i], ta);
    }
    if constexpr (SPLIT) P = gs_look_back<G::kLanes, F>(sp, chain, tile, lane, P, ta, th);
    float q = P;
#pragma unroll
    for (int i = 0; i < G::kParts; ++i) {
      sm.c[i][lane] = q;
      q = gs_apply(xa[i], xh[i], q);
    }
    P = q;
  }
  lds_barrier();
  const int mine = seg / G::kPer;
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = gs_apply(sm.a[v][tid], sm.h[v][tid], sm.c[mine][v * kGsLt + lt]);
}

// The tile of a workgroup.  SPLIT: by ticket, in the order of the steps within a shard of chains, so
// that every tile that one waits on was taken before it and is running or done.  false: none left.
template <bool SPLIT>
__device__ inline bool gs_take(const GsSplit& sp, uint32_t& ticket, uint32_t& chain, uint32_t& tile) {
  chain = blockIdx.x;
  tile = 0;
  if constexpr (SPLIT) {
    const uint32_t shard = blockIdx.x - fd_div(sp.sdiv, blockIdx.x) * sp.shards;
    if (threadIdx.x == 0) ticket = atomicAdd(reinterpret_cast<uint32_t*>(sp.counters + shard * kGsCounterWords), 1u);
    __syncthreads();
    const uint32_t t = ticket;
    tile = fd_div(sp.pdiv, t);
    chain = shard * sp.per_shard + (t - tile * sp.per_shard);
    return chain < sp.chains;
  }
  return true;
}

// Where a thread of a tile works: its vector's first lane, and for thread l the tile lane l's state.
template <int V>
struct GsPlace {
  int nl;                // lanes of the vector; 0: none
  bool state_on;
  int64_t off[kGsOps];
  int64_t state;
  __device__ GsPlace(const GsArgs& p, uint32_t chain) {
    const uint32_t q = chain * kGsLt + threadIdx.x % kGsLt;
    const uint32_t qc = q < p.nvec ? q : p.nvec - 1;  // threads past the last vector stand on it and touch nothing
    const uint32_t row = fd_div(p.nvdiv, qc), col = (qc - row * p.nv) * V;
    nl = q >= p.nvec ? 0 : p.D - col < uint32_t(V) ? int(p.D - col) : V;
    gs_row_offsets(p.ix, row, off);
#pragma unroll
    for (int o = 0; o < kGsOps; ++o) off[o] += int64_t(col) * p.ls[o];
    // thread l's vector is the one that lane l belongs to
    const uint32_t e = threadIdx.x % (kGsLt * V) / kGsLt;
    state_on = threadIdx.x < kWave && e < uint32_t(nl);
    state = off[kGsState] + e;
  }
  // all lanes of the chain's vectors are there (the same for the whole workgroup)
  static __device__ bool whole(const GsArgs& p, uint32_t chain) {
    if ((uint64_t(chain) + 1) * kGsLt > p.nvec) return false;
    const uint32_t q = chain * kGsLt, at = q - fd_div(p.nvdiv, q) * p.nv;
    return p.D % V == 0 || at + kGsLt < p.nv;  // (a row's last vector is a part of one)
  }
};

// ---- host side ----------------------------------------------------------------------------------
struct GsPlan {
  GsArgs a;
  uint64_t rows;  // rows of D lanes
  bool lanes;     // the lanes are unit-stride (gate: or shared), resets shared by the lanes
  bool steps;     // the steps are unit-stride (gate, resets: or shared)
};

// Checks and normalises a call; false with the wrapper error set when an argument is out of range.
// Empty calls (no lanes) come back with rows or D equal to 0.
bool gs_plan(const musapy_gated_scan_args* p, bool grad, GsPlan& out);
inline int gs_vector(int dtype) { return dtype == MUSAPY_DT_F32 ? 4 : 8; }  // 16 bytes of x

// The largest power of two of vectors, up to 8, that divides a row of vectors: neighbouring
// threads that sum a shared gate's gradient before it is stored.
inline int gs_part_shift(uint64_t D, int V) {
  const uint64_t nv = (D + V - 1) / V;
  int s = 0;
  while (s < 3 && nv % (uint64_t(2) << s) == 0) ++s;
  return s;
}

// How a call is launched, and the scratch that takes.
struct GsRoute {
  enum Kind { kWalk, kTiles, kRows } kind = kWalk;
  int V = 1;                               // lanes of a thread
  int group = 0;                           // kRows: threads of a row
  uint64_t chains = 0, tiles = 0;
  uint64_t words = 0, group_words = 0;     // of tiles that wait on each other
};
// Chooses the route and splits the lanes into its vectors.
GsRoute gs_route(GsPlan& pl, int dtype);
// Fills `sp` in and clears its words on `st`; false (wrapper error 1) without room for them.
bool gs_split(GsSplit& sp, const GsRoute& r, void* scratch, size_t scratch_bytes, void* workspace, size_t workspace_bytes,
              hipStream_t st);

// Streaming accesses for large calls; not for tiles whose rows' ends share cache lines with their
// neighbours', which the L2 should keep until those come.
inline bool gs_stream(const GsPlan& pl, const GsRoute& r, int dtype) {
  const uint64_t es = dtype == MUSAPY_DT_F32 ? 4 : 2;
  if (r.kind == GsRoute::kTiles && pl.a.ts[kGsOut] * int64_t(es) % 128 != 0) return false;
  return pl.rows * pl.a.D * pl.a.T * es >= kStreamLoadBytes;
}
inline unsigned gs_grid(const GsRoute& r, const GsSplit& sp) {
  if (r.words) return sp.shards * sp.per_shard * sp.tiles;
  return r.kind == GsRoute::kRows ? unsigned((r.chains * r.group + kGsBlock - 1) / kGsBlock) : sp.chains;
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

// Calls fn with a std::bool_constant for each flag.
template <class Fn, class... Known>
inline void gs_flags_from(Fn&& fn, std::tuple<Known...> known) {
  std::apply(fn, known);
}
template <class Fn, class... Known, class... More>
inline void gs_flags_from(Fn&& fn, std::tuple<Known...> known, bool flag, More... more) {
  if (flag) gs_flags_from(fn, std::tuple_cat(known, std::make_tuple(std::true_type{})), more...);
  else gs_flags_from(fn, std::tuple_cat(known, std::make_tuple(std::false_type{})), more...);
}
template <class Fn, class... Flags>
inline void gs_flags(Fn&& fn, Flags... flags) {
  gs_flags_from(fn, std::tuple<>{}, flags...);
}

}  // namespace mpy
