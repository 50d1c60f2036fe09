// norm_residual.hip -- norms before and after a block with its gate, dropout and residual scale, and
// their gradient, for gfx950.
//
//   n1 = norm(x), u = n1 w1, v = u act(g), d = drop(v), r = res + s d, n2 = norm(r), y = n2 w2
//   D = dr + norm'(r)(dy w2),  dv = drop'(D s),  du = dv act(g),  dx = norm'(x)(du w1),
//   dg = dv u act'(g),  dw1 = sum du n1,  ds = sum D d,  dw2 = sum dy n2
// with norm'(.)(q) = (q - n mean(q n) [- mean(q)]) / deviation, the bracket for layer norms.
#include "kcommon.hpp"
#include "pack.hpp"
#include "philox.hpp"

namespace mpy {

struct NrArgs {
  int post, pre, gate_kind;
  float eps, scale_value;
  uint32_t threshold;
  float keep_scale;
  PhiloxKey key;
  uint32_t rows;
  uint32_t width;
  bool weight_f32;
  const void *x, *res, *gate, *dr, *dy, *w1, *scale, *w2;
  int64_t xp, resp, gatep, drp, dyp;
  void *r, *y, *dx, *dres, *dgate;
  float* part;  // column sums of each workgroup: [workgroup][3][width] (dw1, ds, dw2)
};

// act(g) and its derivative: with m = g (silu) or 1, act = s m and act' = s (1 - s) m [+ s for silu]
__device__ inline void nr_act(int kind, float g, float& a, float& slope) {
  float s, rest;
  sigmoid_pair(g, s, rest);
  const bool silu = kind == MUSAPY_GATE_SILU;
  a = s * (silu ? g : 1.0f);
  slope = __builtin_fmaf(a, rest, silu ? s : 0.0f);
}

template <class T>
__device__ inline float nr_weight(const void* w, bool f32, uint32_t c) {
  if (w == nullptr) return 1.0f;
  return f32 ? static_cast<const float*>(w)[c] : float(static_cast<const T*>(w)[c]);
}

constexpr int kNrBlock = 256;
constexpr int kNrWide = 1024;  // of rows of any width

// Sum over a block of kNrWide, the same for every thread.
__device__ inline float nr_block_sum(float v, float* sm) {
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sm[threadIdx.x / kWave] = v;
  __syncthreads();
  v = sm[threadIdx.x % (kNrWide / kWave)];
  for (int m = kNrWide / kWave / 2; m > 0; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// ---- rows of any width ----------------------------------------------------------------------------
// Rows that do not fit a workgroup's registers are read again for every sum, element by element.  Bound by waits for
// those loads, out of L2, and at the barriers of the sums, three quarters of the waves' time: (2000, 16392) bf16 rms
// 400 us, the gradient at (693, 13056) 336 us, with dropout 361, although that forms eight columns' bits for each one
// and nearly doubles the vector instructions (busy 38% of the time, without it 22%).
template <class T, class TS>
struct NrRow {  // one row of a call, evaluated element by element
  const NrArgs& p;
  uint32_t row;
  float mean1 = 0, inv1 = 1;
  __device__ float x(uint32_t c) const { return float(static_cast<const T*>(p.x)[int64_t(row) * p.xp + c]); }
  __device__ float n1(uint32_t c) const { return (x(c) - mean1) * inv1; }
  __device__ float gate(uint32_t c) const { return float(static_cast<const T*>(p.gate)[int64_t(row) * p.gatep + c]); }
  __device__ float scale(uint32_t c) const { return p.scale_value * nr_weight<T>(p.scale, p.weight_f32, c); }
  __device__ float keep(uint32_t c) const {
    if (p.threshold == 0) return 1.0f;
    return (philox_keep8(p.key, c / 8, row, p.threshold) >> (c % 8)) & 1 ? p.keep_scale : 0.0f;
  }
  __device__ float d(uint32_t c) const {
    float v = n1(c) * nr_weight<T>(p.w1, p.weight_f32, c);
    if (p.gate) {
      float a, s;
      nr_act(p.gate_kind, gate(c), a, s);
      v *= a;
    }
    const float k = keep(c);
    return k == 0.0f ? 0.0f : v * k;
  }
  __device__ float r(uint32_t c) const {
    const float res = p.res ? float(static_cast<const TS*>(p.res)[int64_t(row) * p.resp + c]) : 0.0f;
    return __builtin_fmaf(scale(c), d(c), res);
  }
};

template <class F>
__device__ inline void nr_stats(int kind, uint32_t width, float eps, float* sm, float& mean, float& inv, F&& f) {
  mean = 0.0f;
  inv = 1.0f;
  if (kind == MUSAPY_NORM_NONE) return;
  if (kind == MUSAPY_NORM_LAYER) {
    float s = 0.0f;
    for (uint32_t c = threadIdx.x; c < width; c += kNrWide) s += f(c);
    mean = nr_block_sum(s, sm) / float(width);
  }
  float q = 0.0f;
  for (uint32_t c = threadIdx.x; c < width; c += kNrWide) {
    const float v = f(c) - mean;
    q = __builtin_fmaf(v, v, q);
  }
  inv = 1.0f / sqrtf(nr_block_sum(q, sm) / float(width) + eps);
}

template <class T, class TS>
__global__ __launch_bounds__(kNrWide) void k_nr(NrArgs p) {
  __shared__ float sm[kNrWide / kWave];
  for (uint32_t at = blockIdx.x; at < p.rows; at += gridDim.x) {
    NrRow<T, TS> row{p, at};
    const uint64_t base = uint64_t(at) * p.width;
    nr_stats(p.post, p.width, p.eps, sm, row.mean1, row.inv1, [&](uint32_t c) { return row.x(c); });
    float mean2, inv2;
    nr_stats(p.pre, p.width, p.eps, sm, mean2, inv2, [&](uint32_t c) { return row.r(c); });
    for (uint32_t c = threadIdx.x; c < p.width; c += kNrWide) {
      const float r = row.r(c);
      static_cast<TS*>(p.r)[base + c] = TS(r);
      if (p.y) static_cast<T*>(p.y)[base + c] = T((r - mean2) * inv2 * nr_weight<T>(p.w2, p.weight_f32, c));
    }
  }
}

template <class T, class TS>
__global__ __launch_bounds__(kNrWide) void k_nr_grad(NrArgs p) {
  __shared__ float sm[kNrWide / kWave];
  float* const part = p.part ? p.part + uint64_t(blockIdx.x) * 3 * p.width : nullptr;
  const float over = 1.0f / float(p.width);
  for (uint32_t at = blockIdx.x; at < p.rows; at += gridDim.x) {
    NrRow<T, TS> row{p, at};
    const uint64_t base = uint64_t(at) * p.width;
    nr_stats(p.post, p.width, p.eps, sm, row.mean1, row.inv1, [&](uint32_t c) { return row.x(c); });
    auto r_of = [&](uint32_t c) { return float(static_cast<const TS*>(p.res)[int64_t(at) * p.resp + c]); };
    auto dy_of = [&](uint32_t c) { return p.dy ? float(static_cast<const T*>(p.dy)[int64_t(at) * p.dyp + c]) : 0.0f; };
    float mean2 = 0, inv2 = 1, along2 = 0, flat2 = 0;
    if (p.pre != MUSAPY_NORM_NONE) {
      nr_stats(p.pre, p.width, p.eps, sm, mean2, inv2, r_of);
      float s = 0, q = 0;
      for (uint32_t c = threadIdx.x; c < p.width; c += kNrWide) {
        const float g = dy_of(c) * nr_weight<T>(p.w2, p.weight_f32, c);
        s += g * (r_of(c) - mean2) * inv2;
        q += g;
      }
      along2 = nr_block_sum(s, sm) * over;
      q = nr_block_sum(q, sm) * over;
      flat2 = p.pre == MUSAPY_NORM_LAYER ? q : 0.0f;
    }
    auto total = [&](uint32_t c) {
      float t = p.dr ? float(static_cast<const TS*>(p.dr)[int64_t(at) * p.drp + c]) : 0.0f;
      if (p.pre != MUSAPY_NORM_NONE) {
        const float n2 = (r_of(c) - mean2) * inv2;
        t += inv2 * (dy_of(c) * nr_weight<T>(p.w2, p.weight_f32, c) - n2 * along2 - flat2);
      }
      return t;
    };
    auto dv_of = [&](uint32_t c) {
      const float k = row.keep(c);
      return k == 0.0f ? 0.0f : total(c) * row.scale(c) * k;
    };
    auto back = [&](uint32_t c, float& du, float& dg) {
      const float dv = dv_of(c);
      du = dv;
      dg = 0.0f;
      if (p.gate) {
        float a, slope;
        nr_act(p.gate_kind, row.gate(c), a, slope);
        du = dv * a;
        dg = dv * row.n1(c) * nr_weight<T>(p.w1, p.weight_f32, c) * slope;
      }
    };
    float along1 = 0, flat1 = 0;
    if (p.post != MUSAPY_NORM_NONE) {
      float s = 0, q = 0;
      for (uint32_t c = threadIdx.x; c < p.width; c += kNrWide) {
        float du, dg;
        back(c, du, dg);
        const float g = du * nr_weight<T>(p.w1, p.weight_f32, c);
        s += g * row.n1(c);
        q += g;
      }
      along1 = nr_block_sum(s, sm) * over;
      q = nr_block_sum(q, sm) * over;
      flat1 = p.post == MUSAPY_NORM_LAYER ? q : 0.0f;
    }
    for (uint32_t c = threadIdx.x; c < p.width; c += kNrWide) {
      float du, dg;
      back(c, du, dg);
      const float D = total(c), n1 = row.n1(c);
      if (p.dres) static_cast<TS*>(p.dres)[base + c] = TS(D);
      if (p.dgate) static_cast<T*>(p.dgate)[base + c] = T(dg);
      if (p.dx) {
        float g = du * nr_weight<T>(p.w1, p.weight_f32, c);
        if (p.post != MUSAPY_NORM_NONE) g = row.inv1 * (g - n1 * along1 - flat1);
        static_cast<T*>(p.dx)[base + c] = T(g);
      }
      if (part) {
        const bool first = at == blockIdx.x;
        const float a0 = du * n1, a1 = D * row.d(c) * p.scale_value;
        const float a2 = p.pre != MUSAPY_NORM_NONE ? dy_of(c) * (r_of(c) - mean2) * inv2 : 0.0f;
        part[c] = first ? a0 : part[c] + a0;
        part[p.width + c] = first ? a1 : part[p.width + c] + a1;
        part[2 * uint64_t(p.width) + c] = first ? a2 : part[2 * uint64_t(p.width) + c] + a2;
      }
    }
  }
}

// ---- rows in registers ------------------------------------------------------------------------------
// A thread holds NV vectors of C columns of a row, and a workgroup of as many waves as that takes goes
// from row to row.  With one vector a thread the next row's loads are in flight while this one's is
// summed, and weights and the gradient's column sums stay in registers across rows; with more
// there is no room for that, and the sums stay in LDS.  Forward C = 8, the columns of one call of the random generator; the
// gradient, which holds five inputs, three weights and three sums of a column, C = 4: with 8 it took 180
// registers, one workgroup of 512 a CU.  GL: lanes of a row (16, 32 or a wave's 64, without
// barriers), 0: a workgroup.  LAYER: one of
// the norms is a layer norm.  FULL: the width is a multiple of C, so that every vector is a whole one.

// Sum over a wave, the same in every lane: DPP moves within rows of 16 lanes and across them.
template <int CTRL, int MASK>
__device__ inline float nr_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, MASK, 0xf, false));
}
__device__ inline float nr_wave_sum(float v) {
  v += nr_dpp<0x111, 0xf>(v);  // row_shr:1
  v += nr_dpp<0x112, 0xf>(v);  // row_shr:2
  v += nr_dpp<0x114, 0xf>(v);  // row_shr:4
  v += nr_dpp<0x118, 0xf>(v);  // row_shr:8
  v += nr_dpp<0x142, 0xa>(v);  // row_bcast:15
  v += nr_dpp<0x143, 0xc>(v);  // row_bcast:31
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Sums of N values over the GL lanes of a row, or (GL = 0) over a workgroup's: every wave reads the
// (up to 16) waves' sums with one load and adds them by rotations of 16 lanes.  The two halves of
// `sm` alternate, so that one barrier a sum is enough.
__device__ inline float nr_sum16(float v) {
  v += nr_dpp<0x128, 0xf>(v);  // row_ror:8
  v += nr_dpp<0x124, 0xf>(v);  // row_ror:4
  v += nr_dpp<0x122, 0xf>(v);  // row_ror:2
  v += nr_dpp<0x121, 0xf>(v);  // row_ror:1
  return v;
}
template <int N, int GL>
__device__ inline void nr_sums_of(float (&v)[N], float (*sm)[4][16], int& half, int waves) {
  if constexpr (GL == 16 || GL == 32) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = nr_sum16(v[i]);
      if (GL == 32) v[i] += __shfl_xor(v[i], 16, kWave);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = nr_wave_sum(v[i]);
  if constexpr (GL == 0) {
    const int wv = threadIdx.x / kWave, l = threadIdx.x % 16;
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sm[half][i][wv] = v[i];
    lds_barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = sm[half][i][l];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = nr_sum16(l < waves ? v[i] : 0.0f);
    half ^= 1;
  }
}
// (the hardware's reciprocal square root is within 1 ulp)
__device__ inline float nr_rsqrt(float v) { return __builtin_amdgcn_rsqf(v); }

template <class T, int C, class Place>
__device__ inline void nr_load_weight(const void* w, bool f32, const Place& at, int i, float (&o)[C]) {
  Pack<float, C> p = pack_all<float, C>(at.has(i) ? 1.0f : 0.0f);
  if constexpr (Place::kVectors > 1) asm volatile("" : "+s"(w));  // loaded for each row: kept across rows, they were spilt
  if (w != nullptr && at.has(i)) {
    if (f32) {
      p = pack_load<false, C>(static_cast<const float*>(w) + at.from(i), at.span(i), 0.0f);
      at.put(p, i);
    } else {
      Pack<T, C> q = pack_load<false, C>(static_cast<const T*>(w) + at.from(i), at.span(i), T(0.0f));
      at.put(q, i);
#pragma unroll
      for (int e = 0; e < C; ++e) p.w[e] = __builtin_bit_cast(uint32_t, pack_get(q, e));
    }
  }
#pragma unroll
  for (int e = 0; e < C; ++e) o[e] = pack_get(p, e);
}

// Where a thread works: its row, the rows' step, and its vectors' widths.
template <int C, int NV, int GL, bool FULL>
struct NrPlace {
  static constexpr int kVectors = NV;
  uint32_t t, threads, row, step;
  int waves, n[NV], back[NV];
  __device__ explicit NrPlace(uint32_t width) {
    threads = GL ? GL : blockDim.x;
    waves = int(blockDim.x / kWave);
    t = GL ? threadIdx.x % GL : threadIdx.x;
    const uint32_t per = GL ? blockDim.x / GL : 1;
    // where it is the same for the whole wave, it and the rows' addresses stay in scalar registers
    row = GL == kWave ? blockIdx.x * per + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)
          : GL        ? blockIdx.x * per + threadIdx.x / GL
                      : blockIdx.x;
    step = gridDim.x * per;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = col(i);
      n[i] = c >= width ? 0 : !FULL && width - c < uint32_t(C) ? int(width - c) : C;
      back[i] = !FULL && n[i] && width >= uint32_t(C) ? C - n[i] : 0;
    }
  }
  __device__ uint32_t vec(int i) const { return t + uint32_t(i) * threads; }
  __device__ bool has(int i) const { return n[i] != 0; }
  __device__ int count(int i) const { return FULL ? C : n[i]; }  // where it has one
  __device__ uint32_t col(int i) const { return vec(i) * C; }  // (widths in registers are small: 32-bit offsets)
  // what is loaded for it: a row's last columns in one piece that ends with the row
  __device__ uint32_t from(int i) const { return FULL ? col(i) : col(i) - back[i]; }
  __device__ int span(int i) const { return FULL ? C : n[i] + back[i]; }
  template <class T>
  __device__ void put(Pack<T, C>& p, int i) const {
    if constexpr (!FULL) pack_shift(p, back[i]);
  }
};

// Bound by HBM: (16384, 4096) bf16 with an f32 stream, gate and dropout 169 us, 5.6 TB/s; (16384, 4095) bf16
// 182 us and (16384, 4096) 120 us: stores off 4-byte addresses.
template <class T, class TS, int NV, int BS, int GL, bool LAYER, bool FULL, bool NT>
__global__ __launch_bounds__(BS) void k_nr_rows(NrArgs p) {
  __shared__ float sm[2][4][16];
  const NrPlace<8, NV, GL, FULL> at(p.width);
  int half = 0;
  constexpr bool kAhead = NV == 1;
  const int kind = p.gate ? p.gate_kind : MUSAPY_GATE_SIGMOID;
  float w1[8], sc[8], w2[8];
  auto weights = [&](int i) {
    nr_load_weight<T>(p.w1, p.weight_f32, at, i, w1);
    nr_load_weight<T>(p.scale, p.weight_f32, at, i, sc);
#pragma unroll
    for (int e = 0; e < 8; ++e) sc[e] *= p.scale_value;
  };
  auto pre_weights = [&](int i) { nr_load_weight<T>(p.w2, p.weight_f32, at, i, w2); };
  if (kAhead) {
    weights(0);
    pre_weights(0);
  }
  Pack<T, 8> nx[NV], ng[NV];
  Pack<TS, 8> nres[NV];
  auto load = [&](uint32_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!at.has(i)) continue;
      nx[i] = pack_load<NT, 8>(static_cast<const T*>(p.x) + int64_t(row) * p.xp + at.from(i), at.span(i), T(0.0f));
      if (p.gate) ng[i] = pack_load<NT, 8>(static_cast<const T*>(p.gate) + int64_t(row) * p.gatep + at.from(i), at.span(i), T(0.0f));
      if (p.res) nres[i] = pack_load<NT, 8>(static_cast<const TS*>(p.res) + int64_t(row) * p.resp + at.from(i), at.span(i), TS(0.0f));
    }
  };
  auto fill = [&]() {  // what is not there is zero; no gate: one whose sigmoid is 1
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      nx[i] = pack_all<T, 8>(T(0.0f));
      ng[i] = pack_all<T, 8>(T(p.gate ? 0.0f : __builtin_inff()));
      nres[i] = pack_all<TS, 8>(TS(0.0f));
    }
  };
  fill();
  const float over = 1.0f / float(p.width);
  if (kAhead && at.row < p.rows) load(at.row);
  for (uint32_t row = at.row; row < p.rows; row += at.step) {
    if (!kAhead) {
      fill();  // (kept across rows, it would take the registers that the row is then copied to)
      load(row);
    }
    Pack<T, 8> g[NV];
    Pack<TS, 8> res[NV];
    float u[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Pack<T, 8> x = nx[i];
      g[i] = ng[i];
      res[i] = nres[i];
      at.put(x, i);
      if (p.gate) at.put(g[i], i);
      at.put(res[i], i);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[i][e] = pack_get(x, e);
    }
    if (kAhead && row + at.step < p.rows) load(row + at.step);
    // mean and 1 / deviation of `v`, which is left centred
    auto stats = [&](int kind, float (&v)[NV][8]) {
      if (LAYER && kind == MUSAPY_NORM_LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) s[0] += v[i][e];
        nr_sums_of<1, GL>(s, sm, half, at.waves);
        const float mean = s[0] * over;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[i][e] = e < at.n[i] ? v[i][e] - mean : 0.0f;
      }
      float q[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[0] = __builtin_fmaf(v[i][e], v[i][e], q[0]);
      nr_sums_of<1, GL>(q, sm, half, at.waves);
      return nr_rsqrt(q[0] * over + p.eps);
    };
    const float inv1 = p.post != MUSAPY_NORM_NONE ? stats(p.post, u) : 1.0f;
    const uint64_t base = uint64_t(row) * p.width;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!kAhead) weights(i);
      const uint32_t keep = p.threshold ? philox_keep8(p.key, at.vec(i), row, p.threshold) : 0xffu;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = u[i][e] * inv1 * w1[e];
        const float gv = pack_get(g[i], e);
        float sg, rest;
        sigmoid_pair(gv, sg, rest);
        v *= sg * (kind == MUSAPY_GATE_SILU ? gv : 1.0f);
        v = (keep >> e) & 1 ? v * p.keep_scale : 0.0f;
        u[i][e] = __builtin_fmaf(sc[e], v, pack_get(res[i], e));
      }
      if (at.has(i)) pack_store<NT>(static_cast<TS*>(p.r) + base + at.col(i), at.count(i), u[i]);
    }
    if (p.y) {
      const float inv2 = stats(p.pre, u);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!kAhead) pre_weights(i);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[i][e] = u[i][e] * inv2 * w2[e];
        if (at.has(i)) pack_store<NT>(static_cast<T*>(p.y) + base + at.col(i), at.count(i), u[i]);
      }
    }
  }
}

// The gradient.  With m the mean (0 for rms norms) the sums that depend on the row's inputs alone,
// (x - m)^2, (r - m)^2, dy w2 (r - m) and dy w2, are formed in one round; those of the post norm's input
// gradient, which need D, in a second.  Bound by HBM and by the 16 waves a CU that its registers leave:
// (8192, 4096) bf16 with dropout 109 us with the column sums, 4.9 TB/s; (5003, 1111) f32 layer norms 58 us,
// 3.1 TB/s, on rows off lines; (4096, 8192) bf16 with dropout 153 us, 3.5 TB/s.
template <class T, class TS, int NV, int BS, int GL, bool LAYER, bool FULL, bool NT>
__global__ __launch_bounds__(BS) void k_nr_grad_rows(NrArgs p) {
  __shared__ float sm[2][4][16];
  constexpr int C = 4;
  const NrPlace<C, NV, GL, FULL> at(p.width);
  int half = 0;
  constexpr bool kAhead = NV == 1;
  const int kind = p.gate ? p.gate_kind : MUSAPY_GATE_SIGMOID;
  // The column sums: in registers, or, with more vectors, each thread's in LDS.
  constexpr bool kLds = NV > 1;
  float w1[C], sc[C], w2[C], a1[C], as[C], a2[C];
  __shared__ float4 s_sums[kLds ? 3 * NV : 1][kLds ? BS : 1];
  auto sums = [&](int i, bool store) {
    if constexpr (kLds) {
      float* const to[3] = {a1, as, a2};
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        float4& q = s_sums[3 * i + j][threadIdx.x];
        if (store) {
          q = float4{to[j][0], to[j][1], to[j][2], to[j][3]};
        } else {
          const float4 v = q;
          to[j][0] = v.x;
          to[j][1] = v.y;
          to[j][2] = v.z;
          to[j][3] = v.w;
        }
      }
    }
  };
  auto weights = [&](int i) {
    nr_load_weight<T>(p.w1, p.weight_f32, at, i, w1);
    nr_load_weight<T>(p.scale, p.weight_f32, at, i, sc);
#pragma unroll
    for (int e = 0; e < C; ++e) sc[e] *= p.scale_value * p.keep_scale;
  };
  auto pre_weights = [&](int i) { nr_load_weight<T>(p.w2, p.weight_f32, at, i, w2); };
  if (kAhead) {
    weights(0);
    pre_weights(0);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < C; ++e) a1[e] = as[e] = a2[e] = 0.0f;
    sums(i, true);
  }
  const bool pre = p.pre != MUSAPY_NORM_NONE;
  Pack<T, C> nx[NV], ng[NV], ny[NV];
  Pack<TS, C> nr[NV], nd[NV];
  auto load = [&](uint32_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (!at.has(i)) continue;
      nx[i] = pack_load<NT, C>(static_cast<const T*>(p.x) + int64_t(row) * p.xp + at.from(i), at.span(i), T(0.0f));
      if (p.gate) ng[i] = pack_load<NT, C>(static_cast<const T*>(p.gate) + int64_t(row) * p.gatep + at.from(i), at.span(i), T(0.0f));
      if (pre) nr[i] = pack_load<NT, C>(static_cast<const TS*>(p.res) + int64_t(row) * p.resp + at.from(i), at.span(i), TS(0.0f));
      if (p.dr) nd[i] = pack_load<NT, C>(static_cast<const TS*>(p.dr) + int64_t(row) * p.drp + at.from(i), at.span(i), TS(0.0f));
      if (p.dy) ny[i] = pack_load<NT, C>(static_cast<const T*>(p.dy) + int64_t(row) * p.dyp + at.from(i), at.span(i), T(0.0f));
    }
  };
  auto fill = [&]() {  // what is not there is zero; no gate: one whose sigmoid is 1
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      nx[i] = ny[i] = pack_all<T, C>(T(0.0f));
      ng[i] = pack_all<T, C>(T(p.gate ? 0.0f : __builtin_inff()));
      nr[i] = nd[i] = pack_all<TS, C>(TS(0.0f));
    }
  };
  fill();
  const int shift = at.t % 2 * C;
  uint32_t keeps[NV], later[NV];
  bool spare = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) keeps[i] = later[i] = 0xffu;
  const float over = 1.0f / float(p.width);
  if (kAhead && at.row < p.rows) load(at.row);
  for (uint32_t row = at.row; row < p.rows; row += at.step) {
    if (!kAhead) {
      fill();  // (kept across rows, it would take the registers that the row is then copied to)
      load(row);
    }
    Pack<T, C> x[NV], g[NV], y[NV];
    Pack<TS, C> r[NV], d[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = nx[i];
      g[i] = ng[i];
      y[i] = ny[i];
      r[i] = nr[i];
      d[i] = nd[i];
      at.put(x[i], i);
      if (p.gate) at.put(g[i], i);
      at.put(y[i], i);
      at.put(r[i], i);
      at.put(d[i], i);
    }
    if (kAhead && row + at.step < p.rows) load(row + at.step);
    float m1 = 0.0f, m2 = 0.0f;
    if constexpr (LAYER) {
      float s[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < C; ++e) {
          s[0] += pack_get(x[i], e);
          s[1] += pack_get(r[i], e);
        }
      nr_sums_of<2, GL>(s, sm, half, at.waves);
      if (p.post == MUSAPY_NORM_LAYER) m1 = s[0] * over;
      if (p.pre == MUSAPY_NORM_LAYER) m2 = s[1] * over;
    }
    // (columns that are not there hold zeros, and stay zeros when centred)
    auto xc = [&](int i, int e) {
      const float v = pack_get(x[i], e);
      return !LAYER ? v : e < at.n[i] ? v - m1 : 0.0f;
    };
    auto rc = [&](int i, int e) {
      const float v = pack_get(r[i], e);
      return !LAYER ? v : e < at.n[i] ? v - m2 : 0.0f;
    };
    auto dy = [&](int i, int e) { return pack_get(y[i], e); };
    float inv1 = 1.0f, inv2 = 1.0f, along2 = 0.0f, flat2 = 0.0f;
    if (pre || p.post != MUSAPY_NORM_NONE) {
      float s[LAYER ? 4 : 3] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!kAhead) {
          __builtin_amdgcn_sched_barrier(0);  // else every vector's weights are loaded first, and spilt
          pre_weights(i);
        }
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float a = xc(i, e), b = rc(i, e), q = dy(i, e) * w2[e];
          s[0] = __builtin_fmaf(a, a, s[0]);
          s[1] = __builtin_fmaf(b, b, s[1]);
          s[2] = __builtin_fmaf(q, b, s[2]);
          if constexpr (LAYER) s[3] += q;
        }
        pack_opaque(x[i]);
        pack_opaque(r[i]);
        pack_opaque(y[i]);
      }
      nr_sums_of<LAYER ? 4 : 3, GL>(s, sm, half, at.waves);
      if (p.post != MUSAPY_NORM_NONE) inv1 = nr_rsqrt(s[0] * over + p.eps);
      if (pre) {
        inv2 = nr_rsqrt(s[1] * over + p.eps);
        along2 = s[2] * inv2 * over;
        if constexpr (LAYER)
          if (p.pre == MUSAPY_NORM_LAYER) flat2 = s[3] * over;
      }
    }
    // A call of the generator covers two threads' columns: of each pair one forms this row's bits and the
    // other the next row's, and both use both.
    if (p.threshold) {
      if (!spare) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const uint32_t k = philox_keep8(p.key, at.vec(i) / 2, at.t % 2 ? row + at.step : row, p.threshold);
          keeps[i] = uint32_t(__builtin_amdgcn_update_dpp(0, int(k), 0xa0, 0xf, 0xf, true));  // quad_perm 0, 0, 2, 2
          later[i] = uint32_t(__builtin_amdgcn_update_dpp(0, int(k), 0xf5, 0xf, 0xf, true));  // quad_perm 1, 1, 3, 3
        }
      } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) keeps[i] = later[i];
      }
      spare = !spare;
    }
    const uint64_t base = uint64_t(row) * p.width;
    float q1[NV][C], s2[LAYER ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t keep = keeps[i] >> shift;
      float D[C], dg[C];
      if (!kAhead) {
        __builtin_amdgcn_sched_barrier(0);
        weights(i);
        pre_weights(i);
      }
      sums(i, false);
#pragma unroll
      for (int e = 0; e < C; ++e) {
        const float n1 = xc(i, e) * inv1, n2 = rc(i, e) * inv2, y1 = dy(i, e);
        float q = __builtin_fmaf(-n2, along2, y1 * w2[e]);
        if constexpr (LAYER) q = e < at.n[i] ? q - flat2 : 0.0f;
        D[e] = __builtin_fmaf(inv2, q, pack_get(d[i], e));
        const float Dk = (keep >> e) & 1 ? D[e] : 0.0f;
        float act, slope;
        nr_act(kind, pack_get(g[i], e), act, slope);
        const float dv = Dk * sc[e], u = n1 * w1[e];
        const float du = dv * act;
        dg[e] = dv * u * slope;
        a1[e] = __builtin_fmaf(du, n1, a1[e]);
        as[e] = (keep >> e) & 1 ? __builtin_fmaf(Dk, u * act, as[e]) : as[e];
        a2[e] = __builtin_fmaf(y1, n2, a2[e]);
        q1[i][e] = du * w1[e];
        s2[0] = __builtin_fmaf(q1[i][e], n1, s2[0]);
        if constexpr (LAYER) s2[1] += q1[i][e];
      }
      sums(i, true);
      if (p.dres && at.has(i)) pack_store<NT>(static_cast<TS*>(p.dres) + base + at.col(i), at.count(i), D);
      if (p.dgate && at.has(i)) pack_store<NT>(static_cast<T*>(p.dgate) + base + at.col(i), at.count(i), dg);
      pack_opaque(x[i]);
    }
    if (p.post != MUSAPY_NORM_NONE) {
      nr_sums_of<LAYER ? 2 : 1, GL>(s2, sm, half, at.waves);
      const float along1 = s2[0] * over * inv1;
      float flat1 = 0.0f;
      if constexpr (LAYER)
        if (p.post == MUSAPY_NORM_LAYER) flat1 = s2[1] * over;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < C; ++e) q1[i][e] = inv1 * (__builtin_fmaf(-xc(i, e), along1, q1[i][e]) - flat1);
    }
    if (p.dx)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at.has(i)) pack_store<NT>(static_cast<T*>(p.dx) + base + at.col(i), at.count(i), q1[i]);
  }
  if (p.part == nullptr) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    sums(i, false);
    if constexpr (GL != 0) {  // the rows of a workgroup, in order
      __shared__ float s_rows[3 * C][BS];
#pragma unroll
      for (int e = 0; e < C; ++e) {
        s_rows[e][threadIdx.x] = a1[e];
        s_rows[C + e][threadIdx.x] = as[e];
        s_rows[2 * C + e][threadIdx.x] = a2[e];
        a1[e] = as[e] = a2[e] = 0.0f;
      }
      __syncthreads();
      if (threadIdx.x >= GL) return;
      for (int r = 0; r < BS / GL; ++r)
#pragma unroll
        for (int e = 0; e < C; ++e) {
          a1[e] += s_rows[e][r * GL + threadIdx.x];
          as[e] += s_rows[C + e][r * GL + threadIdx.x];
          a2[e] += s_rows[2 * C + e][r * GL + threadIdx.x];
        }
    }
#pragma unroll
    for (int e = 0; e < C; ++e) as[e] *= p.scale_value * p.keep_scale;
    if (!at.has(i)) continue;
    float* const part = p.part + uint64_t(blockIdx.x) * 3 * p.width;
    pack_store<false>(part + at.col(i), at.count(i), a1);
    pack_store<false>(part + p.width + at.col(i), at.count(i), as);
    pack_store<false>(part + 2 * uint64_t(p.width) + at.col(i), at.count(i), a2);
  }
}

// Column sums over the workers' partial sums: 64 columns a workgroup, each of its sixteen waves a part of
// the workers, joined in order.  256 workers' three sums of 4096 columns 4.7 us, little more than a launch.
constexpr int kNrColumnWaves = 16;
template <class T>
__global__ __launch_bounds__(kNrColumnWaves * kWave) void k_nr_columns(const float* part, uint32_t workers, uint32_t width, bool f32, void* o0,
                                                         void* o1, void* o2) {
  __shared__ float sm[kNrColumnWaves][kWave];
  void* const o = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (o == nullptr) return;
  const uint32_t l = threadIdx.x % kWave, wv = threadIdx.x / kWave;
  const uint32_t c = blockIdx.x * kWave + l;
  const uint32_t per = (workers + kNrColumnWaves - 1) / kNrColumnWaves;
  const uint32_t from = wv * per, to = from + per < workers ? from + per : workers;
  float s[8] = {};
  if (c < width) {
    const float* q = part + uint64_t(blockIdx.y) * width + c;
    const uint64_t step = 3 * uint64_t(width);
    uint32_t b = from;
    for (; b + 8 <= to; b += 8)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += q[(b + i) * step];
    for (; b < to; ++b) s[0] += q[b * step];
  }
  sm[wv][l] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  if (wv != 0 || c >= width) return;
  float v = 0.0f;
#pragma unroll
  for (int i = 0; i < kNrColumnWaves; ++i) v += sm[i][l];
  if (f32) static_cast<float*>(o)[c] = v;
  else static_cast<T*>(o)[c] = T(v);
}

namespace {

// How the rows of a call are spread: `threads` to a workgroup, `blocks` of them.
struct NrRoute {
  int nv = 0;  // vectors to a thread; 0: the kernels for any width
  int lanes = 0;  // of a row; 0: a workgroup
  unsigned threads = kNrBlock, blocks = 0;
  uint32_t workers = 0;
};
NrRoute nr_route(const musapy_norm_residual_args* p, bool grad) {
  NrRoute r;
  const uint64_t vecs = grad ? (p->width + 3) / 4 : (p->width + 7) / 8;
  const uint64_t rows = p->rows;
  if (p->width > (grad ? 12288 : 16384)) {
    r.threads = kNrWide;
    // four times what the CUs hold at a time: a workgroup a row would pass a grid's 2^32 threads from 2^22 rows on
    const uint64_t most = grad ? 512 : 2048;
    r.blocks = r.workers = unsigned(rows < most ? rows : most);
    return r;
  }
  if (vecs <= kWave) {
    r.nv = 1;
    r.lanes = vecs <= 16 ? 16 : vecs <= 32 ? 32 : kWave;
    const uint64_t most = grad ? 512 : 2048, want = (rows * r.lanes + kNrBlock - 1) / kNrBlock;
    r.blocks = r.workers = unsigned(want < most ? want : most);
    return r;
  }
  r.nv = int((vecs + 1023) / 1024);
  r.threads = unsigned((vecs + r.nv * kWave - 1) / (r.nv * kWave) * kWave);
  // forward: about eight rows a workgroup, so that weights are loaded once for them; gradient: as many
  // workgroups as the CUs hold at a time (1024 threads of its registers each), since each leaves a row of
  // column sums.  Either way with as even a number of rows as there can be.
  const uint64_t most = grad ? uint64_t(256) * (1024 / r.threads) : rows < 8192 ? 1024 : (rows + 7) / 8;
  const uint64_t per = (rows + most - 1) / most;
  r.blocks = r.workers = unsigned(per ? (rows + per - 1) / per : 0);
  return r;
}

int nr_bad() {
  g_wrapper_error = 6;
  return -1;
}

int nr_args(const musapy_norm_residual_args* p, NrArgs& a) {
  if (p == nullptr) return nr_bad();
  auto dt = [](int d) { return d == MUSAPY_DT_F32 || d == MUSAPY_DT_F16 || d == MUSAPY_DT_BF16; };
  auto kind = [](int k) { return k >= MUSAPY_NORM_NONE && k <= MUSAPY_NORM_LAYER; };
  if (!dt(p->dtype) || (p->stream_dtype != p->dtype && p->stream_dtype != MUSAPY_DT_F32) ||
      (p->weight_dtype != p->dtype && p->weight_dtype != MUSAPY_DT_F32) || !kind(p->post) || !kind(p->pre) ||
      (p->gate && p->gate_kind != MUSAPY_GATE_SILU && p->gate_kind != MUSAPY_GATE_SIGMOID) || p->threshold > 65536u ||
      p->rows >= (uint64_t(1) << 31) || p->width >= (uint64_t(1) << 31))
    return nr_bad();
  a = NrArgs{};
  a.post = p->post;
  a.pre = p->pre;
  a.gate_kind = p->gate_kind;
  a.eps = p->eps;
  a.scale_value = p->scale_value;
  a.threshold = p->threshold;
  a.keep_scale = dropout_scale(p->threshold);
  a.key = philox_key(p->seed, p->offset);
  a.rows = uint32_t(p->rows);
  a.width = uint32_t(p->width);
  a.weight_f32 = p->weight_dtype == MUSAPY_DT_F32;
  a.x = p->x;
  a.xp = int64_t(p->x_pitch);
  a.res = p->residual;
  a.resp = int64_t(p->residual_pitch);
  a.gate = p->gate;
  a.gatep = int64_t(p->gate_pitch);
  a.dr = p->dr;
  a.drp = int64_t(p->dr_pitch);
  a.dy = p->dy;
  a.dyp = int64_t(p->dy_pitch);
  a.w1 = p->post_weight;
  a.scale = p->scale;
  a.w2 = p->pre_weight;
  a.r = p->r;
  a.y = p->pre == MUSAPY_NORM_NONE ? nullptr : p->y;
  a.dx = p->dx;
  a.dres = p->dresidual;
  a.dgate = p->dgate;
  return 0;
}

// Calls fn(T{}, TS{}) with the element types of the block and of the residual stream.
template <class Fn>
void nr_types(int dtype, int stream_dtype, Fn&& fn) {
  if (dtype == MUSAPY_DT_F32) return fn(float{}, float{});
  if (dtype == MUSAPY_DT_BF16) {
    if (stream_dtype == MUSAPY_DT_F32) return fn(bf16{}, float{});
    return fn(bf16{}, bf16{});
  }
  if (stream_dtype == MUSAPY_DT_F32) return fn(f16{}, float{});
  return fn(f16{}, f16{});
}

bool nr_sums(const musapy_norm_residual_args* p) { return p->dpost_weight || p->dscale || p->dpre_weight; }

// Calls fn with (NV, BS, GL, LAYER, FULL, NT) of the kernel for a call.
template <int C, class Fn>
void nr_kernel(const NrRoute& r, const NrArgs& a, Fn&& fn) {
  using std::false_type;
  using std::integral_constant;
  using std::true_type;
  const bool layer = a.post == MUSAPY_NORM_LAYER || a.pre == MUSAPY_NORM_LAYER;
  const bool nt = uint64_t(a.rows) * a.width * 8 >= kStreamLoadBytes;
  auto more = [&](auto nv, auto bs, auto gl) {
    with_store_policy(layer, [&](auto LAYER) {
      if (a.width % C) fn(nv, bs, gl, LAYER, false_type{}, false_type{});
      else if (nt) fn(nv, bs, gl, LAYER, true_type{}, true_type{});
      else fn(nv, bs, gl, LAYER, true_type{}, false_type{});
    });
  };
  using One = integral_constant<int, 1>;
  using Block = integral_constant<int, 0>;
  if (r.lanes == 16) more(One{}, integral_constant<int, kNrBlock>{}, integral_constant<int, 16>{});
  else if (r.lanes == 32) more(One{}, integral_constant<int, kNrBlock>{}, integral_constant<int, 32>{});
  else if (r.lanes == kWave) more(One{}, integral_constant<int, kNrBlock>{}, integral_constant<int, kWave>{});
  else if (r.nv == 1 && r.threads <= 512) more(One{}, integral_constant<int, 512>{}, Block{});
  else if (r.nv == 1) more(One{}, integral_constant<int, 1024>{}, Block{});
  else if (r.nv == 2) more(integral_constant<int, 2>{}, integral_constant<int, 1024>{}, Block{});
  else if constexpr (C == 4) more(integral_constant<int, 3>{}, integral_constant<int, 1024>{}, Block{});
}

}  // namespace

}  // namespace mpy

using namespace mpy;

extern "C" {

size_t musapy_norm_residual_scratch_v1(const musapy_norm_residual_args* p) {
  if (p == nullptr || !nr_sums(p)) return 0;
  return size_t(nr_route(p, true).workers) * 3 * p->width * sizeof(float);
}

int musapy_norm_residual_v1(const musapy_norm_residual_args* p, hipStream_t st) {
  NrArgs a;
  if (nr_args(p, a) != 0) return -1;
  if (a.rows == 0 || a.width == 0) return 0;
  if (a.x == nullptr || a.r == nullptr) return nr_bad();
  const NrRoute r = nr_route(p, false);
  if (!grid_fits(r.blocks, r.threads)) return nr_bad();
  nr_types(p->dtype, p->stream_dtype, [&](auto t, auto ts) {
    using T = decltype(t);
    using TS = decltype(ts);
    if (r.nv == 0) k_nr<T, TS><<<r.blocks, r.threads, 0, st>>>(a);
    else
      nr_kernel<8>(r, a, [&](auto NV, auto BS, auto GL, auto LAYER, auto FULL, auto NT) {
        k_nr_rows<T, TS, NV.value, BS.value, GL.value, LAYER.value, FULL.value, NT.value><<<r.blocks, r.threads, 0, st>>>(a);
      });
  });
  return 0;
}

int musapy_norm_residual_grad_v1(const musapy_norm_residual_args* p, void* scratch, size_t scratch_bytes, hipStream_t st) {
  NrArgs a;
  if (nr_args(p, a) != 0) return -1;
  if (a.width == 0) return 0;
  if (a.rows > 0 && (a.x == nullptr || (a.pre != MUSAPY_NORM_NONE && a.res == nullptr))) return nr_bad();
  if (a.pre == MUSAPY_NORM_NONE) a.dy = nullptr;
  const NrRoute r = nr_route(p, true);
  if (nr_sums(p) && r.workers > 0) {
    if (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < musapy_norm_residual_scratch_v1(p)) {
      g_wrapper_error = 1;
      return -1;
    }
    a.part = static_cast<float*>(scratch);
  }
  nr_types(p->dtype, p->stream_dtype, [&](auto t, auto ts) {
    using T = decltype(t);
    using TS = decltype(ts);
    if (r.blocks > 0 && r.nv == 0) k_nr_grad<T, TS><<<r.blocks, r.threads, 0, st>>>(a);
    else if (r.blocks > 0)
      nr_kernel<4>(r, a, [&](auto NV, auto BS, auto GL, auto LAYER, auto FULL, auto NT) {
        k_nr_grad_rows<T, TS, NV.value, BS.value, GL.value, LAYER.value, FULL.value, NT.value>
            <<<r.blocks, r.threads, 0, st>>>(a);
      });
    if (nr_sums(p))
      k_nr_columns<T><<<dim3((a.width + kWave - 1) / kWave, 3), kNrColumnWaves * kWave, 0, st>>>(
          a.part, r.workers, a.width, a.weight_f32, p->dpost_weight, p->dscale, p->dpre_weight);
  });
  return 0;
}

}  // extern "C"
