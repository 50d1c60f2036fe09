// norm_residual.hip -- norms before and after a block with its gate, dropout and residual scale, and
// their gradient, for gfx950.
//
//   n1 = norm(x), u = n1 w1, v = u act(g), d = drop(v), r = res + s d, n2 = norm(r), y = n2 w2
//   D = dr + norm'(r)(dy w2),  dv = drop'(D s),  du = dv act(g),  dx = norm'(x)(du w1),
//   dg = dv u act'(g),  dw1 = sum du n1,  ds = sum D d,  dw2 = sum dy n2
// with norm'(.)(q) = (q - n mean(q n) [- mean(q)]) / deviation, the bracket for layer norms.
#include "kcommon.hpp"
#include "philox.hpp"

namespace mpy {

using bf16 = __bf16;
using f16 = _Float16;

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
  float* part;       // column sums of each block: [block][3][width] (dw1, ds, dw2)
};

__device__ inline float nr_sigmoid(float g) {
  const float e = __builtin_amdgcn_exp2f(-1.44269504f * __builtin_fabsf(g));
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return g >= 0.0f ? r : e * r;
}
// act(g) and its derivative
__device__ inline void nr_act(int kind, float g, float& a, float& slope) {
  const float s = nr_sigmoid(g), rest = nr_sigmoid(-g);
  if (kind == MUSAPY_GATE_SILU) {
    a = g * s;
    slope = __builtin_fmaf(a, rest, s);
  } else {
    a = s;
    slope = s * rest;
  }
}

template <class T>
__device__ inline float nr_weight(const void* w, bool f32, uint32_t c) {
  if (w == nullptr) return 1.0f;
  return f32 ? static_cast<const float*>(w)[c] : float(static_cast<const T*>(w)[c]);
}

// Sum over a block of 256, the same for every thread.
__device__ inline float nr_block_sum(float v, float* sm) {
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, kWave);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sm[threadIdx.x / kWave] = v;
  __syncthreads();
  return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

constexpr int kNrBlock = 256;

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
    for (uint32_t c = threadIdx.x; c < width; c += kNrBlock) s += f(c);
    mean = nr_block_sum(s, sm) / float(width);
  }
  float q = 0.0f;
  for (uint32_t c = threadIdx.x; c < width; c += kNrBlock) {
    const float v = f(c) - mean;
    q = __builtin_fmaf(v, v, q);
  }
  inv = 1.0f / sqrtf(nr_block_sum(q, sm) / float(width) + eps);
}

template <class T, class TS>
__global__ __launch_bounds__(kNrBlock) void k_nr(NrArgs p) {
  __shared__ float sm[kNrBlock / kWave];
  NrRow<T, TS> row{p, blockIdx.x};
  const uint64_t base = uint64_t(blockIdx.x) * p.width;
  nr_stats(p.post, p.width, p.eps, sm, row.mean1, row.inv1, [&](uint32_t c) { return row.x(c); });
  float mean2, inv2;
  nr_stats(p.pre, p.width, p.eps, sm, mean2, inv2, [&](uint32_t c) { return row.r(c); });
  for (uint32_t c = threadIdx.x; c < p.width; c += kNrBlock) {
    const float r = row.r(c);
    static_cast<TS*>(p.r)[base + c] = TS(r);
    if (p.y) static_cast<T*>(p.y)[base + c] = T((r - mean2) * inv2 * nr_weight<T>(p.w2, p.weight_f32, c));
  }
}

template <class T, class TS>
__global__ __launch_bounds__(kNrBlock) void k_nr_grad(NrArgs p) {
  __shared__ float sm[kNrBlock / kWave];
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
      for (uint32_t c = threadIdx.x; c < p.width; c += kNrBlock) {
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
      for (uint32_t c = threadIdx.x; c < p.width; c += kNrBlock) {
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
    for (uint32_t c = threadIdx.x; c < p.width; c += kNrBlock) {
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

// Column sums over the blocks' partial sums, in the blocks' order.
template <class T>
__global__ __launch_bounds__(kNrBlock) void k_nr_columns(const float* part, uint32_t blocks, uint32_t width, bool f32, void* o0,
                                                         void* o1, void* o2) {
  const uint32_t c = blockIdx.x * kNrBlock + threadIdx.x;
  void* const o = blockIdx.y == 0 ? o0 : blockIdx.y == 1 ? o1 : o2;
  if (c >= width || o == nullptr) return;
  float s = 0.0f;
  for (uint32_t b = 0; b < blocks; ++b) s += part[(uint64_t(b) * 3 + blockIdx.y) * width + c];
  if (f32) static_cast<float*>(o)[c] = s;
  else static_cast<T*>(o)[c] = T(s);
}

namespace {

constexpr uint32_t kNrGradBlocks = 512;

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

uint32_t nr_grad_blocks(const musapy_norm_residual_args* p) {
  return uint32_t(p->rows < kNrGradBlocks ? p->rows : kNrGradBlocks);
}

}  // namespace

}  // namespace mpy

using namespace mpy;

extern "C" {

size_t musapy_norm_residual_scratch_v1(const musapy_norm_residual_args* p) {
  if (p == nullptr || !nr_sums(p)) return 0;
  return size_t(nr_grad_blocks(p)) * 3 * p->width * sizeof(float);
}

int musapy_norm_residual_v1(const musapy_norm_residual_args* p, hipStream_t st) {
  NrArgs a;
  if (nr_args(p, a) != 0) return -1;
  if (a.rows == 0 || a.width == 0) return 0;
  if (a.x == nullptr || a.r == nullptr) return nr_bad();
  nr_types(p->dtype, p->stream_dtype, [&](auto t, auto ts) {
    k_nr<decltype(t), decltype(ts)><<<a.rows, kNrBlock, 0, st>>>(a);
  });
  return 0;
}

int musapy_norm_residual_grad_v1(const musapy_norm_residual_args* p, void* scratch, size_t scratch_bytes, hipStream_t st) {
  NrArgs a;
  if (nr_args(p, a) != 0) return -1;
  if (a.width == 0) return 0;
  if (a.rows > 0 && (a.x == nullptr || (a.pre != MUSAPY_NORM_NONE && a.res == nullptr))) return nr_bad();
  if (a.pre == MUSAPY_NORM_NONE) a.dy = nullptr;
  const uint32_t blocks = nr_grad_blocks(p);
  if (nr_sums(p) && blocks > 0) {
    if (scratch == nullptr || (reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < musapy_norm_residual_scratch_v1(p)) {
      g_wrapper_error = 1;
      return -1;
    }
    a.part = static_cast<float*>(scratch);
  }
  nr_types(p->dtype, p->stream_dtype, [&](auto t, auto ts) {
    if (blocks > 0) k_nr_grad<decltype(t), decltype(ts)><<<blocks, kNrBlock, 0, st>>>(a);
    if (nr_sums(p))
      k_nr_columns<decltype(t)><<<dim3((a.width + kNrBlock - 1) / kNrBlock, 3), kNrBlock, 0, st>>>(
          a.part, blocks, a.width, a.weight_f32, p->dpost_weight, p->dscale, p->dpre_weight);
  });
  return 0;
}

}  // extern "C"
