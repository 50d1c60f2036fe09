// dropout.hip -- dropout from a counter-based generator, for gfx950.
#include "kcommon.hpp"
#include "philox.hpp"

namespace mpy {

constexpr int kDropBlock = 256;

struct DropArgs {
  RowIndexer<1> ix;   // all axes but the last
  int64_t ls;         // stride of the last axis
  uint64_t width;
  uint32_t groups;    // groups of 8 columns in a row
  uint32_t total;     // groups in all
  FastDiv gdiv;       // divides a group's number by `groups`
  PhiloxKey key;
  uint32_t threshold;
  float scale;
};

// A thread takes kDropGroups groups of eight columns, one call of the generator each, a workgroup's width
// apart: their loads are all in flight before the first is used.  UNIT: the columns are unit-stride.
// Bound by HBM: (16384, 4096) bf16 47.5 us, 5.6 TB/s (one group a thread 126 us); (2047, 999) f32 out of rows
// of 2048 6.4 us, a launch's time.
constexpr int kDropGroups = 4;

template <class T, bool UNIT, bool NT>
__global__ __launch_bounds__(kDropBlock) void k_dropout(const T* __restrict__ a, T* __restrict__ out, DropArgs p) {
  const uint64_t first = uint64_t(blockIdx.x) * (kDropBlock * kDropGroups) + threadIdx.x;
  Vec<T, 8> w[kDropGroups];
  uint32_t row[kDropGroups], g[kDropGroups];
  int n[kDropGroups];
#pragma unroll
  for (int i = 0; i < kDropGroups; ++i) {
    const uint64_t q = first + uint64_t(i) * kDropBlock;
    n[i] = 0;
    if (q >= p.total) continue;
    row[i] = fd_div(p.gdiv, uint32_t(q));
    g[i] = uint32_t(q) - row[i] * p.groups;
    const uint64_t col = uint64_t(g[i]) * 8;
    n[i] = p.width - col < 8 ? int(p.width - col) : 8;
    int64_t off[1];
    row_offsets<1>(p.ix, row[i], off);
    const T* in = a + off[0] + int64_t(col) * p.ls;
    if (UNIT && n[i] == 8) {
      w[i] = vload_el<T, 8, NT>(in);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n[i]) w[i].v[e] = in[e * p.ls];
    }
  }
#pragma unroll
  for (int i = 0; i < kDropGroups; ++i) {
    if (n[i] == 0) continue;
    const uint32_t keep = philox_keep8(p.key, g[i], row[i], p.threshold);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[i].v[e] = (keep >> e) & 1 ? T(float(w[i].v[e]) * p.scale) : T(0.0f);
    T* o = out + uint64_t(row[i]) * p.width + uint64_t(g[i]) * 8;
    if (n[i] == 8) {
      vstore_el<NT, T, 8>(o, w[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n[i]) o[e] = w[i].v[e];
    }
  }
}

template <class T>
int launch_dropout(const void* a, void* out, int ndim, const size_t* shape, const ssize_t* strides, uint32_t threshold,
                   uint64_t seed, uint64_t offset, hipStream_t st) {
  DropArgs p{};
  for (int i = 0; i < ndim; ++i)
    if (shape[i] == 0) return 0;
  constexpr uint64_t kLimit = uint64_t(1) << 32;  // rows, groups of columns and their product are numbered in 32 bits
  uint64_t rows = 1;
  int n = 0;
  uint64_t size[kMaxDims];
  int64_t stride[kMaxDims];
  auto bad = [] {
    g_wrapper_error = 6;
    return -1;
  };
  for (int i = ndim - 2; i >= 0; --i) {
    if (shape[i] >= kLimit || (rows *= shape[i]) >= kLimit) return bad();
    if (shape[i] == 1) continue;
    if (n > 0 && int64_t(strides[i]) == stride[n - 1] * int64_t(size[n - 1])) {
      size[n - 1] *= shape[i];
      continue;
    }
    size[n] = shape[i];
    stride[n++] = strides[i];
  }
  const uint64_t width = ndim ? shape[ndim - 1] : 1;
  const uint64_t groups = width / 8 + (width % 8 != 0);
  if (groups >= kLimit || groups * rows >= kLimit) return bad();
  const uint64_t grid = (groups * rows + kDropBlock * kDropGroups - 1) / (kDropBlock * kDropGroups);
  if (!grid_fits(grid, kDropBlock)) return bad();
  p.ix.nd = n;
  for (int i = 0; i < n; ++i) {
    p.ix.div[i] = make_fastdiv(uint32_t(size[i]));
    p.ix.stride[0][i] = stride[i];
  }
  p.ls = ndim ? strides[ndim - 1] : 1;
  p.width = width;
  p.groups = uint32_t(groups);
  p.total = uint32_t(groups * rows);
  p.gdiv = make_fastdiv(p.groups);
  p.key = philox_key(seed, offset);
  p.threshold = threshold;
  p.scale = dropout_scale(threshold);
  auto go = [&](auto UNIT, auto NT) {
    k_dropout<T, UNIT.value, NT.value><<<unsigned(grid), kDropBlock, 0, st>>>(static_cast<const T*>(a), static_cast<T*>(out), p);
  };
  if (p.ls != 1 && width > 1) go(std::false_type{}, std::false_type{});
  else if (rows * width * sizeof(T) >= kStreamLoadBytes) go(std::true_type{}, std::true_type{});
  else go(std::true_type{}, std::false_type{});
  return 0;
}

}  // namespace mpy

using namespace mpy;

extern "C" int musapy_dropout_v1(const void* a, void* out, int dtype, int ndim, const size_t* shape, const ssize_t* strides,
                                 uint32_t threshold, uint64_t seed, uint64_t offset, hipStream_t st) {
  if (ndim < 0 || ndim > kMaxDims) {
    g_wrapper_error = 3;
    return -1;
  }
  if (threshold > 65536u || (ndim > 0 && (shape == nullptr || strides == nullptr))) {
    g_wrapper_error = 6;
    return -1;
  }
  bool any = true;
  for (int i = 0; i < ndim; ++i) any = any && shape[i] != 0;
  if (any && (a == nullptr || out == nullptr)) {
    g_wrapper_error = 6;
    return -1;
  }
  if (dtype == MUSAPY_DT_F32) return launch_dropout<float>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  if (dtype == MUSAPY_DT_BF16) return launch_dropout<__bf16>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  if (dtype == MUSAPY_DT_F16) return launch_dropout<_Float16>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  g_wrapper_error = 6;
  return -1;
}
