// dropout.hip -- dropout from a counter-based generator, for gfx950.
#include "kcommon.hpp"
#include "philox.hpp"

namespace mpy {

constexpr int kDropBlock = 256;

struct DropArgs {
  RowIndexer<1> ix;   // all axes but the last
  int64_t ls;         // stride of the last axis
  uint32_t width;
  uint32_t groups;    // groups of 8 columns in a row
  uint32_t total;     // groups in all
  FastDiv gdiv;       // divides a group's number by `groups`
  PhiloxKey key;
  uint32_t threshold;
  float scale;
};

// One thread per group of eight columns: one call of the generator.
template <class T>
__global__ __launch_bounds__(kDropBlock) void k_dropout(const T* __restrict__ a, T* __restrict__ out, DropArgs p) {
  const uint64_t q = uint64_t(blockIdx.x) * kDropBlock + threadIdx.x;
  if (q >= p.total) return;
  const uint32_t row = fd_div(p.gdiv, uint32_t(q));
  const uint32_t g = uint32_t(q) - row * p.groups;
  const uint64_t col = uint64_t(g) * 8;
  int64_t off[1];
  row_offsets<1>(p.ix, row, off);
  const T* in = a + off[0] + int64_t(col) * p.ls;
  T* o = out + uint64_t(row) * p.width + col;
  const uint32_t keep = philox_keep8(p.key, g, row, p.threshold);
  const int n = p.width - col < 8 ? int(p.width - col) : 8;
  for (int e = 0; e < n; ++e) o[e] = (keep >> e) & 1 ? T(float(in[e * p.ls]) * p.scale) : T(0.0f);
}

template <class T>
int launch_dropout(const void* a, void* out, int ndim, const size_t* shape, const ssize_t* strides, uint32_t threshold,
                   uint64_t seed, uint64_t offset, hipStream_t st) {
  DropArgs p{};
  uint64_t rows = 1;
  int n = 0;
  uint64_t size[kMaxDims];
  int64_t stride[kMaxDims];
  for (int i = ndim - 2; i >= 0; --i) {
    rows *= shape[i];
    if (shape[i] == 1) continue;
    if (n > 0 && int64_t(strides[i]) == stride[n - 1] * int64_t(size[n - 1])) {
      size[n - 1] *= shape[i];
      continue;
    }
    size[n] = shape[i];
    stride[n++] = strides[i];
  }
  const uint64_t width = ndim ? shape[ndim - 1] : 1;
  if (rows == 0 || width == 0) return 0;
  const uint64_t groups = (width + 7) / 8;
  // rows and groups are numbered in 32 bits
  if (rows >= (uint64_t(1) << 32) || width >= (uint64_t(1) << 32) || groups * rows >= (uint64_t(1) << 32) ||
      !grid_fits((groups * rows + kDropBlock - 1) / kDropBlock, kDropBlock)) {
    g_wrapper_error = 6;
    return -1;
  }
  p.ix.nd = n;
  for (int i = 0; i < n; ++i) {
    p.ix.div[i] = make_fastdiv(uint32_t(size[i]));
    p.ix.stride[0][i] = stride[i];
  }
  p.ls = ndim ? strides[ndim - 1] : 1;
  p.width = uint32_t(width);
  p.groups = uint32_t(groups);
  p.total = uint32_t(groups * rows);
  p.gdiv = make_fastdiv(p.groups);
  p.key = philox_key(seed, offset);
  p.threshold = threshold;
  p.scale = dropout_scale(threshold);
  k_dropout<T><<<unsigned((uint64_t(p.total) + kDropBlock - 1) / kDropBlock), kDropBlock, 0, st>>>(
      static_cast<const T*>(a), static_cast<T*>(out), p);
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
  uint64_t numel = 1;
  for (int i = 0; i < ndim; ++i) numel *= shape[i];
  if (numel > 0 && (a == nullptr || out == nullptr)) {
    g_wrapper_error = 6;
    return -1;
  }
  if (dtype == MUSAPY_DT_F32) return launch_dropout<float>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  if (dtype == MUSAPY_DT_BF16) return launch_dropout<__bf16>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  if (dtype == MUSAPY_DT_F16) return launch_dropout<_Float16>(a, out, ndim, shape, strides, threshold, seed, offset, st);
  g_wrapper_error = 6;
  return -1;
}
