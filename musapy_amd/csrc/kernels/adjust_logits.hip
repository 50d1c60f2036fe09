// adjust_logits.hip -- penalties for repeated tokens, biases and masks on logits, for gfx950.
#include "vocab.hpp"

namespace mpy {

constexpr int kAdjustBlock = 512;
constexpr int kBiasMost = 1024;

// A number for all sequences, or one for each.
struct PerRow {
  const float* at;
  float value;
};
__device__ inline float per_row(const PerRow& v, uint32_t row) { return v.at ? v.at[row] : v.value; }

struct AdjustArgs {
  const void* logits;
  uint64_t pitch;
  void* out;
  uint32_t rows, width;
  Ids history;
  uint64_t history_pitch;
  uint32_t length;         // of a history's row
  Ids lengths;             // at: NULL for `length`
  PerRow repetition, presence, frequency;
  const void* bias;        // dense (entries 0), or of the entries
  int bias_dtype;
  uint64_t bias_pitch;
  Ids bias_index;
  uint64_t index_pitch;
  uint32_t entries;
  const void* allowed;     // bits: 32-bit words; else bytes
  uint64_t allowed_pitch;
  int bits;
  uint32_t tile, tiles;    // columns of a workgroup, workgroups of a row
};

// A workgroup takes a tile of a row's columns.  It counts the tokens of the row's history that fall into the tile, in
// LDS, then reads the tile once and writes it once.  Biased tokens, few, are formed again and stored over the
// first values behind a barrier; a token that several entries name gets the sum of their biases from the first.
template <class T, class O, bool HISTORY>
__global__ __launch_bounds__(kAdjustBlock) void k_adjust(AdjustArgs p) {
  constexpr int N = 8;
  extern __shared__ uint32_t count[];
  const uint32_t row = blockIdx.x / p.tiles;
  const uint32_t first = (blockIdx.x - row * p.tiles) * p.tile;
  const uint32_t last = p.width - first < p.tile ? p.width : first + p.tile;
  const T* z = static_cast<const T*>(p.logits) + uint64_t(row) * p.pitch;
  O* out = static_cast<O*>(p.out) + uint64_t(row) * p.width;
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  if constexpr (HISTORY) {
    for (uint32_t i = threadIdx.x * 4; i < p.tile; i += kAdjustBlock * 4)
      *reinterpret_cast<uint4*>(count + i) = uint4{0, 0, 0, 0};
    rep = per_row(p.repetition, row);
    pres = per_row(p.presence, row);
    freq = per_row(p.frequency, row);
    uint32_t length = p.length;
    if (p.lengths.at) {  // below 0: none; past the row's end: all of it
      const int64_t n = p.lengths.wide ? static_cast<const int64_t*>(p.lengths.at)[row]
                                       : static_cast<const int32_t*>(p.lengths.at)[row];
      length = n < 0 ? 0 : n < int64_t(p.length) ? uint32_t(n) : p.length;
    }
    __syncthreads();
    const uint64_t start = row * p.history_pitch;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < length; i += kAdjustBlock) {
      const uint32_t at = id_at(p.history, start + i, p.width) - first;
      if (at < last - first) atomicAdd(&count[at], 1u);
    }
    __syncthreads();
  }
  const uint8_t* bytes = nullptr;
  const uint32_t* words = nullptr;
  if (p.allowed) {
    if (p.bits) words = static_cast<const uint32_t*>(p.allowed) + uint64_t(row) * p.allowed_pitch;
    else bytes = static_cast<const uint8_t*>(p.allowed) + uint64_t(row) * p.allowed_pitch;
  }
  const uint64_t bias_row = uint64_t(row) * p.bias_pitch;
  const bool dense = p.bias && p.entries == 0;

  auto seen = [&](float x, uint32_t c) {
    const float y = x > 0.0f ? x / rep : x * rep;
    return c ? y - (freq * float(c) + pres) : x;
  };
  auto one = [&](uint32_t i, float bias) {
    float x = float(z[i]);
    if constexpr (HISTORY) x = seen(x, count[i - first]);
    x += bias;
    const bool ok = words ? (words[i / 32] >> (i % 32)) & 1 : bytes ? bytes[i] != 0 : true;
    out[i] = O(ok ? x : -__builtin_inff());
  };
  const uint32_t vectors = (last - first) / N;
  for (uint32_t q = threadIdx.x; q < vectors; q += kAdjustBlock) {
    const uint32_t i = first + q * N;
    const Vec<T, N> v = vload_el<T, N, true>(z + i);
    uint32_t ok = 0xff;
    if (words) {
      ok = words[i / 32] >> (i % 32);
    } else if (bytes) {
      const Vec<uint8_t, N> m = vload_el<uint8_t, N, true>(bytes + i);
      ok = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) ok |= (m.v[e] != 0 ? 1u : 0u) << e;
    }
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = float(v.v[e]);
    if constexpr (HISTORY) {
      const Vec<uint32_t, N> c = *reinterpret_cast<const Vec<uint32_t, N>*>(count + q * N);
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) any |= c.v[e];
      if (any) {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = seen(x[e], c.v[e]);
      }
    }
    if (dense) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[e] += float_at(p.bias, p.bias_dtype, bias_row + i + e);
    }
    Vec<O, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = O((ok >> e) & 1 ? x[e] : -__builtin_inff());
    vstore_el<false, O, N>(out + i, o);
  }
  {
    const uint32_t i = first + vectors * N + threadIdx.x;
    if (i < last) one(i, dense ? float_at(p.bias, p.bias_dtype, bias_row + i) : 0.0f);
  }
  if (p.entries == 0) return;
  __shared__ uint32_t index[kBiasMost];
  __shared__ float value[kBiasMost];
  for (uint32_t k = threadIdx.x; k < p.entries; k += kAdjustBlock) {
    index[k] = id_at(p.bias_index, row * p.index_pitch + k, p.width);
    value[k] = float_at(p.bias, p.bias_dtype, bias_row + k);
  }
  __syncthreads();
  for (uint32_t k = threadIdx.x; k < p.entries; k += kAdjustBlock) {
    const uint32_t i = index[k];
    if (i < first || i >= last) continue;
    float sum = 0.0f;
    bool leads = true;
    for (uint32_t j = 0; j < p.entries; ++j) {
      if (index[j] != i) continue;
      if (j < k) leads = false;
      sum += value[j];
    }
    if (leads) one(i, sum);
  }
}

template <class T, class O>
void launch_adjust(const AdjustArgs& p, bool history, hipStream_t st) {
  const unsigned grid = p.rows * p.tiles;
  if (history) k_adjust<T, O, true><<<grid, kAdjustBlock, p.tile * 4, st>>>(p);
  else k_adjust<T, O, false><<<grid, kAdjustBlock, 0, st>>>(p);
}

}  // namespace mpy

using namespace mpy;

extern "C" int musapy_adjust_logits_v1(const musapy_adjust_logits_args* a, hipStream_t st) {
  if (a == nullptr || !vocab_float(a->dtype) || (a->out_dtype != a->dtype && a->out_dtype != MUSAPY_DT_F32) ||
      a->rows >= kVocabLimit || a->width >= kVocabLimit || a->length >= kVocabLimit || a->entries > size_t(kBiasMost))
    return vocab_bad();
  if (a->rows == 0 || a->width == 0) return 0;
  const bool history = a->history != nullptr && a->length > 0;
  if (a->logits == nullptr || a->out == nullptr || (history && !vocab_id(a->history_dtype)) ||
      (a->lengths != nullptr && !vocab_id(a->lengths_dtype)) || (a->bias != nullptr && !vocab_float(a->bias_dtype)) ||
      (a->entries > 0 && (a->bias == nullptr || a->bias_index == nullptr || !vocab_id(a->index_dtype))) ||
      (a->allowed != nullptr && a->allowed_kind != MUSAPY_ALLOWED_BYTES && a->allowed_kind != MUSAPY_ALLOWED_BITS))
    return vocab_bad();
  AdjustArgs p{};
  p.logits = a->logits;
  p.pitch = a->pitch;
  p.out = a->out;
  p.rows = uint32_t(a->rows);
  p.width = uint32_t(a->width);
  p.history = vocab_ids(a->history, a->history_dtype);
  p.history_pitch = a->history_pitch;
  p.length = uint32_t(a->length);
  p.lengths = vocab_ids(a->lengths, a->lengths_dtype);
  p.repetition = {a->repetition, a->repetition_value};
  p.presence = {a->presence, a->presence_value};
  p.frequency = {a->frequency, a->frequency_value};
  p.bias = a->bias;
  p.bias_dtype = a->bias_dtype;
  p.bias_pitch = a->bias_pitch;
  p.bias_index = vocab_ids(a->bias_index, a->index_dtype);
  p.index_pitch = a->index_pitch;
  p.entries = uint32_t(a->entries);
  p.allowed = a->allowed;
  p.allowed_pitch = a->allowed_pitch;
  p.bits = a->allowed_kind == MUSAPY_ALLOWED_BITS;
  // the widest tile of up to 8192 columns that leaves the chip full: every tile reads the whole history
  p.tile = 8192;
  while (p.tile > 2048 && uint64_t(p.rows) * ((p.width + p.tile - 1) / p.tile) < 1024) p.tile /= 2;
  p.tiles = (p.width + p.tile - 1) / p.tile;
  if (!grid_fits(uint64_t(p.rows) * p.tiles, kAdjustBlock)) return vocab_bad();
  vocab_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if (a->out_dtype == a->dtype) launch_adjust<T, T>(p, history, st);
    else launch_adjust<T, float>(p, history, st);
  });
  return 0;
}
