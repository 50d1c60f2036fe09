// adjust_logits.hip -- penalties for repeated tokens, biases and masks on logits, for gfx950.
#include "vocab.hpp"

namespace mpy {

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
  uint32_t tiles;          // workgroups of a row
};

// Counts of a history's tokens that fall into a tile, in LDS: 16 bits each where no count can pass them.
template <class C>
__device__ inline void count_one(uint32_t* count, uint32_t at) {
  if constexpr (sizeof(C) == 2) atomicAdd(&count[at / 2], at % 2 ? 0x10000u : 1u);
  else atomicAdd(&count[at], 1u);
}

// A workgroup takes a tile of a row's columns, U vectors of 16 bytes of the result to a thread.  The tile, its mask, the first biased
// columns and the first kPast vectors a thread of the row's history are on their way at once, whatever the history's
// length turns out to be; the tokens that fall into the tile are counted in LDS, and the tile is read once and written
// once.
constexpr int kPast = 4;

template <class T, class O, class C, bool HISTORY, int BLOCK, int TILE, bool NT>
__global__ __launch_bounds__(BLOCK) void k_adjust(AdjustArgs p) {
  constexpr int N = 16 / int(sizeof(O)), U = TILE / BLOCK / N;
  static_assert(U > 0 && U * BLOCK * N == TILE, "whole vectors");
  typedef uint32_t Words __attribute__((ext_vector_type(4)));
  typedef Words AnyWords __attribute__((aligned(4)));
  __shared__ Vec<C, N> count[HISTORY ? TILE / N : 1];
  const uint32_t row = blockIdx.x / p.tiles;
  // Rows begin with different tiles: the common tokens' tile, which counts most, would else fall to one XCD of the eight
  // wherever the tiles of a row are a multiple of them.
  const uint32_t turn = blockIdx.x - row * p.tiles + row % p.tiles;
  const uint32_t first = (turn < p.tiles ? turn : turn - p.tiles) * TILE;
  const uint32_t columns = p.width - first < TILE ? p.width - first : TILE;
  const T* z = static_cast<const T*>(p.logits) + uint64_t(row) * p.pitch + first;
  O* out = static_cast<O*>(p.out) + uint64_t(row) * p.width + first;
  const uint32_t vectors = columns / N;

  // the history as 16-byte vectors of 4 or 2 tokens, and the tokens behind the last of them
  const uint32_t per = p.history.wide ? 2 : 4;
  const uint32_t past = HISTORY ? p.length / per : 0;
  const char* ids = static_cast<const char*>(p.history.at) + row * p.history_pitch * (p.history.wide ? 8 : 4);
  Words h[HISTORY ? kPast : 1];
  auto fetch = [&](uint32_t base) {
#pragma unroll
    for (int u = 0; u < kPast; ++u) {
      const uint32_t q = base + u * BLOCK + threadIdx.x;
      h[u] = *reinterpret_cast<const AnyWords*>(ids + uint64_t(q < past ? q : past - 1) * 16);
    }
  };
  float rep = 1.0f, pres = 0.0f, freq = 0.0f;
  RawId raw_length{};
  if constexpr (HISTORY) {
    if (past > 0) fetch(0);
    if (p.lengths.at) raw_length = id_load(p.lengths, row);
    rep = per_row(p.repetition, row);
    pres = per_row(p.presence, row);
    freq = per_row(p.frequency, row);
#pragma unroll
    for (int u = 0; u < U; ++u) count[u * BLOCK + threadIdx.x] = Vec<C, N>{};
  }
  const uint8_t* bytes = nullptr;
  const uint32_t* words = nullptr;
  if (p.allowed) {
    if (p.bits) words = static_cast<const uint32_t*>(p.allowed) + uint64_t(row) * p.allowed_pitch;
    else bytes = static_cast<const uint8_t*>(p.allowed) + uint64_t(row) * p.allowed_pitch + first;
  }
  Vec<T, N> v[U];
  uint32_t mask[U][N / 4];  // bytes, or in the first word bits
  typedef uint32_t AnyWord __attribute__((aligned(1)));
  const auto clamped = [&](int u) {
    const uint32_t q = u * BLOCK + threadIdx.x;
    return q < vectors ? q : vectors - 1;
  };
  if (vectors > 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = vload_el<T, N, true>(z + uint64_t(clamped(u)) * N);
    if (words) {
#pragma unroll
      for (int u = 0; u < U; ++u) mask[u][0] = words[(first + clamped(u) * N) / 32];
    } else if (bytes) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int w = 0; w < N / 4; ++w) mask[u][w] = reinterpret_cast<const AnyWord*>(bytes + clamped(u) * N)[w];
    }
  }
  const uint64_t bias_row = uint64_t(row) * p.bias_pitch;
  // the first 64 biased columns, a lane each; one that is no column of the tile is past it
  const uint32_t lane = threadIdx.x % 64;
  RawId raw_index{};
  uint32_t raw_bias = 0;
  auto entry = [&](uint32_t k) {
    const uint32_t at = k < p.entries ? k : p.entries - 1;
    raw_index = id_load(p.bias_index, row * p.index_pitch + at);
    raw_bias = float_load(p.bias, p.bias_dtype, bias_row + at);
  };
  if (p.entries > 0) entry(lane);
  if constexpr (HISTORY) {
    uint32_t length = p.length;
    if (p.lengths.at) {  // below 0: none; past the row's end: all of it
      const bool below = (p.lengths.wide ? raw_length.high : raw_length.low) >> 31;
      length = below ? 0 : id_of(raw_length, p.length);
    }
    lds_barrier();
    uint32_t* counts = reinterpret_cast<uint32_t*>(count);
    auto one = [&](uint32_t low, uint32_t high, uint32_t at) {  // a token that is no column of the tile, by all its bits, does not count
      const uint32_t i = low - first;
      if (i < columns && high == 0 && at < length) count_one<C>(counts, i);
    };
    for (uint32_t base = 0; base < past && base * per < length; base += BLOCK * kPast) {
      if (base > 0) fetch(base);
#pragma unroll
      for (int u = 0; u < kPast; ++u) {
        const uint32_t q = base + u * BLOCK + threadIdx.x;
        if (q >= past) continue;
        if (p.history.wide) {
          one(h[u].x, h[u].y, q * 2);
          one(h[u].z, h[u].w, q * 2 + 1);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) one(h[u][e], 0, q * 4 + e);
        }
      }
    }
    const uint32_t rest = past * per + threadIdx.x;
    if (threadIdx.x < per && rest < length) {
      const uint32_t i = id_at(p.history, row * p.history_pitch + rest, p.width) - first;
      if (i < columns) count_one<C>(counts, i);
    }
  }
  if constexpr (HISTORY) lds_barrier();
  const bool dense = p.bias && p.entries == 0;
  auto seen = [&](float x, uint32_t c) { return (x > 0.0f ? x / rep : x * rep) - (freq * float(c) + pres); };
  float x[U][N];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t q = u * BLOCK + threadIdx.x, i = q * N;
    if (q >= vectors) continue;
#pragma unroll
    for (int e = 0; e < N; ++e) x[u][e] = float(v[u].v[e]);
    if constexpr (HISTORY) {
      const Vec<C, N> c = count[q];
#pragma unroll
      for (int e = 0; e < N; ++e)  // (a branch each: few columns of a wave were seen, and the division is long)
        if (c.v[e]) x[u][e] = seen(x[u][e], c.v[e]);
    }
    if (dense) {
      if (p.bias_dtype == MUSAPY_DT_F32) {
        const Vec<float, N> b = vload_el<float, N, false>(static_cast<const float*>(p.bias) + bias_row + first + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[u][e] += b.v[e];
      } else {
        const Vec<T, N> b = vload_el<T, N, false>(static_cast<const T*>(p.bias) + bias_row + first + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[u][e] += float(b.v[e]);
      }
    }
  }
  const uint32_t behind = vectors * N + threadIdx.x;  // a column behind the vectors
  float y = behind < columns ? float(z[behind]) : 0.0f;
  if constexpr (HISTORY) {
    const uint32_t c = behind < columns ? reinterpret_cast<const C*>(count)[behind] : 0;
    if (c) y = seen(y, c);
  }
  if (dense && behind < columns) y += float_at(p.bias, p.bias_dtype, bias_row + first + behind);
  // Each wave adds the biases of its own columns, in the entries' order.
  for (uint32_t k0 = 0; k0 < p.entries; k0 += 64) {
    if (k0 > 0) entry(k0 + lane);
    const uint32_t bi = id_of(raw_index, p.width) - first, q = bi / N;
    const float bv = float_of(raw_bias, p.bias_dtype);
    const bool mine = k0 + lane < p.entries && bi < columns && (q >= vectors || q % BLOCK / 64 == threadIdx.x / 64);
    for (uint64_t those = __ballot(mine); those; those &= those - 1) {
      const int from = __builtin_ctzll(those);
      const uint32_t i = uint32_t(__builtin_amdgcn_readlane(int(bi), from));
      const float b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bv), from));
      if (i == behind) y += b;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (i == (u * BLOCK + threadIdx.x) * N + e) x[u][e] += b;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t q = u * BLOCK + threadIdx.x, i = q * N;
    if (q >= vectors) continue;
    uint32_t ok = 0xff;
    if (words) {
      ok = mask[u][0] >> (i % 32);
    } else if (bytes) {
      ok = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) ok |= ((mask[u][e / 4] >> (8 * (e % 4))) & 0xff ? 1u : 0u) << e;
    }
    Vec<O, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = O((ok >> e) & 1 ? x[u][e] : -__builtin_inff());
    vstore_el<NT, O, N>(out + i, o);
  }
  if (behind >= columns) return;
  const bool ok = words ? (words[(first + behind) / 32] >> ((first + behind) % 32)) & 1 : bytes ? bytes[behind] != 0 : true;
  out[behind] = O(ok ? y : -__builtin_inff());
}

// The tile: 2048 columns without a history ((256, 131072) bf16 with packed masks and biases into f32 34.6 us, 35.1 with 8192); with one, which
// every tile reads, 8192 (42.4, with 2048 54.6, for 4096 tokens each), and 4096 where that leaves the chip's 256 CUs few
// ((4, 32768) f32 4.2 us, with 8192 4.9; (32, 50001) with 30000 tokens 13.8, with 2048 18.1).  Histories of 128 KB and more are read from
// the L2 longer than the logits: 16384 there, if that is a workgroup for every CU ((256, 50001) f16 with 30000 tokens of 64 bits
// 46.5 us, with 8192 63; but with 5000 27.2 and 26.8, and (256, 131072) with 4096 of 32 bits 45.4 and 42.4).
//
// Results stream from kStreamStoreBytes on, as elsewhere: a smaller one is read by whatever chooses the token while the caches hold it.
// Alone, the call is as long either way up to some 8 MB and up to a fifth longer with default stores from there; with a reader of
// the result behind it (a maximum of each row), both together take 13.0 us, streamed 15.8, for (4, 32768) f32 with 500 tokens; 29.6
// and 41.5 for (16, 131072) bf16 into f32; 35.8 and 48.8 for 64 of them with 500 tokens.
template <class T, class O>
int launch_adjust(AdjustArgs& p, bool history, hipStream_t st) {
  auto go = [&](auto HISTORY, auto BLOCK, auto TILE) {
    constexpr uint32_t kTile = TILE.value;
    p.tiles = (p.width + kTile - 1) / kTile;
    const uint64_t grid = uint64_t(p.rows) * p.tiles;
    if (!grid_fits(grid, BLOCK.value)) return vocab_bad();
    with_store_policy(uint64_t(p.rows) * p.width * sizeof(O) >= kStreamStoreBytes, [&](auto NT) {
      if (p.length < 65536) k_adjust<T, O, uint16_t, HISTORY.value, BLOCK.value, kTile, NT.value><<<unsigned(grid), BLOCK.value, 0, st>>>(p);
      else if constexpr (HISTORY.value) k_adjust<T, O, uint32_t, true, BLOCK.value, kTile, NT.value><<<unsigned(grid), BLOCK.value, 0, st>>>(p);
    });
    return 0;
  };
  using Few = std::integral_constant<int, 256>;
  using Many = std::integral_constant<int, 512>;
  using Most = std::integral_constant<int, 1024>;
  if (!history) {
    p.length = 0;
    return go(std::false_type{}, Few{}, std::integral_constant<int, 2048>{});
  }
  if (uint64_t(p.length) * (p.history.wide ? 8 : 4) >= 128 * 1024 && p.rows * ((uint64_t(p.width) + 16383) / 16384) >= 256)
    return go(std::true_type{}, Most{}, std::integral_constant<int, 16384>{});
  if (p.rows * ((uint64_t(p.width) + 8191) / 8192) >= 512) return go(std::true_type{}, Many{}, std::integral_constant<int, 8192>{});
  return go(std::true_type{}, Many{}, std::integral_constant<int, 4096>{});
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
      (a->lengths != nullptr && !vocab_id(a->lengths_dtype)) || (a->bias != nullptr && a->bias_dtype != a->dtype && a->bias_dtype != MUSAPY_DT_F32) ||
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
  int rc = 0;
  vocab_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    if (a->out_dtype == a->dtype) rc = launch_adjust<T, T>(p, history, st);
    else rc = launch_adjust<T, float>(p, history, st);
  });
  return rc;
}
