// embedding.hip -- rows of a table by token number, and the gradient of the table, for gfx950.
#include "vocab.hpp"

namespace mpy {

constexpr int kEmbedBlock = 256;

// ---- lookup -----------------------------------------------------------------------------------------
struct EmbedArgs {
  const void* table;
  int64_t rs, cs;     // strides of the table's rows and columns
  Ids ids;
  void* out;
  uint32_t rows;      // of the table
  uint32_t width;
  uint32_t groups;    // groups of N columns in a row
  uint32_t total;     // groups in all
  FastDiv gdiv;       // divides a group's number by `groups`
  float scale;
};

// A thread takes kEmbedGroups groups of N columns, a workgroup's width apart: their token numbers, then
// their table rows, are all in flight at once.  A row's last group ends with the row, so that it overlaps its
// neighbour where N does not divide the width (both store the same values there); rows of fewer than N
// columns take N = 1.
constexpr int kEmbedGroups = 4;

template <class T, class O, int N, bool UNIT, bool NT>
__global__ __launch_bounds__(kEmbedBlock) void k_embedding(EmbedArgs p) {
  const uint64_t first = uint64_t(blockIdx.x) * (kEmbedBlock * kEmbedGroups) + threadIdx.x;
  uint32_t token[kEmbedGroups], row[kEmbedGroups], col[kEmbedGroups];
#pragma unroll
  for (int i = 0; i < kEmbedGroups; ++i) {
    const uint64_t q = first + uint64_t(i) * kEmbedBlock;
    const uint32_t at = q < p.total ? uint32_t(q) : p.total - 1;
    row[i] = fd_div(p.gdiv, at);
    const uint32_t c = (at - row[i] * p.groups) * N;
    col[i] = c + N <= p.width ? c : p.width - N;
    token[i] = id_at(p.ids, row[i], p.rows);
  }
  Vec<T, N> v[kEmbedGroups];
#pragma unroll
  for (int i = 0; i < kEmbedGroups; ++i) {
    const uint32_t t = token[i] < p.rows ? token[i] : 0;  // the first row in the place of none
    const T* at = static_cast<const T*>(p.table) + int64_t(t) * p.rs + int64_t(col[i]) * p.cs;
    if constexpr (UNIT) {
      v[i] = vload_el<T, N, false>(at);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[i].v[e] = at[e * p.cs];
    }
  }
#pragma unroll
  for (int i = 0; i < kEmbedGroups; ++i) {
    if (first + uint64_t(i) * kEmbedBlock >= p.total) continue;
    Vec<O, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = token[i] < p.rows ? O(float(v[i].v[e]) * p.scale) : O(0.0f);
    vstore_el<NT, O, N>(static_cast<O*>(p.out) + uint64_t(row[i]) * p.width + col[i], o);
  }
}

template <class T, class O>
int launch_embedding(const musapy_embedding_args* a, hipStream_t st) {
  constexpr int kN = sizeof(T) == 2 && sizeof(O) == 2 ? 8 : 4;
  const bool narrow = a->width < uint64_t(kN);
  const uint64_t groups = narrow ? a->width : (a->width + kN - 1) / kN;
  const uint64_t total = groups * a->tokens;
  if (total >= uint64_t(1) << 32) return vocab_bad();
  const uint64_t grid = (total + kEmbedBlock * kEmbedGroups - 1) / (kEmbedBlock * kEmbedGroups);
  if (!grid_fits(grid, kEmbedBlock)) return vocab_bad();
  EmbedArgs p{};
  p.table = a->table;
  p.rs = a->row_stride;
  p.cs = a->column_stride;
  p.ids = vocab_ids(a->ids, a->id_dtype);
  p.out = a->out;
  p.rows = uint32_t(a->rows);
  p.width = uint32_t(a->width);
  p.groups = uint32_t(groups);
  p.total = uint32_t(total);
  p.gdiv = make_fastdiv(p.groups);
  p.scale = a->scale;
  const bool unit = p.cs == 1 || p.width == 1;
  const bool nt = a->tokens * a->width * sizeof(O) >= kStreamStoreBytes;
  auto go = [&](auto N, auto UNIT, auto NT) {
    k_embedding<T, O, N.value, UNIT.value, NT.value><<<unsigned(grid), kEmbedBlock, 0, st>>>(p);
  };
  using Full = std::integral_constant<int, kN>;
  using One = std::integral_constant<int, 1>;
  if (narrow && unit) go(One{}, std::true_type{}, std::false_type{});
  else if (narrow) go(One{}, std::false_type{}, std::false_type{});
  else if (!unit) go(Full{}, std::false_type{}, std::false_type{});
  else if (nt) go(Full{}, std::true_type{}, std::true_type{});
  else go(Full{}, std::true_type{}, std::false_type{});
  return 0;
}

// ---- gradient: the tokens in order ------------------------------------------------------------------
// Token numbers with their places, sorted by number and, among equals, by place: sums over a token's
// rows then run in one order, whatever the hardware does, and no two workgroups add to one row.  A
// number outside the table becomes `rows`, behind all others.
struct OrderArgs {
  Ids ids;
  uint32_t n, rows;
  uint32_t *keys, *pos;              // the order
  const uint32_t *keys_in, *pos_in;  // of a later pass
  uint32_t* hist;                    // [tile][bin]
  uint32_t tile, tiles;              // tokens of a workgroup, and workgroups
  int shift, bits;
};

// Up to 16 * 1024 tokens: the place of a token in the order is the number of tokens in front of it, counted against
// all others, 64 comparisons an instruction.  A workgroup ranks 64 tokens, its 16 waves hold G groups of 64
// others each.  One launch without a wait; n^2 / 64 comparisons of four cycles on 1024 SIMDs.
constexpr int kRankWaves = 16;

template <int G>
__global__ __launch_bounds__(kRankWaves * 64) void k_embed_rank(OrderArgs p) {
  __shared__ uint32_t part[kRankWaves][64];
  const int lane = threadIdx.x % 64;
  const uint32_t wave = wave_uniform(threadIdx.x / 64);
  uint32_t other[G];
  uint32_t before[G];  // 1 where the group stands in front of this workgroup's: equals count there
#pragma unroll
  for (int i = 0; i < G; ++i) {
    const uint32_t g = uint32_t(i) * kRankWaves + wave;
    const uint32_t at = g * 64 + lane;
    other[i] = at < p.n ? id_at(p.ids, at, p.rows) : ~0u;
    before[i] = g < blockIdx.x ? 1u : 0u;
  }
  const uint32_t own = blockIdx.x * 64 + lane;
  const uint32_t mine = own < p.n ? id_at(p.ids, own, p.rows) : ~0u;
  uint32_t count = 0;
#pragma unroll 4
  for (int e = 0; e < 64; ++e) {
    const uint32_t key = uint32_t(__builtin_amdgcn_readlane(int(mine), e));
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < G; ++i) c += uint32_t(__popcll(__ballot(other[i] < key + before[i])));
    if (wave == 0) c += uint32_t(__popcll(__ballot(mine == key) & ((uint64_t(1) << e) - 1)));
    if (lane == e) count = c;
  }
  part[wave][lane] = count;
  __syncthreads();
  if (wave == 0 && own < p.n) {
    uint32_t rank = 0;
#pragma unroll
    for (int w = 0; w < kRankWaves; ++w) rank += part[w][lane];
    p.keys[rank] = mine;
    p.pos[rank] = own;
  }
}

// More tokens: passes over up to nine bits each, lowest first; a pass counts its digits in every tile of
// tokens (at most 256 tiles), then every workgroup adds up what lies in front of its own and places its
// tokens, in order.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortWaves = 8, kSortBlock = kSortWaves * 64, kSortRounds = 4, kSortStep = kSortBlock * kSortRounds;
constexpr uint32_t kSortTiles = 256;

template <bool FIRST>
__device__ inline uint32_t order_key(const OrderArgs& p, uint32_t i) {
  return FIRST ? id_at(p.ids, i, p.rows) : p.keys_in[i];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void k_embed_digits(OrderArgs p) {
  __shared__ uint32_t count[kDigits];
  static_assert(kSortBlock == kDigits, "a thread to a digit");
  count[threadIdx.x] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * p.tile;
  const uint32_t last = p.n - first < p.tile ? p.n : first + p.tile;
  for (uint32_t i = first + threadIdx.x; i < last; i += kSortBlock)
    atomicAdd(&count[(order_key<FIRST>(p, i) >> p.shift) & ((1u << p.bits) - 1)], 1u);
  __syncthreads();
  p.hist[blockIdx.x * kDigits + threadIdx.x] = count[threadIdx.x];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void k_embed_place(OrderArgs p) {
  __shared__ uint32_t base[kDigits];
  __shared__ uint32_t at[kSortWaves][kDigits];
  const int lane = threadIdx.x % 64;
  const uint32_t wave = wave_uniform(threadIdx.x / 64);
  // tokens with a lower digit, and those with this thread's digit in the tiles in front
  {
    const uint32_t* h = p.hist + threadIdx.x;
    uint32_t front = 0, total = 0;
#pragma unroll 8
    for (uint32_t t = 0; t < p.tiles; ++t) {
      const uint32_t c = h[t * kDigits];
      front += t < blockIdx.x ? c : 0;
      total += c;
    }
    uint32_t run = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t v = __shfl_up(run, d, kWave);
      if (lane >= d) run += v;
    }
    if (lane == 63) at[0][wave] = run;
    __syncthreads();
    uint32_t lower = run - total;
    for (uint32_t w = 0; w < wave; ++w) lower += at[0][w];
    base[threadIdx.x] = lower + front;
    __syncthreads();
  }
  const uint32_t first = blockIdx.x * p.tile;
  const uint32_t last = p.n - first < p.tile ? p.n : first + p.tile;
  for (uint32_t s = first; s < last; s += kSortStep) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) at[w][threadIdx.x] = 0;
    __syncthreads();
    uint32_t key[kSortRounds], place[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const uint32_t i = s + wave * (kSortRounds * 64) + uint32_t(r) * 64 + lane;
      key[r] = i < last ? order_key<FIRST>(p, i) : ~0u;
      place[r] = FIRST || i >= last ? i : p.pos_in[i];
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const bool there = s + wave * (kSortRounds * 64) + uint32_t(r) * 64 + lane < last;
      const uint32_t digit = (key[r] >> p.shift) & ((1u << p.bits) - 1);
      uint64_t same = __ballot(there);  // the lanes with this lane's digit
      for (int b = 0; b < p.bits; ++b) {
        const uint64_t set = __ballot((digit >> b) & 1);
        same &= (digit >> b) & 1 ? set : ~set;
      }
      const uint64_t lower = same & ((uint64_t(1) << lane) - 1);
      uint32_t* slot = &at[wave][digit];
      const uint32_t before = there ? *static_cast<volatile uint32_t*>(slot) : 0;
      rank[r] = before + uint32_t(__popcll(lower));
      __builtin_amdgcn_wave_barrier();
      if (there && lower == 0) *static_cast<volatile uint32_t*>(slot) = before + uint32_t(__popcll(same));
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    {
      uint32_t off = base[threadIdx.x];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t c = at[w][threadIdx.x];
        at[w][threadIdx.x] = off;
        off += c;
      }
      base[threadIdx.x] = off;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (s + wave * (kSortRounds * 64) + uint32_t(r) * 64 + lane >= last) continue;
      const uint32_t to = at[wave][(key[r] >> p.shift) & ((1u << p.bits) - 1)] + rank[r];
      p.keys[to] = key[r];
      p.pos[to] = place[r];
    }
    __syncthreads();
  }
}

// ---- gradient: the sums --------------------------------------------------------------------------------
struct EmbedGradArgs {
  const uint32_t *keys, *pos;  // the order
  uint32_t n, rows, width;
  const void* dy;
  uint64_t pitch;
  void* out;
  float* slots;                // [chunk][2][padded]: sums of runs that cross a chunk's start, and its end
  uint32_t padded;             // the width, rounded up to 4
  uint32_t chunk, chunks;      // tokens of a chunk, and chunks
  uint32_t tiles;              // of 64 * N columns
  uint32_t sum_blocks;         // workgroups that sum; those behind them fill
  uint32_t fill_rows;          // rows of a workgroup that fills
  uint32_t fill_groups;        // groups of a row there
  FastDiv fill_div;
  float scale;
};

// How many of the sorted keys are below `key`; all lanes of a wave take part, 64 probes a step.
__device__ inline uint32_t wave_lower_bound(const uint32_t* keys, uint32_t lo, uint32_t hi, uint32_t key, int lane) {
  while (hi - lo > 64) {
    const uint32_t step = (hi - lo + 63) / 64;
    const uint64_t at = uint64_t(lo) + uint64_t(lane) * step;
    const uint32_t below = uint32_t(__popcll(__ballot(at < hi && keys[at < hi ? at : lo] < key)));
    if (below == 0) return lo;
    const uint64_t end = uint64_t(lo) + uint64_t(below) * step;  // (the first probe that is not below, or behind all)
    lo += (below - 1) * step + 1;
    hi = end < hi ? uint32_t(end) : hi;
  }
  return lo + uint32_t(__popcll(__ballot(lo + lane < hi && keys[lo + lane < hi ? lo + lane : lo] < key)));
}

// Rows of zeros for the tokens that do not occur.
template <class O, int N>
__device__ inline void embed_fill(const EmbedGradArgs& p, uint32_t block) {
  __shared__ uint32_t present[2];
  const uint32_t first = block * p.fill_rows;
  const uint32_t count = p.rows - first < p.fill_rows ? p.rows - first : p.fill_rows;
  if (threadIdx.x < 64) {
    const uint32_t lane = threadIdx.x;
    uint32_t lo = wave_lower_bound(p.keys, 0, p.n, first, int(lane));
    uint32_t hi = wave_lower_bound(p.keys, lo, p.n, first + count, int(lane));
    const uint32_t end = hi, key = first + lane;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (p.keys[mid] < key) lo = mid + 1;
      else hi = mid;
    }
    const uint64_t m = __ballot(lane < count && lo < end && p.keys[lo < end ? lo : 0] == key);
    if (lane == 0) {
      present[0] = uint32_t(m);
      present[1] = uint32_t(m >> 32);
    }
  }
  __syncthreads();
  const uint64_t mask = present[0] | uint64_t(present[1]) << 32;
  Vec<O, N> zero;
#pragma unroll
  for (int e = 0; e < N; ++e) zero.v[e] = O(0.0f);
  const uint32_t total = count * p.fill_groups;
  O* out = static_cast<O*>(p.out) + uint64_t(first) * p.width;
  for (uint32_t q = threadIdx.x; q < total; q += kEmbedBlock) {
    const uint32_t row = fd_div(p.fill_div, q);
    const uint32_t c = (q - row * p.fill_groups) * N;
    if ((mask >> row) & 1) continue;
    vstore_el<true, O, N>(out + uint64_t(row) * p.width + (c + N <= p.width ? c : p.width - N), zero);
  }
}

template <class O, int N, bool ADD>
__device__ inline void embed_store(O* at, int skip, const float (&sum)[N], float scale) {
  if constexpr (ADD) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e >= skip) at[e] = O(float(at[e]) + sum[e] * scale);
  } else {
    Vec<O, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = O(sum[e] * scale);
    vstore_el<true, O, N>(at, v);
  }
}

// A wave sums a chunk of the order over 64 * N columns, eight rows of dy in flight, and stores a row of the
// table wherever the token changes.  What belongs to a token that the chunk shares with a neighbour goes to a
// slot in f32.  A row's last columns overlap as in the lookup; `skip` of them are the neighbour's where the
// store adds to what is there.
constexpr int kEmbedRows = 8;

template <class T, class O, int N, bool ADD>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_sum(EmbedGradArgs p) {
  if (blockIdx.x >= p.sum_blocks) {
    if constexpr (!ADD) embed_fill<O, N == 1 ? 1 : 16 / int(sizeof(O))>(p, blockIdx.x - p.sum_blocks);
    return;
  }
  const int lane = threadIdx.x % 64;
  const uint32_t unit = blockIdx.x * (kEmbedBlock / 64) + wave_uniform(threadIdx.x / 64);
  const uint32_t chunk = unit / p.tiles;
  if (chunk >= p.chunks) return;
  const uint32_t c = ((unit - chunk * p.tiles) * 64 + lane) * N;
  const bool active = c < p.width;
  const uint32_t col = c + N <= p.width ? c : p.width - N;
  const int skip = active ? int(c - col) : 0;
  const uint32_t first = chunk * p.chunk;
  const uint32_t last = p.n - first < p.chunk ? p.n : first + p.chunk;
  uint32_t cur = wave_uniform(p.keys[first]);
  if (cur >= p.rows) return;
  bool shared = first > 0 && wave_uniform(p.keys[first - 1]) == cur;  // the run began in front of the chunk
  const uint32_t next = last < p.n ? wave_uniform(p.keys[last]) : ~0u;
  const T* dy = static_cast<const T*>(p.dy) + col;
  float sum[N] = {};

  auto store = [&](bool goes_on) {
    if (cur < p.rows && active) {
      if (!shared && !goes_on) {
        embed_store<O, N, ADD>(static_cast<O*>(p.out) + uint64_t(cur) * p.width + col, skip, sum, p.scale);
      } else {
        float* slot = p.slots + (uint64_t(chunk) * 2 + (shared ? 0 : 1)) * p.padded + col;
        Vec<float, N> v;
#pragma unroll
        for (int e = 0; e < N; ++e) v.v[e] = sum[e];
        vstore_el<false, float, N>(slot, v);
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) sum[e] = 0.0f;
  };

  for (uint32_t base = first; base < last; base += 64) {
    const uint32_t at = base + lane;
    const uint32_t key = at < last ? p.keys[at] : ~0u, place = at < last ? p.pos[at] : 0;
    const int count = last - base < 64 ? int(last - base) : 64;
    for (int i = 0; i < count; i += kEmbedRows) {
      Vec<T, N> v[kEmbedRows];
#pragma unroll
      for (int u = 0; u < kEmbedRows; ++u) {
        const int j = i + u < count ? i + u : count - 1;
        v[u] = vload_el<T, N, true>(dy + uint64_t(uint32_t(__builtin_amdgcn_readlane(int(place), j))) * p.pitch);
      }
#pragma unroll
      for (int u = 0; u < kEmbedRows; ++u) {
        if (i + u >= count) continue;
        const uint32_t k = uint32_t(__builtin_amdgcn_readlane(int(key), i + u));
        if (k != cur) {
          store(false);
          cur = k;
          shared = false;
        }
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] += float(v[u].v[e]);
      }
    }
  }
  store(next == cur);
}

// The rows of tokens that cross from chunk to chunk: the workgroups of the chunk where a token begins add
// up its slots, the four waves a quarter of them each, always in the same order.
template <class O, bool ADD>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_join(EmbedGradArgs p) {
  __shared__ float part[4][64][4];
  const uint32_t chunk = blockIdx.x;
  const uint32_t first = chunk * p.chunk, last = first + p.chunk;
  if (last >= p.n) return;
  const uint32_t key = wave_uniform(p.keys[last - 1]);
  if (key >= p.rows || wave_uniform(p.keys[last]) != key) return;
  if (first > 0 && wave_uniform(p.keys[first]) == key && wave_uniform(p.keys[first - 1]) == key) return;  // it began before
  const int lane = threadIdx.x % 64;
  const uint32_t wave = wave_uniform(threadIdx.x / 64);
  uint32_t n = 1;  // slots: this chunk's second, then the first of each chunk that begins with the token
  while (true) {
    const uint64_t j = uint64_t(chunk) + n + lane;
    const uint64_t same = __ballot(j < p.chunks && p.keys[j < p.chunks ? j * p.chunk : 0] == key);
    const uint32_t more = same == ~uint64_t(0) ? 64u : uint32_t(__builtin_ctzll(~same));
    n += more;
    if (more < 64) break;
  }
  const uint32_t col = (blockIdx.y * 64 + lane) * 4;
  const uint32_t from = uint32_t(uint64_t(n) * wave / 4), to = uint32_t(uint64_t(n) * (wave + 1) / 4);
  float sum[4] = {};
  if (col < p.padded) {
#pragma unroll 8
    for (uint32_t s = from; s < to; ++s) {
      const Vec<float, 4> v =
          vload<float, 4>(p.slots + (uint64_t(chunk + s) * 2 + (s == 0 ? 1 : 0)) * p.padded + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += v.v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) part[wave][lane][e] = sum[e];
  __syncthreads();
  if (wave != 0) return;
  O* out = static_cast<O*>(p.out) + uint64_t(key) * p.width + col;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (col + e >= p.width) break;
    float s = part[0][lane][e];
#pragma unroll
    for (int w = 1; w < 4; ++w) s += part[w][lane][e];
    out[e] = ADD ? O(float(out[e]) + s * p.scale) : O(s * p.scale);
  }
}

// ---- launches -------------------------------------------------------------------------------------------
struct EmbedGradPlan {
  int passes, bits;         // 0 passes: by rank
  uint32_t tile, tiles;     // of a pass
  uint32_t chunk, chunks;
  uint32_t padded;
  size_t keys, pos, keys2, pos2, hist, slots, bytes;  // offsets into the scratch
};

constexpr uint64_t kRankMost = uint64_t(kRankWaves) * 64 * 16;

inline EmbedGradPlan embed_grad_plan(const musapy_embedding_grad_args* a) {
  EmbedGradPlan pl{};
  const uint64_t n = a->tokens;
  if (n > kRankMost) {
    int bits = 1;
    while (bits < 32 && (uint64_t(a->rows) >> bits) != 0) ++bits;
    pl.passes = (bits + kDigitBits - 1) / kDigitBits;
    pl.bits = (bits + pl.passes - 1) / pl.passes;
    const uint64_t steps = (n + kSortStep - 1) / kSortStep;
    pl.tile = uint32_t((steps + kSortTiles - 1) / kSortTiles * kSortStep);
    pl.tiles = uint32_t((n + pl.tile - 1) / pl.tile);
  }
  pl.chunk = 32;
  while (n / pl.chunk > 2048) pl.chunk *= 2;
  pl.chunks = uint32_t((n + pl.chunk - 1) / pl.chunk);
  pl.padded = uint32_t((a->width + 3) / 4 * 4);
  auto take = [&](size_t bytes) {
    const size_t at = pl.bytes;
    pl.bytes += (bytes + 15) / 16 * 16;
    return at;
  };
  pl.keys = take(n * 4);
  pl.pos = take(n * 4);
  if (pl.passes > 0) {
    pl.keys2 = take(n * 4);
    pl.pos2 = take(n * 4);
    pl.hist = take(size_t(pl.tiles) * kDigits * 4);
  }
  pl.slots = take(size_t(pl.chunks) * 2 * pl.padded * 4);
  return pl;
}

inline void launch_order(const musapy_embedding_grad_args* a, const EmbedGradPlan& pl, char* ws, hipStream_t st) {
  OrderArgs o{};
  o.ids = vocab_ids(a->ids, a->id_dtype);
  o.n = uint32_t(a->tokens);
  o.rows = uint32_t(a->rows);
  uint32_t* keys[2] = {reinterpret_cast<uint32_t*>(ws + pl.keys), reinterpret_cast<uint32_t*>(ws + pl.keys2)};
  uint32_t* pos[2] = {reinterpret_cast<uint32_t*>(ws + pl.pos), reinterpret_cast<uint32_t*>(ws + pl.pos2)};
  if (pl.passes == 0) {
    o.keys = keys[0];
    o.pos = pos[0];
    const unsigned grid = unsigned((o.n + 63) / 64);
    const int most = kRankWaves * 64;
    if (o.n <= 1 * most) k_embed_rank<1><<<grid, most, 0, st>>>(o);
    else if (o.n <= 2 * most) k_embed_rank<2><<<grid, most, 0, st>>>(o);
    else if (o.n <= 4 * most) k_embed_rank<4><<<grid, most, 0, st>>>(o);
    else if (o.n <= 8 * most) k_embed_rank<8><<<grid, most, 0, st>>>(o);
    else k_embed_rank<16><<<grid, most, 0, st>>>(o);
    return;
  }
  o.hist = reinterpret_cast<uint32_t*>(ws + pl.hist);
  o.tile = pl.tile;
  o.tiles = pl.tiles;
  o.bits = pl.bits;
  for (int i = 0; i < pl.passes; ++i) {
    const int to = (pl.passes - 1 - i) % 2;  // the last pass ends in the first buffers
    o.shift = i * pl.bits;
    o.keys = keys[to];
    o.pos = pos[to];
    o.keys_in = keys[1 - to];
    o.pos_in = pos[1 - to];
    if (i == 0) {
      k_embed_digits<true><<<pl.tiles, kSortBlock, 0, st>>>(o);
      k_embed_place<true><<<pl.tiles, kSortBlock, 0, st>>>(o);
    } else {
      k_embed_digits<false><<<pl.tiles, kSortBlock, 0, st>>>(o);
      k_embed_place<false><<<pl.tiles, kSortBlock, 0, st>>>(o);
    }
  }
}

template <class T, class O>
int launch_embedding_grad(const musapy_embedding_grad_args* a, char* ws, hipStream_t st) {
  const EmbedGradPlan pl = embed_grad_plan(a);
  constexpr int kN = sizeof(T) == 2 ? 8 : 4;
  constexpr int kFill = 16 / int(sizeof(O));
  const bool narrow = a->width < uint64_t(kN) || a->width < uint64_t(kFill);
  const int n = narrow ? 1 : kN, fill = narrow ? 1 : kFill;
  EmbedGradArgs p{};
  p.keys = reinterpret_cast<uint32_t*>(ws + pl.keys);
  p.pos = reinterpret_cast<uint32_t*>(ws + pl.pos);
  p.n = uint32_t(a->tokens);
  p.rows = uint32_t(a->rows);
  p.width = uint32_t(a->width);
  p.dy = a->dy;
  p.pitch = a->dy_pitch;
  p.out = a->out;
  p.slots = reinterpret_cast<float*>(ws + pl.slots);
  p.padded = pl.padded;
  p.chunk = pl.chunk;
  p.chunks = pl.chunks;
  p.tiles = uint32_t((a->width + 64 * n - 1) / (64 * n));
  p.scale = a->scale;
  const uint64_t units = uint64_t(p.chunks) * p.tiles;
  p.sum_blocks = uint32_t((units + 3) / 4);
  p.fill_groups = uint32_t((a->width + fill - 1) / fill);
  p.fill_div = make_fastdiv(p.fill_groups);
  p.fill_rows = 64;  // rows of some 128 KB a workgroup, 8 at least
  while (p.fill_rows > 8 && uint64_t(p.fill_rows) * a->width * sizeof(O) > (128u << 10)) p.fill_rows /= 2;
  const uint64_t fills = a->accumulate ? 0 : (a->rows + p.fill_rows - 1) / p.fill_rows;
  if (units >= kVocabLimit || !grid_fits(p.sum_blocks + fills, kEmbedBlock)) return vocab_bad();
  const uint64_t joins = (pl.padded + 255) / 256;
  if (joins > 65535) return vocab_bad();
  if (p.n > 0) launch_order(a, pl, ws, st);
  const unsigned grid = unsigned(p.sum_blocks + fills);
  const dim3 join(pl.chunks, unsigned(joins));
  auto go = [&](auto N, auto ADD) {
    if (grid > 0) k_embed_sum<T, O, N.value, ADD.value><<<grid, kEmbedBlock, 0, st>>>(p);
    if (pl.chunks > 1) k_embed_join<O, ADD.value><<<join, kEmbedBlock, 0, st>>>(p);
  };
  using Full = std::integral_constant<int, kN>;
  using One = std::integral_constant<int, 1>;
  if (narrow && a->accumulate) go(One{}, std::true_type{});
  else if (narrow) go(One{}, std::false_type{});
  else if (a->accumulate) go(Full{}, std::true_type{});
  else go(Full{}, std::false_type{});
  return 0;
}

}  // namespace mpy

using namespace mpy;

extern "C" {

int musapy_embedding_v1(const musapy_embedding_args* a, hipStream_t st) {
  if (a == nullptr || !vocab_float(a->table_dtype) || !vocab_float(a->out_dtype) || !vocab_id(a->id_dtype) ||
      a->tokens >= kVocabLimit || a->rows >= kVocabLimit || a->width >= kVocabLimit)
    return vocab_bad();
  if (a->tokens == 0 || a->width == 0) return 0;
  if (a->rows == 0 || a->table == nullptr || a->ids == nullptr || a->out == nullptr) return vocab_bad();
  int rc = 0;
  vocab_type(a->table_dtype, [&](auto t) {
    vocab_type(a->out_dtype, [&](auto o) { rc = launch_embedding<decltype(t), decltype(o)>(a, st); });
  });
  return rc;
}

static bool embedding_grad_ok(const musapy_embedding_grad_args* a) {
  return a != nullptr && vocab_float(a->dy_dtype) && vocab_float(a->out_dtype) && vocab_id(a->id_dtype) &&
         (a->accumulate == 0 || a->accumulate == 1) && a->tokens < kVocabLimit && a->rows < kVocabLimit &&
         a->width < kVocabLimit;
}

size_t musapy_embedding_grad_scratch_v1(const musapy_embedding_grad_args* a) {
  if (!embedding_grad_ok(a) || a->tokens == 0 || a->rows == 0 || a->width == 0) return 0;
  return embed_grad_plan(a).bytes;
}

int musapy_embedding_grad_v1(const musapy_embedding_grad_args* a, void* scratch, size_t scratch_bytes, hipStream_t st) {
  if (!embedding_grad_ok(a)) return vocab_bad();
  if (a->rows == 0 || a->width == 0 || (a->tokens == 0 && a->accumulate)) return 0;
  if (a->out == nullptr || (a->tokens > 0 && (a->dy == nullptr || a->ids == nullptr))) return vocab_bad();
  const size_t need = musapy_embedding_grad_scratch_v1(a);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15)))
    return vocab_bad(1);
  int rc = 0;
  vocab_type(a->dy_dtype, [&](auto t) {
    vocab_type(a->out_dtype, [&](auto o) {
      rc = launch_embedding_grad<decltype(t), decltype(o)>(a, static_cast<char*>(scratch), st);
    });
  });
  return rc;
}

}  // extern "C"
