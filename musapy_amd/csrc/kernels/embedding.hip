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
  RawId raw[kEmbedGroups];
  uint32_t token[kEmbedGroups], row[kEmbedGroups], col[kEmbedGroups];
#pragma unroll
  for (int i = 0; i < kEmbedGroups; ++i) {
    const uint64_t q = first + uint64_t(i) * kEmbedBlock;
    const uint32_t at = q < p.total ? uint32_t(q) : p.total - 1;
    row[i] = fd_div(p.gdiv, at);
    const uint32_t c = (at - row[i] * p.groups) * N;
    col[i] = c + N <= p.width ? c : p.width - N;
    raw[i] = id_load(p.ids, row[i]);
  }
  Vec<T, N> v[kEmbedGroups];
#pragma unroll
  for (int i = 0; i < kEmbedGroups; ++i) {
    token[i] = id_of(raw[i], p.rows);
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
  // 16 bytes of the result to a lane: with 32, each store leaves every other 16 bytes of a line to the next one (16384 rows of 4096 bf16
  // into f32 104 us, so 51), and with 8, (f32 into bf16) 68 against 50.
  constexpr int kN = 16 / int(sizeof(O));
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
  char* zero;                        // part of the table's gradient, which the launch clears
  uint64_t zero_bytes;
  uint32_t order_blocks;             // workgroups in front of those that clear
  uint32_t zero_pieces;              // of a vector for every thread, of a workgroup that clears
};

// Every row is cleared while the order begins, though those of tokens are written again: 4 KB a workgroup, one vector a
// thread, in the order of addresses, run at 6.7 TB/s (8 to 128 KB a workgroup 5.5 to 6.1).  Clearing only the other
// rows beside the sums, with the sorted tokens or bits of the rows to look up, took the (131072, 2048) f32 gradient of 16384
// tokens 225 to 240 us, against 157 for this and some 30 for the sums.  The later launches of an order by digits, whose few
// workgroups take 5 to 10 us whatever is cleared beside them, take 40 MB of it each.
constexpr uint64_t kClearBeside = uint64_t(40) << 20;

template <int BLOCK>
__device__ inline void order_clear(const OrderArgs& p, uint32_t block) {
  typedef uint32_t W __attribute__((ext_vector_type(4)));
  const uint64_t past = reinterpret_cast<uintptr_t>(p.zero) % 16;
  const uint64_t head = past == 0 ? 0 : 16 - past < p.zero_bytes ? 16 - past : p.zero_bytes;
  const uint64_t vectors = (p.zero_bytes - head) / 16;
  W* out = reinterpret_cast<W*>(p.zero + head);
  for (uint32_t k = 0; k < p.zero_pieces; ++k) {
    const uint64_t at = (uint64_t(block) * p.zero_pieces + k) * BLOCK + threadIdx.x;
    if (at < vectors) out[at] = W{0, 0, 0, 0};
  }
  if (block != 0 || threadIdx.x >= 32) return;
  const uint64_t edge = threadIdx.x < 16 ? threadIdx.x : head + vectors * 16 + threadIdx.x - 16;  // single bytes at both ends
  if (threadIdx.x < 16 ? edge < head : edge < p.zero_bytes) p.zero[edge] = 0;
}

// Up to 5120 tokens, in one launch: a token's place is the number of tokens in front of it, counted against all others.  All lie in
// LDS (20 KB a workgroup, so that eight that clear fit a CU); a workgroup places 16 tokens, and sixteen threads to each count a
// sixteenth of the others, four at a time.  Against two launches, as below: 1584 tokens 20 us, so 14; 5120 of 1024 into (50000,
// 1024) f32 50.2 and 46.6, but numbers of 64 bits, which every workgroup reads, 52.4, and 4096 of them level.
constexpr int kRankBlock = 256, kRankTokens = 16;
inline bool embed_ranks(uint64_t tokens, int id_dtype) { return tokens <= (id_dtype == MUSAPY_DT_I64 ? 4096u : 5120u); }

__global__ __launch_bounds__(kRankBlock) void k_embed_rank(OrderArgs p) {
  if (blockIdx.x >= p.order_blocks) return order_clear<kRankBlock>(p, blockIdx.x - p.order_blocks);
  typedef uint32_t W __attribute__((ext_vector_type(4)));
  extern __shared__ W groups[];  // four tokens each
  __shared__ uint32_t part[kRankBlock / 64][kRankTokens];
  uint32_t* all = reinterpret_cast<uint32_t*>(groups);
  const uint32_t most = (p.n + 63) / 64 * 64;
  for (uint32_t base = threadIdx.x; base < most; base += 8 * kRankBlock) {
    RawId raw[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t i = base + u * kRankBlock;
      raw[u] = id_load(p.ids, i < p.n ? i : p.n - 1);
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t i = base + u * kRankBlock;
      if (i < most) all[i] = i < p.n ? id_of(raw[u], p.rows) : ~0u;
    }
  }
  __syncthreads();
  const uint32_t item = threadIdx.x % kRankTokens, share = threadIdx.x / kRankTokens;
  const uint32_t at = blockIdx.x * kRankTokens + item, own = at / 4;
  const uint32_t key = all[at];
  uint32_t count = 0;
#pragma unroll 4
  for (uint32_t g = share; g < most / 4; g += kRankBlock / kRankTokens) {
    const W k = groups[g];
    const uint32_t limit = g < own ? key + 1 : key;  // equals count in front of the token
#pragma unroll
    for (int e = 0; e < 4; ++e) count += k[e] < limit ? 1 : 0;
  }
  count += uint32_t(__shfl_xor(int(count), 16, kWave));
  count += uint32_t(__shfl_xor(int(count), 32, kWave));
  if (threadIdx.x % 64 < kRankTokens) part[threadIdx.x / 64][item] = count;
  __syncthreads();
  if (threadIdx.x >= kRankTokens || at >= p.n) return;
  for (int w = 1; w < kRankBlock / 64; ++w) count += part[w][item];
  for (uint32_t e = 0; e < at % 4; ++e) count += all[own * 4 + e] == key ? 1 : 0;
  p.keys[count] = key;
  p.pos[count] = at;
}

// Up to kOrderMost tokens, in two launches.  First, blocks of 256 tokens, a quarter of one a workgroup: a token's place in its block
// is the number of tokens in front of it, counted by each wave against a quarter of the block.
constexpr int kBlockTokens = 256, kOrderBlock = 1024, kOrderWaves = kOrderBlock / 64;
constexpr int kOrderMost = 32768;

__global__ __launch_bounds__(kBlockTokens) void k_embed_blocks(OrderArgs p) {
  if (blockIdx.x >= p.order_blocks) return order_clear<kBlockTokens>(p, blockIdx.x - p.order_blocks);
  typedef uint32_t W __attribute__((ext_vector_type(4)));
  __shared__ W groups[kBlockTokens / 4];
  __shared__ uint32_t part[kBlockTokens / 64][64];
  uint32_t* all = reinterpret_cast<uint32_t*>(groups);
  const uint32_t lane = threadIdx.x % 64, wave = wave_uniform(threadIdx.x / 64), quarter = blockIdx.x % 4;
  const uint32_t first = blockIdx.x / 4 * kBlockTokens, at = first + quarter * 64 + lane;
  all[threadIdx.x] = first + threadIdx.x < p.n ? id_at(p.ids, first + threadIdx.x, p.rows) : ~0u;
  __syncthreads();
  const uint32_t key = all[quarter * 64 + lane];
  const uint32_t limit = wave < quarter ? key + 1 : key;  // equals count in front of the token (a missing one's limit is not used)
  uint32_t count = 0;
#pragma unroll
  for (uint32_t g = 0; g < 16; ++g) {
    const W k = groups[wave * 16 + g];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
      count += k[e] < limit ? 1 : 0;
      if (wave == quarter) count += k[e] == key && g * 4 + e < lane ? 1 : 0;
    }
  }
  part[wave][lane] = count;
  __syncthreads();
  if (wave != 0 || at >= p.n) return;
  count = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
  p.keys[first + count] = key;
  p.pos[first + count] = at;
}

// Then a token's place among all is its place in its block and, of every other block, the number of keys below
// its own (or not above it, of the blocks in front), each found by halving.  All keys lie in LDS; a workgroup places 64
// tokens at a time, 128 in all beyond 16384, where one workgroup has a CU for itself, and each of its 16 waves searches every sixteenth
// block, four at a time.  (26784 tokens 9.8 us behind some 4 for the blocks; in passes over their digits 33.)
__global__ __launch_bounds__(kOrderBlock) void k_embed_merge(OrderArgs p) {
  typedef uint32_t W __attribute__((ext_vector_type(4)));
  extern __shared__ W sorted[];
  __shared__ uint32_t part[kOrderWaves][64];
  uint32_t* all = reinterpret_cast<uint32_t*>(sorted);
  const uint32_t blocks = (p.n + kBlockTokens - 1) / kBlockTokens, vectors = p.n / 4;
  for (uint32_t base = threadIdx.x; base < vectors; base += 4 * kOrderBlock) {
    W k[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t i = base + u * kOrderBlock;
      k[u] = reinterpret_cast<const W*>(p.keys_in)[i < vectors ? i : vectors - 1];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (base + u * kOrderBlock < vectors) sorted[base + u * kOrderBlock] = k[u];
  }
  for (uint32_t i = vectors * 4 + threadIdx.x; i < blocks * kBlockTokens; i += kOrderBlock) all[i] = i < p.n ? p.keys_in[i] : ~0u;
  __syncthreads();
  const int lane = threadIdx.x % 64;
  const uint32_t wave = wave_uniform(threadIdx.x / 64);
  for (uint32_t set = blockIdx.x; set * 64 < p.n; set += gridDim.x) {
    const uint32_t at = set * 64 + lane, own = set * 64 / kBlockTokens;
    const uint32_t key = all[at];
    uint32_t count = 0;
    for (uint32_t b0 = wave; b0 < blocks; b0 += 4 * kOrderWaves) {
      uint32_t base[4], limit[4], c[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t b = b0 + i * kOrderWaves;
        base[i] = b < blocks ? b * kBlockTokens : 0;
        limit[i] = b < blocks && b != own ? key + (b < own ? 1 : 0) : 0;  // nothing is below 0
      }
#pragma unroll
      for (uint32_t step = kBlockTokens / 2; step > 0; step /= 2)
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += all[base[i] + c[i] + step - 1] < limit[i] ? step : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) count += c[i] + (all[base[i] + c[i]] < limit[i] ? 1 : 0);
    }
    if (set != blockIdx.x) __syncthreads();
    part[wave][lane] = count;
    __syncthreads();
    if (wave != 0 || at >= p.n) continue;
    uint32_t to = at - own * kBlockTokens;
#pragma unroll
    for (int w = 0; w < kOrderWaves; ++w) to += part[w][lane];
    p.keys[to] = key;
    p.pos[to] = p.pos_in[at];
  }
}

// More tokens: passes over up to nine bits each, lowest first; a pass counts its digits in every tile of
// tokens (at most 256 tiles), then every workgroup adds up what lies in front of its own and places its
// tokens, in order.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kSortWaves = 8, kSortBlock = kSortWaves * 64, kSortRounds = 4, kSortStep = kSortBlock * kSortRounds;
constexpr uint32_t kSortTiles = 256;

template <bool FIRST>
__device__ inline RawId order_load(const OrderArgs& p, uint32_t i) {
  if constexpr (FIRST) return id_load(p.ids, i);
  else return RawId{p.keys_in[i], 0};
}
template <bool FIRST>
__device__ inline uint32_t order_key(const OrderArgs& p, const RawId& r) {
  return FIRST ? id_of(r, p.rows) : r.low;
}

template <bool FIRST>
__global__ __launch_bounds__(kBlockTokens) void k_embed_digits(OrderArgs p) {
  if (blockIdx.x >= p.order_blocks) return order_clear<kBlockTokens>(p, blockIdx.x - p.order_blocks);
  __shared__ uint32_t count[kDigits];
  for (int d = threadIdx.x; d < kDigits; d += kBlockTokens) count[d] = 0;
  __syncthreads();
  const uint32_t first = blockIdx.x * p.tile;
  const uint32_t last = p.n - first < p.tile ? p.n : first + p.tile;
  for (uint32_t i = first + threadIdx.x; i < last; i += kBlockTokens)
    atomicAdd(&count[(order_key<FIRST>(p, order_load<FIRST>(p, i)) >> p.shift) & ((1u << p.bits) - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kBlockTokens) p.hist[blockIdx.x * kDigits + d] = count[d];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void k_embed_place(OrderArgs p) {
  if (blockIdx.x >= p.order_blocks) return order_clear<kSortBlock>(p, blockIdx.x - p.order_blocks);
  static_assert(kSortBlock == kDigits, "a thread to a digit");
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
    RawId raw[kSortRounds];
    uint32_t key[kSortRounds], place[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      const uint32_t i = s + wave * (kSortRounds * 64) + uint32_t(r) * 64 + lane, at = i < last ? i : last - 1;
      raw[r] = order_load<FIRST>(p, at);
      place[r] = FIRST ? at : p.pos_in[at];
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) key[r] = order_key<FIRST>(p, raw[r]);
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
  float scale;
};

template <class O, int N, bool ADD, bool NT>
__device__ inline void embed_store(O* at, int skip, const float (&sum)[N], float scale) {
  if constexpr (ADD) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e >= skip) at[e] = O(float(at[e]) + sum[e] * scale);
  } else {
    Vec<O, N> v;
#pragma unroll
    for (int e = 0; e < N; ++e) v.v[e] = O(sum[e] * scale);
    vstore_el<NT, O, N>(at, v);
  }
}

// A wave sums a chunk of the order over 64 * N columns and stores a row of the
// table wherever the token changes.  What belongs to a token that the chunk shares with a neighbour goes to a
// slot in f32.  A row's last columns overlap as in the lookup; `skip` of them are the neighbour's where the
// store adds to what is there.  NT: streaming stores, where the table's gradient has kStreamStoreBytes or more, as elsewhere (alone level;
// 1000 tokens into (5000, 1024) f32 with a maximum of each row behind 22.6 us streamed, 21.5 not; 8000 into (32000, 512) 42.5 and 40.6).
template <class T, class O, int N, bool ADD, bool NT>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_sum(EmbedGradArgs p) {
  constexpr int kEmbedRows = N * sizeof(T) > 16 ? 4 : 8;
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
  // the first 64 tokens of the chunk and its neighbours, all on their way at once
  uint32_t key = p.keys[first + lane < last ? first + lane : last - 1], place = p.pos[first + lane < last ? first + lane : last - 1];
  const uint32_t before = p.keys[first > 0 ? first - 1 : 0], behind = p.keys[last < p.n ? last : p.n - 1];
  uint32_t cur = wave_uniform(key);
  if (cur >= p.rows) return;
  bool shared = first > 0 && wave_uniform(before) == cur;  // the run began in front of the chunk
  const uint32_t next = last < p.n ? wave_uniform(behind) : ~0u;
  const T* dy = static_cast<const T*>(p.dy) + col;
  float sum[N] = {};

  auto store = [&](bool goes_on) {
    if (cur < p.rows && active) {
      if (!shared && !goes_on) {
        embed_store<O, N, ADD, NT>(static_cast<O*>(p.out) + uint64_t(cur) * p.width + col, skip, sum, p.scale);
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

  // As many rows are added up while the next are on their way: a load behind a store is waited for with it, and stores are slow (100000
  // tokens of 1024 bf16 113.8 us, so 118.9).
  Vec<T, N> va[kEmbedRows], vb[kEmbedRows];
  for (uint32_t base = first; base < last; base += 64) {
    if (base > first) {
      const uint32_t at = base + lane < last ? base + lane : last - 1;
      key = p.keys[at];
      place = p.pos[at];
    }
    const int count = last - base < 64 ? int(last - base) : 64;
    auto fetch = [&](Vec<T, N>(&v)[kEmbedRows], int i) {
      if (i >= count) return;
#pragma unroll
      for (int u = 0; u < kEmbedRows; ++u) {
        const int j = i + u < count ? i + u : count - 1;
        v[u] = vload_el<T, N, true>(dy + uint64_t(uint32_t(__builtin_amdgcn_readlane(int(place), j))) * p.pitch);
      }
    };
    auto add = [&](const Vec<T, N>(&v)[kEmbedRows], int i) {
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
    };
    fetch(va, 0);
    for (int i = 0; i < count; i += 2 * kEmbedRows) {
      fetch(vb, i + kEmbedRows);
      add(va, i);
      fetch(va, i + 2 * kEmbedRows);
      add(vb, i + kEmbedRows);
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

// ---- gradient: few tokens --------------------------------------------------------------------------------
// In one launch: a wave takes 1 KB of the table's gradient, a vector a lane, finds the tokens of its rows among all, and adds up
// their rows of dy; most find none and clear.
constexpr int kGatherMost = 256;

struct EmbedGatherArgs {
  Ids ids;
  uint32_t n, rows, width;
  const void* dy;
  uint64_t pitch;
  void* out;
  uint32_t total, head, vectors;  // values, those in front of the first address that is a multiple of 16 bytes, vectors behind them
  FastDiv wdiv;                   // divides by the width
  float scale;
};

// K: tokens a lane looks at.  EVEN: every vector lies in one row.  Else one may end a row and begin the next (width >= N): its first
// values are summed as the last N of its row, the others as the first N of the next.
template <class T, class O, int K, bool EVEN>
__global__ __launch_bounds__(kEmbedBlock) void k_embed_gather(EmbedGatherArgs p) {
  constexpr int N = 16 / int(sizeof(O)), kRows = 128 / int(sizeof(T) * N);  // rows of dy in flight, in 32 registers
  __shared__ uint2 lists[kEmbedBlock / 64][K * 64];  // token and place of each that is found, in order of places
  const uint32_t lane = threadIdx.x % 64, wave = wave_uniform(threadIdx.x / 64);
  RawId raw[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t i = k * 64 + lane;
    raw[k] = p.n > 0 ? id_load(p.ids, i < p.n ? i : p.n - 1) : RawId{0, 1};
  }
  const uint32_t base = blockIdx.x * kEmbedBlock + wave * 64, at = base + lane;
  if (base > 0 && base >= p.vectors) return;
  const bool ends = base + 64 >= p.vectors;
  const uint32_t first = base == 0 ? 0 : p.head + base * N, past = ends ? p.total : p.head + (base + 64) * N;
  const uint32_t low = fd_div(p.wdiv, first), high = fd_div(p.wdiv, past - 1);
  uint2* list = lists[wave];
  uint32_t count = 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint32_t token = id_of(raw[k], p.rows);
    const uint64_t here = __ballot(k * 64 + lane < p.n && token >= low && token <= high);
    if (here == 0) continue;
    if ((here >> lane) & 1) list[count + uint32_t(__popcll(here & ((uint64_t(1) << lane) - 1)))] = uint2{token, k * 64 + lane};
    count += uint32_t(__popcll(here));
  }
  O* out = static_cast<O*>(p.out);
  // a value of its own in front of the vectors (the first wave's) or behind them (the last one's)
  uint32_t lone = p.total;
  if (base == 0 && lane < p.head) lone = lane;
  if (ends && lane >= 32 && lane < 32 + N) lone = p.head + p.vectors * N + lane - 32;
  if (count == 0) {
    if (at < p.vectors) vstore_el<false, O, N>(out + p.head + at * N, Vec<O, N>{});
    if (lone < p.total) out[lone] = O(0.0f);
    return;
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  const T* dy = static_cast<const T*>(p.dy);
  if (at < p.vectors) {
    const uint32_t value = p.head + at * N, row = fd_div(p.wdiv, value), col = value - row * p.width;
    const uint32_t cut = EVEN || p.width - col > uint32_t(N) ? uint32_t(N) : p.width - col;  // values of `row`
    const uint32_t next = EVEN || cut == uint32_t(N) ? row : row + 1, from = EVEN || cut == uint32_t(N) ? col : p.width - N;
    float sum[N] = {}, sum2[N] = {};
    for (uint32_t b = 0; b < count; b += kRows) {
      Vec<T, N> v[kRows];
      uint32_t whose[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const uint2 l = list[b + i < count ? b + i : count - 1];
        whose[i] = b + i < count ? l.x : p.rows;
        v[i] = vload_el<T, N, true>(dy + l.y * p.pitch + (EVEN || l.x == row ? from : 0));
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          sum[e] += whose[i] == row ? float(v[i].v[e]) : 0.0f;
          if (!EVEN) sum2[e] += whose[i] == next ? float(v[i].v[e]) : 0.0f;
        }
      }
    }
    Vec<O, N> o;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      float x = sum[e];
      if (!EVEN && cut < uint32_t(N)) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (uint32_t(e) < cut ? e + N == int(cut) + j : e == int(cut) + j) x = uint32_t(e) < cut ? sum[j] : sum2[j];
        }
      }
      o.v[e] = O(x * p.scale);
    }
    vstore_el<false, O, N>(out + value, o);
  }
  if (lone < p.total) {
    const uint32_t row = fd_div(p.wdiv, lone), col = lone - row * p.width;
    float sum = 0.0f;
#pragma unroll 8
    for (uint32_t b = 0; b < count; ++b) {
      const uint2 l = list[b];
      const float x = float(dy[l.y * p.pitch + col]);
      sum += l.x == row ? x : 0.0f;
    }
    out[lone] = O(sum * p.scale);
  }
}

// Whether a gradient goes that way: not one that is added to what is there, whose rows without tokens are not touched.  Up to 64
// tokens, one a lane, (131072, 1024) f32 takes 79 us at 6.8 TB/s, by an order and sums 87, and a table of a few MB 6, so 10 to 14.  With 250
// tokens a wave's search costs more than a launch where the table is large ((131072, 2048) f32 209 us, so 165; (16384, 1024) 20.4 and
// 18.7; (8704, 232) 6.6 and 14.7).  A wave's time grows by 0.12 us for every row that one token has (256 rows of one 32 us, so 16).
constexpr uint64_t kGatherBytes = uint64_t(32) << 20;
inline bool embed_gathers(const musapy_embedding_grad_args* a) {
  const uint64_t size = a->out_dtype == MUSAPY_DT_F32 ? 4 : 2, values = a->rows * a->width;
  return !a->accumulate && a->width >= 16 / size && values < kVocabLimit &&
         (a->tokens <= 64 || (a->tokens <= uint64_t(kGatherMost) && values * size <= kGatherBytes));
}

template <class T, class O>
int launch_embedding_gather(const musapy_embedding_grad_args* a, hipStream_t st) {
  constexpr uint32_t kN = 16 / sizeof(O);
  EmbedGatherArgs p{};
  p.ids = vocab_ids(a->ids, a->id_dtype);
  p.n = uint32_t(a->tokens);
  p.rows = uint32_t(a->rows);
  p.width = uint32_t(a->width);
  p.dy = a->dy;
  p.pitch = a->dy_pitch;
  p.out = a->out;
  p.total = uint32_t(a->rows * a->width);
  const uint32_t past = uint32_t(reinterpret_cast<uintptr_t>(a->out) / sizeof(O) % kN);
  p.head = past == 0 ? 0 : kN - past;  // (a row has as many)
  p.vectors = (p.total - p.head) / kN;
  p.wdiv = make_fastdiv(p.width);
  p.scale = a->scale;
  const unsigned grid = p.vectors == 0 ? 1 : (p.vectors + kEmbedBlock - 1) / kEmbedBlock;
  auto go = [&](auto K, auto EVEN) { k_embed_gather<T, O, K.value, EVEN.value><<<grid, kEmbedBlock, 0, st>>>(p); };
  using All = std::integral_constant<int, kGatherMost / 64>;
  using One = std::integral_constant<int, 1>;
  const bool even = p.head == 0 && p.width % kN == 0;
  if (p.n <= 64 && even) go(One{}, std::true_type{});
  else if (p.n <= 64) go(One{}, std::false_type{});
  else if (even) go(All{}, std::true_type{});
  else go(All{}, std::false_type{});
  return 0;
}

// ---- launches -------------------------------------------------------------------------------------------
struct EmbedGradPlan {
  int passes, bits;         // 0 passes: by rank or by blocks
  uint32_t tile, tiles;     // of a pass
  uint32_t chunk, chunks;
  uint32_t padded;
  size_t keys, pos, keys2, pos2, hist, slots, bytes;  // offsets into the scratch
};

inline EmbedGradPlan embed_grad_plan(const musapy_embedding_grad_args* a) {
  EmbedGradPlan pl{};
  const uint64_t n = a->tokens;
  if (n > uint64_t(kOrderMost)) {
    int bits = 1;
    while (bits < 32 && (uint64_t(a->rows) >> bits) != 0) ++bits;
    pl.passes = (bits + kDigitBits - 1) / kDigitBits;
    pl.bits = (bits + pl.passes - 1) / pl.passes;
    const uint64_t steps = (n + kSortStep - 1) / kSortStep;
    pl.tile = uint32_t((steps + kSortTiles - 1) / kSortTiles * kSortStep);
    pl.tiles = uint32_t((n + pl.tile - 1) / pl.tile);
  }
  // Chunks of 8 to 64 tokens that give some 4096 waves (longer ones beyond 131072 tokens): shorter ones keep more rows in flight (20000
  // tokens of 512 bf16 take 10 us less than with chunks of 64), longer ones have fewer tokens that cross.
  pl.chunk = 8;
  const uint64_t tiles = (a->width + 255) / 256;
  while ((pl.chunk < 64 && n / pl.chunk * tiles > 4096) || n / pl.chunk > 2048) pl.chunk *= 2;
  pl.chunks = uint32_t((n + pl.chunk - 1) / pl.chunk);
  pl.padded = uint32_t((a->width + 3) / 4 * 4);
  auto take = [&](size_t bytes) {
    const size_t at = pl.bytes;
    pl.bytes += (bytes + 15) / 16 * 16;
    return at;
  };
  pl.keys = take(n * 4);
  pl.pos = take(n * 4);
  if (!embed_ranks(n, a->id_dtype)) {
    pl.keys2 = take(n * 4);
    pl.pos2 = take(n * 4);
  }
  if (pl.passes > 0) {
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
  const uint32_t blocks = pl.passes ? pl.tiles : (o.n + kBlockTokens - 1) / kBlockTokens;
  const int launches = pl.passes ? 2 * pl.passes : 1;
  uint64_t bytes = a->accumulate ? 0 : a->rows * a->width * (a->out_dtype == MUSAPY_DT_F32 ? 4 : 2);
  char* out = static_cast<char*>(a->out);
  uint64_t beside = bytes / uint64_t(launches) < kClearBeside ? bytes / uint64_t(launches) : kClearBeside;
  beside = beside / 4096 * 4096;
  // the workgroups of a launch: those that order, and those that clear the next `part` bytes
  auto grid = [&](uint32_t order, uint64_t threads, uint64_t part) {
    o.order_blocks = order;
    o.zero = out;
    o.zero_bytes = part;
    out += part;
    bytes -= part;
    const uint64_t pieces = part ? part / (16 * threads) + 1 : 0;
    o.zero_pieces = 1;
    while (!grid_fits(order + (pieces + o.zero_pieces - 1) / o.zero_pieces, threads)) o.zero_pieces *= 2;
    return unsigned(order + (pieces + o.zero_pieces - 1) / o.zero_pieces);
  };
  const uint64_t most = bytes - beside * uint64_t(launches - 1);  // of the first launch
  if (embed_ranks(o.n, a->id_dtype)) {
    o.keys = keys[0];
    o.pos = pos[0];
    const unsigned count = grid((o.n + kRankTokens - 1) / kRankTokens, kRankBlock, most);
    if (count > 0) k_embed_rank<<<count, kRankBlock, (o.n + 63) / 64 * 256, st>>>(o);
    return;
  }
  if (pl.passes == 0) {
    o.keys = keys[1];
    o.pos = pos[1];
    k_embed_blocks<<<grid((o.n + 63) / 64, kBlockTokens, most), kBlockTokens, 0, st>>>(o);
    o.keys_in = o.keys;
    o.pos_in = o.pos;
    o.keys = keys[0];
    o.pos = pos[0];
    const unsigned sets = (o.n + 63) / 64;
    k_embed_merge<<<o.n > 16384 ? (sets + 1) / 2 : sets, kOrderBlock, blocks * kBlockTokens * 4, st>>>(o);
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
    const unsigned count = grid(blocks, kBlockTokens, i == 0 ? most : beside);
    if (i == 0) k_embed_digits<true><<<count, kBlockTokens, 0, st>>>(o);
    else k_embed_digits<false><<<count, kBlockTokens, 0, st>>>(o);
    const unsigned place = grid(blocks, kSortBlock, beside);
    if (i == 0) k_embed_place<true><<<place, kSortBlock, 0, st>>>(o);
    else k_embed_place<false><<<place, kSortBlock, 0, st>>>(o);
  }
}

template <class T, class O>
int launch_embedding_grad(const musapy_embedding_grad_args* a, char* ws, hipStream_t st) {
  const EmbedGradPlan pl = embed_grad_plan(a);
  constexpr int kN = 16 / int(sizeof(O));  // 16 bytes of the result to a lane, as in the lookup
  const bool narrow = a->width < uint64_t(kN);
  const int n = narrow ? 1 : kN;
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
  const uint64_t units = uint64_t(p.chunks) * p.tiles, grid = (units + 3) / 4;  // (at most 2049 by 2^14)
  launch_order(a, pl, ws, st);
  const dim3 join(pl.chunks, (pl.padded + 255) / 256);
  const bool nt = a->rows * a->width * sizeof(O) >= kStreamStoreBytes;
  auto go = [&](auto N, auto ADD) {
    if (grid > 0) {
      if constexpr (ADD.value) k_embed_sum<T, O, N.value, true, false><<<unsigned(grid), kEmbedBlock, 0, st>>>(p);
      else with_store_policy(nt, [&](auto NT) { k_embed_sum<T, O, N.value, false, NT.value><<<unsigned(grid), kEmbedBlock, 0, st>>>(p); });
    }
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

// A row's columns, so that launches stay within a grid.
constexpr uint64_t kGradColumns = uint64_t(1) << 22;

static bool embedding_grad_ok(const musapy_embedding_grad_args* a) {
  return a != nullptr && vocab_float(a->dy_dtype) && vocab_float(a->out_dtype) && vocab_id(a->id_dtype) &&
         (a->accumulate == 0 || a->accumulate == 1) && a->tokens < kVocabLimit && a->rows < kVocabLimit &&
         a->width <= kGradColumns;
}

size_t musapy_embedding_grad_scratch_v1(const musapy_embedding_grad_args* a) {
  if (!embedding_grad_ok(a) || a->tokens == 0 || a->rows == 0 || a->width == 0 || embed_gathers(a)) return 0;
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
      if (embed_gathers(a)) rc = launch_embedding_gather<decltype(t), decltype(o)>(a, st);
      else rc = launch_embedding_grad<decltype(t), decltype(o)>(a, static_cast<char*>(scratch), st);
    });
  });
  return rc;
}

}  // extern "C"
