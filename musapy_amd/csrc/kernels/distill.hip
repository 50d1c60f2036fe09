// distill.hip -- a student's loss against a teacher's top entries and labels, and its gradient, for gfx950.
#include "vocab.hpp"

namespace mpy {

constexpr float kLog2e = 1.44269504f, kLn2 = 0.69314718f;
constexpr int kEntriesMost = 1024;

struct DistillArgs {
  const void* logits;
  uint64_t pitch;
  Ids index;
  uint64_t index_pitch;
  const void* teacher;
  int teacher_dtype;
  uint64_t teacher_pitch;
  Ids labels;              // at: NULL for none
  uint32_t rows, width, entries;
  float inv_t;             // 1 / T
  float c;                 // log2(e) / T
  float near;              // of the loss: logits below it in size take one multiply-add an exponent
  float soft;              // weight T^2; of the gradient, weight T
  float hard;              // 1 - weight
  int use_soft;            // weight is not 0
  float* loss;
  float* sums;             // (rows, 3): m, log sum exp((z - m) / T), log sum exp(z - m); of the gradient, read
  const float* dloss;
  int64_t dloss_stride;
  void* grad;
  uint32_t segments;       // workgroups of a row
  uint32_t segment;        // of the loss: columns of each
  float* parts;            // of the loss, with more than one: (rows, segments, 3), a segment's maximum and sums
};

__device__ inline float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A teacher's entry as it is loaded (any one where there is none of that number), and its column and value: the width where
// it does not count (there is none, its index is no column, or its value is -inf).
struct RawEntry {
  RawId index;
  uint32_t value;
};
__device__ inline RawEntry entry_load(const DistillArgs& p, uint32_t row, uint32_t k) {
  if (!p.use_soft) return RawEntry{RawId{0, 1}, 0};
  const uint32_t at = k < p.entries ? k : p.entries - 1;
  return RawEntry{id_load(p.index, row * p.index_pitch + at), float_load(p.teacher, p.teacher_dtype, row * p.teacher_pitch + at)};
}
__device__ inline void entry_of(const DistillArgs& p, const RawEntry& r, uint32_t k, uint32_t& i, float& x) {
  x = float_of(r.value, p.teacher_dtype);
  i = k < p.entries && x != -__builtin_inff() ? id_of(r.index, p.width) : p.width;
}
__device__ inline void teacher_entry(const DistillArgs& p, uint32_t row, uint32_t k, uint32_t& i, float& x) {
  entry_of(p, entry_load(p, row, k), k, i, x);
}

// The columns of a row in front of its first address that is a multiple of 16 bytes.
template <class T>
__device__ inline uint32_t row_head(const T* row, uint32_t width) {
  constexpr uint32_t N = 16 / sizeof(T);
  const uint32_t head = (N - uint32_t(reinterpret_cast<uintptr_t>(row) / sizeof(T)) % N) % N;
  return head < width ? head : width;
}

// A workgroup takes a row, or a segment of one where there are few: every thread keeps the maximum m of its logits and the sums of
// exp((z - m) / T) and, with labels at a T other than 1, exp(z - m), rescaled when m rises; they are joined at the
// end.  A wave then forms the teacher's part, which needs K logits and the sum only:
//   sum_k p_k (log p_k - log q_k) = B / A - log A + (m - r) / T + log sum exp((z - m) / T),
//   e_k = exp((v_k - max v) / T),  A = sum e_k,  B = sum e_k ((v_k - max v) - (z_k - r)) / T
// with r the highest of the entries' logits: all differences are of near numbers, so that logits far from 0 lose nothing.
//
// For maxima below `near` in size, exponents are one multiply-add, x c - round(m c): the sums are then relative to 2^round(m c), and
// what m c was rounded by, the same for all terms, is taken off at the end.  That lies in the terms' exponents meanwhile, half a unit of
// m c's last place at most: `near` is where m c, at T and at 1, reaches 2^24, so that it is 1/2 at most there.  For maxima beyond (rows
// that a mask of -1e10, the types' lowest value or -inf leaves nothing else, T of 2^-20 with logits above 11) exponents are (x - m) c, a
// subtraction more, and sums are relative to 2^(m c) itself.
enum { kOne = 0, kTwo = 1, kSquare = 2 };  // one sum; two; two at T = 2, where exp(z - m) is the square of exp((z - m) / 2)

constexpr float kNearExponent = 0x1p24f;
// What sums relative to the maximum `from` are multiplied with to be relative to `to`.  Waves of near maxima, nearly all, pass the other
// forms by one branch: (1023, 50001) f32 36.6 us, by selects 38.3; (256, 131072) bf16 15.9 and 18.3.
__device__ inline float sum_change(float from, float to, float c, float near) {
  const bool a = __builtin_fabsf(from) < near, b = __builtin_fabsf(to) < near;
  float e = from * c - to * c;
  if (__ballot(!(a && b)) != 0) {
    if (!a && !b) e = (from - to) * c;
    else if (!a) e = __builtin_fmaf(from, c, -(to * c));
    else if (!b) e = -__builtin_fmaf(to, c, -(from * c));
  }
  return exp2_fast(e);
}

// What a wave knows of a row before its logits: the first 64 entries and the label, and which terms the row has.
struct RowTerms {
  uint32_t i0, label;  // an entry's column to a lane
  float x0;
  bool soft, hard;
};
__device__ inline RowTerms row_terms(const DistillArgs& p, uint32_t row, int lane, const RawEntry& e0, const RawId& raw_label) {
  RowTerms r;
  entry_of(p, e0, lane, r.i0, r.x0);
  r.label = id_of(raw_label, p.width);
  r.hard = r.label < p.width;
  r.soft = __ballot(r.i0 < p.width) != 0;
  for (uint32_t k0 = 64; k0 < p.entries && !r.soft; k0 += 64) {
    uint32_t i;
    float x;
    teacher_entry(p, row, k0 + lane, i, x);
    r.soft = __ballot(i < p.width) != 0;
  }
  return r;
}
__device__ inline void row_unused(const DistillArgs& p, uint32_t row) {
  p.loss[row] = 0.0f;
  for (int i = 0; i < 3; ++i) p.sums[uint64_t(row) * 3 + i] = 0.0f;
}

// The row's results, by one wave, from its maximum and sums; z0: the logits of the first 64 entries.  KR: entries that a lane
// loads at once ((16384, 4000) with 128 entries 47.5 us, 64 at a time 55.5).
template <class T, int SUMS, int KR>
__device__ inline void row_finish(const DistillArgs& p, uint32_t row, int lane, const T* z, const RowTerms& t, float z0, float most, float s, float s1) {
  float a = 0.0f, b = 0.0f, r = -__builtin_inff();
  if (t.soft) {
    RawEntry raw[KR];
    uint32_t ki[KR];
    float kx[KR], ky[KR];
#pragma unroll
    for (int k = 1; k < KR; ++k) raw[k] = entry_load(p, row, k * 64 + lane);
    ki[0] = t.i0;
    kx[0] = t.x0;
    ky[0] = z0;
#pragma unroll
    for (int k = 1; k < KR; ++k) {
      entry_of(p, raw[k], k * 64 + lane, ki[k], kx[k]);
      ky[k] = float(z[ki[k] < p.width ? ki[k] : 0]);
    }
    auto each = [&](auto fn) {
#pragma unroll
      for (int k = 0; k < KR; ++k)
        if (ki[k] < p.width) fn(kx[k], ky[k]);
      for (uint32_t k0 = KR * 64; k0 < p.entries; k0 += 64) {
        uint32_t i;
        float x;
        teacher_entry(p, row, k0 + lane, i, x);
        if (i < p.width) fn(x, float(z[i]));
      }
    };
    float top = -__builtin_inff();
    each([&](float x, float y) {
      top = fmaxf(top, x);
      r = fmaxf(r, y);
    });
    top = wave_max(top);
    r = wave_max(r);
    if (r == -__builtin_inff()) r = 0.0f;
    each([&](float x, float y) {
      const float d = x - top, e = exp2_fast(d * p.c);
      a += e;
      if (!(e == 0.0f)) b += e * ((d - (y - r)) * p.inv_t);
    });
    a = wave_sum(a);
    b = wave_sum(b);
  }
  if (lane != 0) return;
  auto log_sum = [&](float sum, float c) {
    const float off = __builtin_fabsf(most) < p.near ? __builtin_fmaf(most, c, -(most * c)) : 0.0f;
    return kLn2 * (__builtin_amdgcn_logf(sum) - off);
  };
  const float ls = log_sum(s, p.c), ls1 = SUMS != kOne ? log_sum(s1, kLog2e) : ls;
  float loss = 0.0f;
  if (t.soft) loss = p.soft * (b / a - kLn2 * __builtin_amdgcn_logf(a) + (most - r) * p.inv_t + ls);
  if (t.hard) loss += p.hard * ((most - float(z[t.label])) + ls1);
  p.loss[row] = loss;
  float* sums = p.sums + uint64_t(row) * 3;
  sums[0] = most;
  sums[1] = t.soft ? ls : 0.0f;
  sums[2] = t.hard ? ls1 : 0.0f;
}

template <class T, int BLOCK, int SUMS, bool PART, int KR>
__global__ __launch_bounds__(BLOCK) void k_distill_loss(DistillArgs p) {
  constexpr int N = 16 / int(sizeof(T)), U = 4, kWaves = BLOCK / 64;
  constexpr bool TWO = SUMS != kOne;
  __shared__ float part[kWaves][3];
  const uint32_t row = PART ? blockIdx.x / p.segments : blockIdx.x, seg = PART ? blockIdx.x - row * p.segments : 0;
  const int lane = threadIdx.x % 64;
  const uint32_t wave = wave_uniform(threadIdx.x / 64);
  const uint32_t first = PART ? seg * p.segment : 0;
  const uint32_t width = PART && p.width - first > p.segment ? p.segment : p.width - first;
  const T* z = static_cast<const T*>(p.logits) + uint64_t(row) * p.pitch;
  const T* zs = z + first;
  const uint32_t head = row_head<T>(zs, width), vectors = (width - head) / N;
  Vec<T, N> v[U];
  const uint32_t whole = vectors / (BLOCK * U) * (BLOCK * U);  // vectors in rounds of U for every thread
  auto fetch = [&](uint32_t base) {
    const T* at = zs + head + (uint64_t(base) + threadIdx.x) * N;
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = vload_el<T, N, true>(at + u * BLOCK * N);
  };
  auto fetch_rest = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = whole + u * BLOCK + threadIdx.x;
      v[u] = vload_el<T, N, true>(zs + head + uint64_t(at < vectors ? at : vectors - 1) * N);
    }
  };
  // the first 64 entries and the first logits, all on their way at once
  const RawEntry e0 = entry_load(p, row, lane);
  const RawId raw_label = p.labels.at ? id_load(p.labels, row) : RawId{0, 1};
  if (whole > 0) fetch(0);
  else if (vectors > 0) fetch_rest();
  const RowTerms terms = row_terms(p, row, lane, e0, raw_label);
  if (!terms.soft && !terms.hard) {
    if (!PART && threadIdx.x == 0) row_unused(p, row);
    return;
  }
  float z0 = 0.0f;
  if (!PART && wave == 0 && terms.i0 < p.width) z0 = float(z[terms.i0]);

  float m = -__FLT_MAX__, s = 0.0f, s1 = 0.0f;
  auto raise = [&](float high) {
    s *= sum_change(m, high, p.c, p.near);
    if (TWO) s1 *= sum_change(m, high, kLog2e, p.near);
    m = high;
  };
  auto one = [&](float w, float w1) {
    s += w;
    if (SUMS == kTwo) s1 += w1;
    if (SUMS == kSquare) s1 = __builtin_fmaf(w, w, s1);
  };
  auto sum = [&](const auto& x, auto COUNT) {
    if (__builtin_fabsf(m) < p.near) {
      const float mc = -(m * p.c), mc1 = -(m * kLog2e);
#pragma unroll
      for (int e = 0; e < COUNT.value; ++e)
        one(exp2_fast(__builtin_fmaf(x[e], p.c, mc)), SUMS == kTwo ? exp2_fast(__builtin_fmaf(x[e], kLog2e, mc1)) : 0.0f);
    } else {
#pragma unroll
      for (int e = 0; e < COUNT.value; ++e)
        one(exp2_fast((x[e] - m) * p.c), SUMS == kTwo ? exp2_fast((x[e] - m) * kLog2e) : 0.0f);
    }
  };
  auto add = [&](auto REST) {
    float x[N * U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e)
        x[u * N + e] = !REST.value || whole + u * BLOCK + threadIdx.x < vectors ? float(v[u].v[e]) : -__builtin_inff();
    float high = m;
#pragma unroll
    for (int e = 0; e < N * U; ++e) high = fmaxf(high, x[e]);
    raise(high);
    sum(x, std::integral_constant<int, N * U>{});
  };
  for (uint32_t base = 0; base < whole; base += BLOCK * U) {
    if (base > 0) fetch(base);
    add(std::false_type{});
  }
  if (whole < vectors) {
    if (whole > 0) fetch_rest();
    add(std::true_type{});
  }
  if (threadIdx.x < width - vectors * N) {  // the columns in front of and behind the vectors
    const float x[1] = {float(zs[threadIdx.x < head ? threadIdx.x : threadIdx.x + vectors * N])};
    raise(fmaxf(m, x[0]));
    sum(x, std::integral_constant<int, 1>{});
  }
  float most = wave_max(m);
  s = wave_sum(s * sum_change(m, most, p.c, p.near));
  if (TWO) s1 = wave_sum(s1 * sum_change(m, most, kLog2e, p.near));
  if constexpr (kWaves > 1) {
    if (lane == 0) {
      part[wave][0] = most;
      part[wave][1] = s;
      part[wave][2] = s1;
    }
    __syncthreads();
    if (wave != 0) return;
    m = lane < kWaves ? part[lane][0] : -__FLT_MAX__;
    most = wave_max(m);
    s = wave_sum(lane < kWaves ? part[lane][1] * sum_change(m, most, p.c, p.near) : 0.0f);
    if (TWO) s1 = wave_sum(lane < kWaves ? part[lane][2] * sum_change(m, most, kLog2e, p.near) : 0.0f);
  }
  if constexpr (PART) {
    if (lane != 0) return;
    float* to = p.parts + (uint64_t(row) * p.segments + seg) * 3;
    to[0] = most;
    to[1] = s;
    to[2] = s1;
  } else {
    row_finish<T, SUMS, KR>(p, row, lane, z, terms, z0, most, s, s1);
  }
}

// The segments of a row, at most 64, to a wave.
template <class T, int SUMS, int KR>
__global__ __launch_bounds__(64) void k_distill_join(DistillArgs p) {
  const uint32_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const T* z = static_cast<const T*>(p.logits) + uint64_t(row) * p.pitch;
  const RawEntry e0 = entry_load(p, row, lane);
  const RawId raw_label = p.labels.at ? id_load(p.labels, row) : RawId{0, 1};
  const float* from = p.parts + (uint64_t(row) * p.segments + (uint32_t(lane) < p.segments ? lane : 0)) * 3;
  const float m0 = from[0], s0 = from[1], s10 = from[2];
  const RowTerms terms = row_terms(p, row, lane, e0, raw_label);
  if (!terms.soft && !terms.hard) {
    if (lane == 0) row_unused(p, row);
    return;
  }
  const float z0 = terms.i0 < p.width ? float(z[terms.i0]) : 0.0f;
  const bool there = uint32_t(lane) < p.segments;
  const float m = there ? m0 : -__FLT_MAX__, most = wave_max(m);
  const float s = wave_sum(there ? s0 * sum_change(m, most, p.c, p.near) : 0.0f);
  const float s1 = SUMS != kOne ? wave_sum(there ? s10 * sum_change(m, most, kLog2e, p.near) : 0.0f) : 0.0f;
  row_finish<T, SUMS, KR>(p, row, lane, z, terms, z0, most, s, s1);
}

// A workgroup of one wave takes a segment of a row, four vectors of 16 bytes to a lane: dloss (weight T softmax(z / T) +
// (1 - weight) softmax(z)) of every column, from the maximum and the logarithms of the sums that the loss left, less what
// the teacher's entries and the label take off.  While the logits are on their way the wave lists the segment's
// entries in LDS, and under every column the place of what is taken off there; a column that several entries name has
// one place, with their sum.  So every value is stored once, and no wave waits for another.
constexpr int kGradVectors = 4;
constexpr unsigned grad_lds(uint32_t entries) { return (entries + 1) * 12; }

// KR: entries that a lane loads at once, before everything else ((3000, 32000) with 200 entries 101 us, 64 at a time 115).
// NT: streaming stores, from kStreamStoreBytes on, as elsewhere.  Alone, smaller gradients take up to an eighth longer without ((128,
// 32768) bf16 8.9 us, streamed 7.9; (512, 32768) 15.2 and 14.0), but whatever reads them next finds them in the caches (the two
// together with a maximum of each row 18.7 and 21.0, 26.9 and 29.3).
template <class T, bool SQUARE, int KR, bool NT>
__global__ __launch_bounds__(64, KR > 2 ? 7 : 8) void k_distill_grad(DistillArgs p) {
  constexpr int N = 16 / int(sizeof(T)), U = kGradVectors, kColumns = 64 * U * N;
  __shared__ Vec<uint16_t, N> map[64 * U];  // of the vectors' columns: 0, or 1 + the place in the list
  extern __shared__ uint32_t column[];      // [entries + 1] the list: columns, the entries' exponentials, what is taken off
  float* part = reinterpret_cast<float*>(column + p.entries + 1);
  float* taken = part + p.entries + 1;
  const uint32_t row = blockIdx.x / p.segments, seg = blockIdx.x - row * p.segments, lane = threadIdx.x;
  const T* z = static_cast<const T*>(p.logits) + uint64_t(row) * p.pitch;
  T* out = static_cast<T*>(p.grad) + uint64_t(row) * p.width;

  // Vectors lie where the results' addresses are multiples of 16 bytes, segments where they are multiples of 4 KB (and the
  // logits' too, where both rows begin alike): no line is shared with another wave, but at a row's ends.  The first segment has
  // the columns in front of the vectors, the last one those behind.
  const uint32_t head = row_head<T>(out, p.width), vectors = (p.width - head) / N;
  const int32_t start = int32_t(seg * (64 * U)) - int32_t(reinterpret_cast<uintptr_t>(out + head) / 16 % (64 * U));
  if (seg > 0 && start >= int32_t(vectors)) return;
  const uint32_t from = start < 0 ? 0 : uint32_t(start);
  const uint32_t to = start + 64 * U < int32_t(vectors) ? uint32_t(start + 64 * U) : vectors;
  const uint32_t base = head + uint32_t(start) * N;  // the first vector's column (below 0: past all columns)
  const uint32_t first = seg == 0 ? 0 : base, last = to == vectors ? p.width : head + to * N;
  const uint32_t before = seg == 0 ? head : 0;
  uint32_t lone = lane < before ? lane : head + vectors * N + (lane - before);
  if (lane >= before && to < vectors) lone = p.width;
  auto vector = [&](int u) { return uint32_t(start + u * 64) + lane; };
  // The first entries, which are waited for before the logits are asked for: with all loads under way at once (4096, 131072) bf16
  // took 350 us, so 342.
  RawEntry raw[KR];
#pragma unroll
  for (int k = 0; k < KR; ++k) raw[k] = entry_load(p, row, k * 64 + lane);
  const RawId raw_label = p.labels.at ? id_load(p.labels, row) : RawId{0, 1};
  uint32_t ki[KR];
  float kx[KR];
#pragma unroll
  for (int k = 0; k < KR; ++k) entry_of(p, raw[k], k * 64 + lane, ki[k], kx[k]);
  const float dl = p.dloss[int64_t(row) * p.dloss_stride];
  const float m = p.sums[uint64_t(row) * 3];
  const float ls = p.sums[uint64_t(row) * 3 + 1], ls1 = p.sums[uint64_t(row) * 3 + 2];
  Vec<T, N> v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t at = vector(u);
    if (at >= from && at < to) v[u] = vload_el<T, N, true>(z + head + uint64_t(at) * N);
    map[u * 64 + lane] = Vec<uint16_t, N>{};
  }

  const uint32_t label = id_of(raw_label, p.width);
  const bool hard = label < p.width;
  const float ka = dl * p.soft, kb = dl * p.hard, la = ls * kLog2e, lb = ls1 * kLog2e;
  auto each = [&](auto fn) {  // an entry that counts to a lane, or the width in its place
#pragma unroll
    for (int k = 0; k < KR; ++k)
      if (k == 0 || k * 64 < int(p.entries)) fn(ki[k], kx[k]);
    for (uint32_t k0 = KR * 64; k0 < p.entries; k0 += 64) {
      uint32_t i;
      float x;
      teacher_entry(p, row, k0 + lane, i, x);
      fn(i, x);
    }
  };
  float top = -__builtin_inff(), a = 0.0f;
  bool some = false;
  each([&](uint32_t i, float x) {
    if (i >= p.width) return;
    some = true;
    top = fmaxf(top, x);
  });
  const bool soft = __ballot(some) != 0;
  uint32_t listed = 0;
  if (soft) {
    top = wave_max(top);
    each([&](uint32_t i, float x) {
      const float e = i < p.width ? exp2_fast((x - top) * p.c) : 0.0f;
      a += e;
      const bool here = i >= first && i < last;
      const uint64_t those = __ballot(here);
      if (here) {
        const uint32_t at = listed + uint32_t(__popcll(those & ((uint64_t(1) << lane) - 1)));
        column[at] = i;
        part[at] = e;
      }
      listed += uint32_t(__popcll(those));
    });
    a = wave_sum(a);
  }
  {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    uint16_t* place = reinterpret_cast<uint16_t*>(map);
    bool labelled = false;  // whether an entry's column is the label's
    // Every entry writes its place; one that finds another's there, or has no vector, has the list searched for columns that are
    // named more than once ((16384, 4000) with 128 entries 68 us, with a search each time 112).
    for (uint32_t k = lane; k < listed; k += 64)
      if (column[k] - base < uint32_t(kColumns)) place[column[k] - base] = uint16_t(k + 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    bool again = false;
    for (uint32_t k = lane; k < listed; k += 64)
      if (column[k] - base >= uint32_t(kColumns) || place[column[k] - base] != k + 1) again = true;
    const bool search = __ballot(again) != 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    for (uint32_t k = lane; k < listed; k += 64) {
      const uint32_t i = column[k];
      float sum = part[k];
      bool leads = true;
      if (search) {
        sum = 0.0f;
        for (uint32_t j = 0; j < listed; ++j) {
          if (column[j] != i) continue;
          if (j < k) leads = false;
          sum += part[j];
        }
      }
      sum = ka * (sum / a);
      if (hard && i == label) {
        labelled = true;
        sum += kb;
      }
      taken[k] = sum;
      if (leads && i - base < uint32_t(kColumns)) place[i - base] = uint16_t(k + 1);
    }
    if (__ballot(labelled) == 0 && hard && label >= first && label < last) {
      if (lane == 0) {
        column[listed] = label;
        taken[listed] = kb;
        if (label - base < uint32_t(kColumns)) place[label - base] = uint16_t(listed + 1);
      }
      ++listed;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  }

  auto stream = [&](auto fn) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t at = vector(u);
      if (at < from || at >= to) continue;
      const Vec<uint16_t, N> where = map[u * 64 + lane];
      float g[N];
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        g[e] = fn(float(v[u].v[e]));
        any |= where.v[e];
      }
      if (any) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (where.v[e]) g[e] -= taken[where.v[e] - 1];
      }
      Vec<T, N> o;
#pragma unroll
      for (int e = 0; e < N; ++e) o.v[e] = T(g[e]);
      vstore_el<NT, T, N>(out + head + uint64_t(at) * N, o);
    }
    if (lone < p.width) {
      float g = fn(float(z[lone]));
      for (uint32_t j = 0; j < listed; ++j)
        if (column[j] == lone) {  // the first of those that name it
          g -= taken[j];
          break;
        }
      out[lone] = T(g);
    }
  };
  auto q = [&](float x) { return exp2_fast(__builtin_fmaf(x - m, p.c, -la)); };
  auto s = [&](float x) { return exp2_fast(__builtin_fmaf(x - m, kLog2e, -lb)); };
  if (soft && hard && SQUARE) {  // exp(z - m) is the square of exp((z - m) / 2)
    const float kc = kb * exp2_fast(2.0f * la - lb);
    stream([&](float x) {
      const float w = q(x);
      return w * __builtin_fmaf(kc, w, ka);
    });
  } else if (soft && hard && p.c == kLog2e) {  // T = 1: one softmax
    stream([&](float x) { return (ka + kb) * q(x); });
  } else if (soft && hard) {
    stream([&](float x) { return ka * q(x) + kb * s(x); });
  } else if (soft) {
    stream([&](float x) { return ka * q(x); });
  } else if (hard) {
    stream([&](float x) { return kb * s(x); });
  } else {
    stream([&](float) { return 0.0f; });
  }
}

// Segments of a row in the loss: few rows are split into what fills the chip, if they are long enough to be worth a second launch (one
// row of 262144 bf16 8 us, whole 16; 64 of 131072 11.3 and 14.6; but 256 of them 20 and 17, 64 of 32768 9 and 6).
static uint32_t distill_segments(uint64_t rows, uint64_t width, uint64_t size) {
  if (rows == 0 || rows > 128 || width * size < 192 * 1024) return 1;
  const uint64_t wanted = (1024 + rows - 1) / rows, most = width * size / 8192;
  const uint64_t n = wanted < most ? wanted : most;
  return uint32_t(n < 64 ? n : 64);
}

static bool distill_args(const musapy_distill_args* a, bool grad, DistillArgs& p) {
  if (a == nullptr || !vocab_float(a->dtype) || a->rows >= kVocabLimit || a->width >= kVocabLimit) return false;
  if (a->entries > size_t(kEntriesMost) || !(a->temperature >= 0x1p-20f && a->temperature <= 0x1p20f)) return false;
  if (!(a->weight >= 0.0f && a->weight <= 1.0f)) return false;
  if (a->entries > 0 && (!vocab_id(a->index_dtype) || !vocab_float(a->teacher_dtype))) return false;
  if (a->labels != nullptr && !vocab_id(a->label_dtype)) return false;
  p.logits = a->logits;
  p.pitch = a->pitch;
  p.index = vocab_ids(a->index, a->index_dtype);
  p.index_pitch = a->index_pitch;
  p.teacher = a->teacher;
  p.teacher_dtype = a->teacher_dtype;
  p.teacher_pitch = a->teacher_pitch;
  p.use_soft = a->weight > 0.0f && a->entries > 0;
  p.labels = vocab_ids(a->weight < 1.0f ? a->labels : nullptr, a->label_dtype);
  p.rows = uint32_t(a->rows);
  p.width = uint32_t(a->width);
  p.entries = uint32_t(a->entries);
  p.inv_t = 1.0f / a->temperature;
  p.c = kLog2e / a->temperature;
  p.near = kNearExponent / (p.c > kLog2e ? p.c : kLog2e);
  p.soft = a->weight * a->temperature * (grad ? 1.0f : a->temperature);
  p.hard = 1.0f - a->weight;
  p.loss = a->loss;
  p.sums = a->sums;
  p.dloss = a->dloss;
  p.dloss_stride = a->dloss_stride;
  p.grad = a->dlogits;
  return true;
}

}  // namespace mpy

using namespace mpy;

extern "C" {

size_t musapy_distill_loss_scratch_v1(const musapy_distill_args* a) {
  DistillArgs p{};
  if (!distill_args(a, false, p)) return 0;
  const uint32_t n = distill_segments(p.rows, p.width, a->dtype == MUSAPY_DT_F32 ? 4 : 2);
  return n > 1 ? size_t(p.rows) * n * 3 * sizeof(float) : 0;
}

int musapy_distill_loss_v1(const musapy_distill_args* a, void* scratch, size_t scratch_bytes, hipStream_t st) {
  DistillArgs p{};
  if (!distill_args(a, false, p)) return vocab_bad();
  if (p.rows == 0) return 0;
  // The fewest waves a row that still fill the chip, since a row takes some 6 us however short it is: one with 2048 rows of up to 16 KB
  // or 8192 of up to 32 KB (bf16, (5000, 1408) 9.8 us, with four waves 17.0, with eight 30.2; (7500, 8000) 24.5, 25.5 and 42.9), four
  // with 2048 of up to 128 KB.  With more than 32 vectors a thread the larger workgroups are level or better, and with 1000 rows all are.
  const uint64_t vectors = uint64_t(p.width) * (a->dtype == MUSAPY_DT_F32 ? 4 : 2) / 16;
  const bool one_wave = (p.rows >= 2048 && vectors <= 16 * 64) || (p.rows >= 8192 && vectors <= 32 * 64);
  const unsigned block = one_wave ? 64 : p.rows >= 2048 && vectors <= 32 * 256 ? 256 : 512;
  if (p.loss == nullptr || p.sums == nullptr || (p.width > 0 && p.logits == nullptr) ||
      (p.entries > 0 && (p.index.at == nullptr || p.teacher == nullptr)) || !grid_fits(p.rows, block))
    return vocab_bad();
  const size_t need = musapy_distill_loss_scratch_v1(a);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 3))) return vocab_bad(1);
  const bool two = p.labels.at != nullptr && a->temperature != 1.0f;
  vocab_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto SUMS, auto KEPT) {
      constexpr int kS = SUMS.value, kK = KEPT.value;
      p.segments = distill_segments(p.rows, p.width, sizeof(T));
      if (p.segments > 1) {
        p.parts = static_cast<float*>(scratch);
        p.segment = (p.width / p.segments + 64) / 64 * 64;  // at least width / segments: no more segments than asked for
        p.segments = (p.width + p.segment - 1) / p.segment;
        k_distill_loss<T, 512, kS, true, 1><<<p.rows * p.segments, 512, 0, st>>>(p);
        k_distill_join<T, kS, kK><<<p.rows, 64, 0, st>>>(p);
        return;
      }
      if (block == 64) k_distill_loss<T, 64, kS, false, kK><<<p.rows, 64, 0, st>>>(p);
      else if (block == 256) k_distill_loss<T, 256, kS, false, kK><<<p.rows, 256, 0, st>>>(p);
      else k_distill_loss<T, 512, kS, false, kK><<<p.rows, 512, 0, st>>>(p);
    };
    auto sums = [&](auto KEPT) {
      if (two && a->temperature == 2.0f) go(std::integral_constant<int, kSquare>{}, KEPT);
      else if (two) go(std::integral_constant<int, kTwo>{}, KEPT);
      else go(std::integral_constant<int, kOne>{}, KEPT);
    };
    if (p.entries <= 64) sums(std::integral_constant<int, 1>{});
    else sums(std::integral_constant<int, 4>{});
  });
  return 0;
}

int musapy_distill_loss_grad_v1(const musapy_distill_args* a, hipStream_t st) {
  DistillArgs p{};
  if (!distill_args(a, true, p)) return vocab_bad();
  if (p.rows == 0 || p.width == 0) return 0;
  if (p.logits == nullptr || p.sums == nullptr || p.dloss == nullptr || p.grad == nullptr ||
      (p.entries > 0 && (p.index.at == nullptr || p.teacher == nullptr)))
    return vocab_bad();
  vocab_type(a->dtype, [&](auto t) {
    using T = decltype(t);
    // of 4 KB; one more where rows begin between them
    constexpr uint64_t kSegment = 64 * kGradVectors * 16;
    const uint64_t bytes = p.width * sizeof(T);
    const bool even = reinterpret_cast<uintptr_t>(p.grad) % kSegment == 0 && bytes % kSegment == 0;
    p.segments = uint32_t((bytes + kSegment - 1) / kSegment + (even ? 0 : 1));
    const uint64_t grid = uint64_t(p.rows) * p.segments;
    if (!grid_fits(grid, 64)) {
      p.segments = 0;
      return;
    }
    auto go = [&](auto SQUARE, auto KR) {
      with_store_policy(p.rows * bytes >= kStreamStoreBytes, [&](auto NT) {
        k_distill_grad<T, SQUARE.value, KR.value, NT.value><<<unsigned(grid), 64, grad_lds(p.entries), st>>>(p);
      });
    };
    auto entries = [&](auto SQUARE) {
      if (p.entries <= 64) go(SQUARE, std::integral_constant<int, 1>{});
      else if (p.entries <= 128) go(SQUARE, std::integral_constant<int, 2>{});
      else go(SQUARE, std::integral_constant<int, 4>{});
    };
    if (a->temperature == 2.0f) entries(std::true_type{});
    else entries(std::false_type{});
  });
  if (p.segments == 0) return vocab_bad();
  return 0;
}

}  // extern "C"
