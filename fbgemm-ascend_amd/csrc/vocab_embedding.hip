// vocab_embedding.hip — gfx950 kernels and C ABI of the token embedding and its gradient
// (include/tbe_vocab_ops.h).
//
//   out[i, :]  = scale * W[id_i, :]                        N rows read (distinct ones), N written
//   dW[v, :]   = scale * sum_{i : id_i = v} dOut[i, :]     N rows read, V written
//
// One multiplication or addition per element: both are bound by HBM traffic.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "tbe_internal.h"
#include "tbe_nbit.h"
#include "tbe_vocab_ops.h"
#include "vocab_device.h"

namespace tbe {
namespace vocab {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxBlocks = 0xFFFFFFFFLL / kThreads;  // a launch holds fewer than 2^32 threads

// n / d by one multiply-high (Granlund & Montgomery, PLDI 1994), for n < 2^32 and d >= 1.
struct FastDiv {
  uint32_t d, mul, shift;
  FastDiv(uint32_t by = 1) : d(by), shift(0) {
    while ((uint64_t(1) << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << shift) - d)) / d + 1);
  }
  __device__ uint32_t operator()(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(__umulhi(n, mul)) + n) >> shift);
  }
};

struct LookupParams {
  const void* __restrict__ weight;
  const void* __restrict__ ids;
  void* __restrict__ out;
  int64_t stride;    // of the table, in elements
  int64_t num_rows;
  int64_t width;
  int64_t num_tokens;
  float scale;
  int32_t index_size;
  FastDiv row_vecs;  // vectors of a row of the output
};

__device__ __forceinline__ int64_t load_id(const void* ids, int32_t index_size, int64_t i) {
  return index_size == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// scale * x rounded to 32 bits: without the barrier the compiler fuses it with a rounding to
// 16 bits into one instruction that rounds once, for fp16 only.
__device__ __forceinline__ float scaled(float x, float scale) {
  float r = x * scale;
  asm("" : "+v"(r));
  return r;
}

// A lane's VEC consecutive columns.  The last lanes of a row (of at least VEC columns) are moved
// back to end with it, so that every load and store is a whole vector, at any alignment of the
// element: lanes that overlap hold the same values.
template <typename T, int VEC>
struct Cols {
  typename T::raw r[VEC];
  static constexpr int kWords = static_cast<int>(VEC * sizeof(typename T::raw) / 4);
  typedef uint32_t Words __attribute__((ext_vector_type(kWords > 0 ? kWords : 1), aligned(2)));
  __device__ __forceinline__ void load(const typename T::raw* p) { __builtin_memcpy(r, p, sizeof(r)); }
  __device__ __forceinline__ void store(typename T::raw* p) const { __builtin_memcpy(p, r, sizeof(r)); }
  // The same past the caches' keeping, for what is read or written once.
  __device__ __forceinline__ void load_once(const typename T::raw* p) {
    if constexpr (kWords == 0) {
      load(p);
    } else {
      const Words w = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p));
      __builtin_memcpy(r, &w, sizeof(r));
    }
  }
  __device__ __forceinline__ void store_once(typename T::raw* p) const {
    if constexpr (kWords == 0) {
      store(p);
    } else {
      Words w;
      __builtin_memcpy(&w, r, sizeof(r));
      __builtin_nontemporal_store(w, reinterpret_cast<Words*>(p));
    }
  }
  __device__ __forceinline__ float operator[](int e) const { return to_f32<T>(r[e]); }
};

// Bound by HBM.  kLookupUnroll vectors a thread, consecutive ones (over the ends of rows) in
// consecutive threads; all of a thread's rows are in flight before the first is written.  A
// row's last vector ends with it and overlaps the one before.  Results of more than the L2s
// hold are stored non-temporally.  us, 1 / 2 / 4 vectors a thread, then 2 and non-temporal:
// 16384 rows of 4096 bf16 39.2 / 38.0 / 37.8, 30.4 (5.9 TB/s with the cached rows' reads); 65536 of 512 fp32
// 34.0 / 32.7 / 32.4, 28.6; 65536 of 64 bf16 4.2 / 4.4 / 5.0 (a work-group per row 16.7).
constexpr int kLookupUnroll = 2;
constexpr int64_t kLookupCached = int64_t(32) << 20;  // bytes of a result that is stored to be cached

template <typename TW, typename TO, bool kOnce>
__global__ __launch_bounds__(kThreads) void lookup_kernel(LookupParams p, int64_t first) {
  constexpr int E = kElems<TW> < kElems<TO> ? kElems<TW> : kElems<TO>;
  const uint32_t vecs = p.row_vecs.d;
  const uint64_t base = (static_cast<uint64_t>(first) + blockIdx.x) * (kThreads * kLookupUnroll);
  const uint64_t token0 = base / vecs;
  const uint32_t at0 = static_cast<uint32_t>(base - token0 * vecs) + threadIdx.x;  // < 2^32: vecs < 2^30
  Cols<TW, E> x[kLookupUnroll];
  bool ok[kLookupUnroll];
  int64_t id[kLookupUnroll];
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const int64_t i = std::min<int64_t>(token0 + p.row_vecs(at0 + u * kThreads), p.num_tokens - 1);
    id[u] = load_id(p.ids, p.index_size, i);
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t at = at0 + u * kThreads, r = p.row_vecs(at);
    ok[u] = id[u] >= 0 && id[u] < p.num_rows;
    const auto* src = static_cast<const typename TW::raw*>(p.weight) + (ok[u] ? id[u] : 0) * p.stride;
    x[u] = {};
    if (p.width >= E) {
      if (ok[u]) x[u].load(src + std::min<int64_t>(int64_t(at - r * vecs) * E, p.width - E));
    } else if (ok[u]) {
#pragma unroll
      for (int e = 0; e < E - 1; ++e)
        if (e < p.width) x[u].r[e] = src[e];
    }
  }
#pragma unroll
  for (int u = 0; u < kLookupUnroll; ++u) {
    const uint32_t at = at0 + u * kThreads, r = p.row_vecs(at);
    const int64_t i = static_cast<int64_t>(token0 + r);
    if (i >= p.num_tokens) break;
    auto* dst = static_cast<typename TO::raw*>(p.out) + i * p.width;
    Cols<TO, E> y;
#pragma unroll
    for (int e = 0; e < E; ++e) y.r[e] = from_f32<TO>(ok[u] ? scaled(x[u][e], p.scale) : 0.f);
    if (p.width >= E) {
      auto* to = dst + std::min<int64_t>(int64_t(at - r * vecs) * E, p.width - E);
      if constexpr (kOnce) {
        y.store_once(to);
      } else {
        y.store(to);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E - 1; ++e)
        if (e < p.width) dst[e] = y.r[e];
    }
  }
}

// ---------------------------------------------------------------- gradient

struct GradParams {
  const void* __restrict__ grad;
  const void* __restrict__ ids;
  void* __restrict__ out;
  int64_t stride;    // of grad, in elements
  int64_t padding;
  int64_t width;
  uint32_t num_tokens;
  uint32_t num_rows;
  float scale;
  int32_t index_size;
  int32_t accumulate;
  int32_t col_tiles;    // of kWave * VEC columns
  uint32_t work_groups;  // that sum rows; the other `fills` of the launch fill, spread among them
  uint32_t fills;
  uint32_t fill_reps;    // vectors a thread of a filling work-group writes
  uint32_t few_rows;     // rows of a filling work-group of grad_few_kernel
  FastDiv row_vecs;      // 16-byte vectors of a row of the table
};

// The row of position i, or num_rows where it has none.
__device__ __forceinline__ uint32_t row_of(const GradParams& p, uint32_t i) {
  const int64_t id = load_id(p.ids, p.index_size, i);
  return id < 0 || id >= p.num_rows || id == p.padding ? p.num_rows : static_cast<uint32_t>(id);
}

// The sum of a row's gradients, into the table's gradient.  `col` is where the lane's columns
// would begin, `at` where they do.
template <typename TW, int VEC>
__device__ __forceinline__ void write_sum(const GradParams& p, uint32_t row, int64_t col, int64_t at,
                                          const float (&acc)[VEC]) {
  if (col >= p.width) return;
  auto* dst = static_cast<typename TW::raw*>(p.out) + row * p.width + at;
  Cols<TW, VEC> out;
  if (!p.accumulate) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out.r[e] = from_f32<TW>(p.scale * acc[e]);
    out.store_once(dst);
  } else if (at == col) {
    out.load(dst);
#pragma unroll
    for (int e = 0; e < VEC; ++e) out.r[e] = from_f32<TW>(fmaf(p.scale, acc[e], out[e]));
    out.store(dst);
  } else {  // the columns that no other lane adds to
    for (int e = static_cast<int>(col - at); e < VEC; ++e) {
      float sum = acc[0];
#pragma unroll
      for (int i = 1; i < VEC; ++i) sum = i == e ? acc[i] : sum;
      dst[e] = from_f32<TW>(fmaf(p.scale, sum, to_f32<TW>(dst[e])));
    }
  }
}

// Zeros are written in the order of the work-groups, 16 bytes a thread: 512 MiB in 80 us; with 16
// to 64 KiB a work-group, or a grid that strides over the whole, 86-138 us.  They are not read
// here and stored non-temporally.
__device__ __forceinline__ void store_zeros(uint8_t* p) { store16_once(p, Vec16{}); }

// Whether this work-group fills, and its number among its kind.
__device__ __forceinline__ bool is_fill(const GradParams& p, uint32_t& number) {
  number = blockIdx.x;
  if (p.fills == 0) return false;
  const uint64_t all = static_cast<uint64_t>(p.work_groups) + p.fills;
  const uint32_t sums = static_cast<uint32_t>(static_cast<uint64_t>(blockIdx.x) * p.work_groups / all);
  const uint32_t next = static_cast<uint32_t>((static_cast<uint64_t>(blockIdx.x) + 1) * p.work_groups / all);
  number = next > sums ? sums : blockIdx.x - sums;
  return next == sums;
}

// Zeros to the vec-th 16 bytes of a row of the table.
template <typename TW>
__device__ __forceinline__ void zero_vec(const GradParams& p, int64_t row, uint32_t vec) {
  const int64_t row_bytes = p.width * sizeof(typename TW::raw);
  auto* to = static_cast<uint8_t*>(p.out) + row * row_bytes;
  if (row_bytes >= 16) {
    store_zeros(to + std::min<int64_t>(int64_t(vec) * 16, row_bytes - 16));  // the last one ends with the row
  } else {
    for (int64_t e = 0; e < p.width; ++e) reinterpret_cast<typename TW::raw*>(to)[e] = 0;
  }
}

// Zeros to the rows that no token names (all rows without marks): a piece of kThreads *
// p.fill_reps vectors per work-group.
template <typename TW>
__device__ __forceinline__ void fill_piece(const GradParams& p, uint32_t piece, const uint8_t* present) {
  const uint32_t vecs = p.row_vecs.d;
  uint64_t first = static_cast<uint64_t>(piece) * kThreads * p.fill_reps;
  for (uint32_t rep = 0; rep < p.fill_reps; ++rep, first += kThreads) {
    const uint64_t row0 = first / vecs;
    const uint32_t at = static_cast<uint32_t>(first - row0 * vecs) + threadIdx.x;  // < 2^32: vecs < 2^29
    const uint32_t r = p.row_vecs(at);
    const uint64_t row = row0 + r;
    if (row < p.num_rows && !(present && present[row])) zero_vec<TW>(p, row, at - r * vecs);
  }
}

template <typename TW>
__global__ __launch_bounds__(kThreads) void fill_kernel(GradParams p) {
  fill_piece<TW>(p, blockIdx.x, nullptr);
}

// Few tokens (kFewTokens at most): one launch.  A work-group per position and tile of columns;
// the first position of a token lists all of them in order, its four waves sum every fourth
// row, and the waves' sums are added in their order.  The other work-groups fill, each the rows
// of kFewFill bytes, after a look through the tokens for those it must leave out.  Past
// kFewFillAll bytes of table the whole of it is filled by a launch before instead.
constexpr uint32_t kFewTokens = 1024;
constexpr uint32_t kFewRows = 8192;  // most rows of one filling work-group
constexpr int64_t kFewFill = 65536;
constexpr int64_t kFewFillAll = int64_t(64) << 20;
// The sort's three launches take 15-18 us of themselves; the reads of the token list by one
// work-group per token and tile cost 10 us at 1000 tokens of 1024 columns (2 tiles), 18-22 us of
// 4096 columns.
constexpr int64_t kFewReads = int64_t(4) << 20;

template <typename TG, typename TW, int VEC>
__global__ __launch_bounds__(kThreads) void grad_few_kernel(GradParams p) {
  constexpr int kWaves = kThreads / kWave;
  __shared__ uint32_t shared[kFewTokens];
  uint32_t group;
  if (is_fill(p, group)) {
    const uint32_t r0 = group * p.few_rows, r1 = std::min(r0 + p.few_rows, p.num_rows);
    for (uint32_t i = threadIdx.x; i < kFewRows / 32; i += kThreads) shared[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < p.num_tokens; i += kThreads) {
      const uint32_t row = row_of(p, i);
      if (row >= r0 && row < r1) atomicOr(&shared[(row - r0) / 32], 1u << ((row - r0) & 31));
    }
    __syncthreads();
    const uint32_t vecs = p.row_vecs.d, items = (r1 - r0) * vecs;
    for (uint32_t it = threadIdx.x; it < items; it += kThreads) {
      const uint32_t r = p.row_vecs(it);
      if (!((shared[r / 32] >> (r & 31)) & 1)) zero_vec<TW>(p, r0 + r, it - r * vecs);
    }
    return;
  }
  __shared__ uint32_t counts[kWaves];
  __shared__ float sums[kWaves - 1][VEC][kWave];
  const uint32_t at = group / p.col_tiles, tile = group % p.col_tiles;
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const uint32_t row = row_of(p, at);
  if (row == p.num_rows) return;
  uint32_t found = 0;
  for (uint32_t j0 = 0; j0 < p.num_tokens; j0 += kThreads) {
    const uint32_t j = j0 + threadIdx.x;
    const bool match = j < p.num_tokens && row_of(p, j) == row;
    if (__syncthreads_or(match && j < at)) return;  // an earlier position's work-group sums
    const uint64_t mask = __ballot(match);
    if (lane == 0) counts[wave] = __popcll(mask);
    __syncthreads();
    uint32_t before = found;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += counts[w];
      found += counts[w];
    }
    if (match) shared[before + __popcll(mask & ((1ull << lane) - 1))] = j;
  }
  __syncthreads();
  const int64_t col = (static_cast<int64_t>(tile) * kWave + lane) * VEC;
  const int64_t col_at = std::min(col, p.width - VEC);
  const auto* grad = static_cast<const typename TG::raw*>(p.grad) + col_at;
  float acc[VEC] = {};
#pragma unroll 8
  for (uint32_t k = wave; k < found; k += kWaves) {
    Cols<TG, VEC> x;
    x.load_once(grad + shared[k] * p.stride);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] += x[e];
  }
  if (found > 1) {
    if (wave > 0) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[wave - 1][e][lane] = acc[e];
    }
    __syncthreads();
    if (wave == 0) {
      for (int w = 0; w < kWaves - 1; ++w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += sums[w][e][lane];
      }
    }
  }
  if (wave == 0) write_sum<TW, VEC>(p, row, col, col_at, acc);
}

// Many tokens: positions are sorted by row (a stable radix sort of kBits a pass), and the rows
// are summed from chunks of sorted positions.
constexpr int kBits = 9;
constexpr uint32_t kBins = 1u << kBits;
constexpr uint32_t kBlock = 4 * kThreads;  // items a work-group sorts at a time
constexpr uint32_t kMaxTiles = 256;        // work-groups of a pass

struct SortParams {
  const uint2* __restrict__ in;          // (row, position); of the first pass, the ids
  uint2* __restrict__ out;
  uint32_t* __restrict__ counts;         // [tiles][kBins] of this pass
  uint8_t* __restrict__ present;         // [num_rows] or null: set in the first pass
  uint32_t tile, tiles;                  // items of a tile, a multiple of kBlock
  int32_t shift;
};

// Counts of a pass's digits, a tile per work-group.  In the first pass, zeros to `present` too.
__global__ __launch_bounds__(kThreads) void sort_count_kernel(GradParams p, SortParams s, int64_t zero_vecs) {
  __shared__ uint32_t bins[kBins];
  for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) bins[b] = 0;
  __syncthreads();
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * s.tile;
  const uint32_t end = static_cast<uint32_t>(std::min<uint64_t>(first + s.tile, p.num_tokens));
#pragma unroll 4
  for (uint64_t i = first + threadIdx.x; i < end; i += kThreads) {
    const uint32_t row = s.shift == 0 ? row_of(p, static_cast<uint32_t>(i)) : s.in[i].x;
    atomicAdd(&bins[(row >> s.shift) & (kBins - 1)], 1u);
  }
  __syncthreads();
  if (first < p.num_tokens) {
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) s.counts[blockIdx.x * kBins + b] = bins[b];
  }
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < zero_vecs;
       i += static_cast<int64_t>(gridDim.x) * kThreads)
    store16(s.present + 16 * i, Vec16{});
}

// A wave's lanes of the same digit before this one, added to the digit's count so far in the wave.
template <typename C>
__device__ __forceinline__ uint32_t rank_of(uint32_t digit, bool in, C* count) {
  uint64_t same = __ballot(in);
#pragma unroll
  for (int k = 0; k < kBits; ++k) {
    const uint64_t ones = __ballot((digit >> k) & 1);
    same &= (digit >> k) & 1 ? ones : ~ones;
  }
  const int before = __popcll(same & ((1ull << lane_id()) - 1));
  const uint32_t rank = count[digit] + before;
  wave_fence();
  if (in && before == 0) count[digit] += __popcll(same);
  wave_fence();
  return rank;
}

// One pass: a tile per work-group.  An item's place is the number of items of lower digits, of
// its digit in earlier tiles, in earlier waves of the block and before it in its wave.  The last
// pass's launch also fills the rows that no token names, beside the few work-groups that sort.
template <typename TW>
__global__ __launch_bounds__(kThreads) void sort_pass_kernel(GradParams p, SortParams s) {
  constexpr int kWaves = kThreads / kWave, kRounds = kBlock / kThreads;
  __shared__ uint32_t base[kBins];
  __shared__ uint32_t place[kWaves][kBins];
  if (blockIdx.x >= s.tiles) {
    fill_piece<TW>(p, blockIdx.x - s.tiles, s.present);
    return;
  }
  const int wave = threadIdx.x / kWave, lane = lane_id();
  {  // the bases: totals of the digits scanned, and what earlier tiles hold
    uint32_t total[2] = {}, before[2] = {};
#pragma unroll 8
    for (uint32_t t = 0; t < s.tiles; ++t) {
      const uint2 c = reinterpret_cast<const uint2*>(s.counts + t * kBins)[threadIdx.x];
      if (t < blockIdx.x) before[0] += c.x, before[1] += c.y;
      total[0] += c.x, total[1] += c.y;
    }
    uint32_t sum = total[0] + total[1], scan = sum;
    for (int j = 1; j < kWave; j *= 2) {
      const uint32_t o = __shfl_up(scan, j);
      if (lane >= j) scan += o;
    }
    if (lane == kWave - 1) place[0][wave] = scan;
    __syncthreads();
    scan -= sum;
    for (int w = 0; w < wave; ++w) scan += place[0][w];
    base[2 * threadIdx.x] = scan + before[0];
    base[2 * threadIdx.x + 1] = scan + total[0] + before[1];
  }
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * s.tile;
  const uint32_t end = static_cast<uint32_t>(std::min<uint64_t>(first + s.tile, p.num_tokens));
  for (uint64_t b0 = first; b0 < end; b0 += kBlock) {
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kWaves * kBins; b += kThreads) place[b / kBins][b % kBins] = 0;
    __syncthreads();
    uint2 item[kRounds];
    uint32_t digit[kRounds], rank[kRounds];
    const uint64_t i0 = b0 + wave * (kBlock / kWaves) + lane;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      const uint64_t i = i0 + r * kWave;
      item[r] = uint2{0, 0};
      if (i < end) item[r] = s.shift == 0 ? uint2{row_of(p, static_cast<uint32_t>(i)), static_cast<uint32_t>(i)} : s.in[i];
    }
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      digit[r] = (item[r].x >> s.shift) & (kBins - 1);
      rank[r] = rank_of(digit[r], i0 + r * kWave < end, place[wave]);
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < kBins; b += kThreads) {
      uint32_t at = base[b];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t c = place[w][b];
        place[w][b] = at;
        at += c;
      }
      base[b] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (i0 + r * kWave >= end) continue;
      s.out[place[wave][digit[r]] + rank[r]] = item[r];
      if (s.shift == 0 && s.present && item[r].x < p.num_rows) s.present[item[r].x] = 1;
    }
  }
}

constexpr int kSortThreads = 1024;

// Zeros to the whole table's gradient, by the work-groups from `first` on.
__device__ __forceinline__ void fill_all(uint8_t* zeros, int64_t bytes, uint32_t first) {
  const int64_t n = bytes / 16, group = blockIdx.x - first;
  for (int64_t i = group * kSortThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x - first) * kSortThreads)
    store_zeros(zeros + 16 * i);
  if (group == 0 && threadIdx.x < bytes % 16) zeros[16 * n + threadIdx.x] = 0;
}

// Up to kSmallSort tokens and kSmallGroups * kBins rows: one launch sorts.  A work-group per kBins rows
// of the table looks at every id, gathers the positions of its rows in their order and sorts them
// by counting; the number of ids of lower rows is where they begin in the sorted order, so no
// work-group needs another's result.  The last work-groups write zeros to the whole table's
// gradient (a row in four is written again at most, or the zeros take no longer than the sort: else
// the rows are filled after the sort, by their marks).  Against the passes, which are four launches
// (us, the whole gradient): 8192 tokens, 32000 x 1024 bf16 37.7 -> 25.2, 8000 x 64 26.3 -> 20.9.  With as
// many groups as CUs the zeros wait for them (128256 x 2048 105 -> 112), and up to kBins rows are one group
// whatever the tokens (300 x 2048 26.5 -> 32.4).
constexpr uint32_t kSmallSort = 8192;
constexpr int64_t kSmallGroups = 224, kFillBeside = int64_t(80) << 20;

__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(GradParams p, SortParams s, uint32_t groups,
                                                                  uint8_t* zeros, int64_t zero_bytes) {
  constexpr int kWaves = kSortThreads / kWave, kRounds = kSmallSort / kSortThreads;
  static_assert(kSmallSort <= 1u << 16 && kBins <= 1u << 16, "an item is a row of the group's and a position");
  __shared__ uint32_t items[kSmallSort];
  __shared__ uint16_t place[kWaves][kBins];
  __shared__ uint32_t base[kBins], sums[kWaves], lower[kWaves];
  if (blockIdx.x >= groups) {
    fill_all(zeros, zero_bytes, groups);
    return;
  }
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const uint32_t row0 = blockIdx.x * kBins;
  // a wave looks at consecutive positions, as many rounds of 64 as there are
  const uint32_t rounds = (p.num_tokens + kSortThreads - 1) / kSortThreads;
  const uint32_t i0 = wave * rounds * kWave + lane;
  uint32_t row[kRounds], mine = 0, less = 0;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = i0 + r * kWave;
    row[r] = static_cast<uint32_t>(r) < rounds && i < p.num_tokens ? row_of(p, i) : 0xFFFFFFFFu;
  }
  for (uint32_t b = threadIdx.x; b < kWaves * kBins; b += kSortThreads) place[b / kBins][b % kBins] = 0;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    mine += __popcll(__ballot(row[r] - row0 < kBins));
    less += __popcll(__ballot(row[r] < row0));
  }
  if (lane == 0) {
    sums[wave] = mine;
    lower[wave] = less;
  }
  __syncthreads();
  uint32_t at = 0, count = 0, first = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    at += w < wave ? sums[w] : 0;
    count += sums[w];
    first += lower[w];
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const bool in = row[r] - row0 < kBins;
    const uint64_t all = __ballot(in);
    if (in) items[at + __popcll(all & ((1ull << lane) - 1))] = (row[r] - row0) << 16 | (i0 + r * kWave);
    at += __popcll(all);
  }
  __syncthreads();
  const uint32_t turns = (count + kSortThreads - 1) / kSortThreads;
  const uint32_t j0 = wave * turns * kWave + lane;
  uint32_t item[kRounds], rank[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t j = j0 + r * kWave;
    if (static_cast<uint32_t>(r) < turns) {
      item[r] = j < count ? items[j] : 0;
      rank[r] = rank_of(item[r] >> 16, j < count, place[wave]);
    }
  }
  __syncthreads();
  uint32_t total = 0, scan = 0;
  if (threadIdx.x < kBins) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t c = place[w][threadIdx.x];
      place[w][threadIdx.x] = static_cast<uint16_t>(total);
      total += c;
    }
    scan = total;
    for (int j = 1; j < kWave; j *= 2) {
      const uint32_t o = __shfl_up(scan, j);
      if (lane >= j) scan += o;
    }
    if (lane == kWave - 1) sums[wave] = scan;
    const uint64_t marked = static_cast<uint64_t>(row0) + threadIdx.x;
    if (s.present && marked < p.num_rows) s.present[marked] = total > 0;
  }
  __syncthreads();
  if (threadIdx.x < kBins) {
    scan -= total;
    for (int w = 0; w < wave; ++w) scan += sums[w];
    base[threadIdx.x] = first + scan;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    if (static_cast<uint32_t>(r) >= turns || j0 + r * kWave >= count) continue;
    const uint32_t digit = item[r] >> 16;
    s.out[base[digit] + place[wave][digit] + rank[r]] = uint2{row0 + digit, item[r] & 0xFFFF};
  }
}

// Up to kOneSort tokens of another table: the first work-group sorts them in LDS, all passes, and
// the others write zeros (2000 tokens, 1000000 x 64 bf16 29 us, by passes 50).
constexpr uint32_t kOneSort = 4096;

__global__ __launch_bounds__(kSortThreads) void sort_one_kernel(GradParams p, SortParams s, int32_t passes,
                                                                uint8_t* zeros, int64_t zero_bytes) {
  constexpr int kWaves = kSortThreads / kWave, kRounds = kOneSort / kSortThreads;
  __shared__ uint2 items[kOneSort];
  __shared__ uint16_t place[kWaves][kBins];
  __shared__ uint32_t base[kBins], sums[kWaves];
  if (blockIdx.x > 0) {
    fill_all(zeros, zero_bytes, 1);
    return;
  }
  const int wave = threadIdx.x / kWave, lane = lane_id();
  // a wave takes consecutive items, as many rounds of 64 as the tokens need
  const uint32_t rounds = (p.num_tokens + kSortThreads - 1) / kSortThreads;
  const uint32_t i0 = wave * rounds * kWave + lane;
  uint2 item[kRounds];
  if (s.present) {
    for (uint32_t i = threadIdx.x; i < p.num_rows; i += kSortThreads) s.present[i] = 0;
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const uint32_t i = i0 + r * kWave;
    item[r] = uint2{0, 0};
    if (static_cast<uint32_t>(r) < rounds && i < p.num_tokens) {
      item[r] = uint2{row_of(p, i), i};
      if (s.present && item[r].x < p.num_rows) s.present[item[r].x] = 1;
    }
  }
  for (int32_t pass = 0; pass < passes; ++pass) {
    const int32_t shift = pass * kBits;
    for (uint32_t b = threadIdx.x; b < kWaves * kBins; b += kSortThreads) place[b / kBins][b % kBins] = 0;
    __syncthreads();
    uint32_t rank[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (static_cast<uint32_t>(r) < rounds)
        rank[r] = rank_of((item[r].x >> shift) & (kBins - 1), i0 + r * kWave < p.num_tokens, place[wave]);
    }
    __syncthreads();
    uint32_t total = 0, scan = 0;
    if (threadIdx.x < kBins) {
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const uint32_t c = place[w][threadIdx.x];
        place[w][threadIdx.x] = static_cast<uint16_t>(total);
        total += c;
      }
      scan = total;
      for (int j = 1; j < kWave; j *= 2) {
        const uint32_t o = __shfl_up(scan, j);
        if (lane >= j) scan += o;
      }
      if (lane == kWave - 1) sums[wave] = scan;
    }
    __syncthreads();
    if (threadIdx.x < kBins) {
      scan -= total;
      for (int w = 0; w < wave; ++w) scan += sums[w];
      base[threadIdx.x] = scan;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      if (static_cast<uint32_t>(r) < rounds && i0 + r * kWave < p.num_tokens) {
        const uint32_t digit = (item[r].x >> shift) & (kBins - 1);
        items[base[digit] + place[wave][digit] + rank[r]] = item[r];
      }
    }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const uint32_t i = i0 + r * kWave;
        if (static_cast<uint32_t>(r) < rounds && i < p.num_tokens) item[r] = items[i];
      }
    }
  }
  for (uint32_t i = threadIdx.x; i < p.num_tokens; i += kSortThreads) s.out[i] = items[i];
}

struct SumParams {
  const uint2* __restrict__ sorted;       // (row, position)
  const uint8_t* __restrict__ present;
  float* __restrict__ parts;              // [chunks][2][col_tiles * kWave * VEC]: a chunk's first and last run
  uint32_t chunk, chunks;
};

constexpr int kRowsAhead = 8;  // rows a wave has in flight

// A wave per chunk of sorted positions and tile of columns, in one pass over its rows.  A row of
// the table whose run of positions lies inside the chunk is written; the part of a run that
// reaches over the chunk's start or end goes to `parts`, and join_kernel adds the parts of such
// runs.  Bound by HBM: every row of the gradient is read once, non-temporally (65536 distinct tokens
// added to a table of 2048 bf16 columns: 201 -> 163 us with the sort; 4 or 16 rows ahead instead
// of 8: 214, 281).
template <typename TG, typename TW, int VEC>
__global__ __launch_bounds__(kThreads) void grad_sum_kernel(GradParams p, SumParams s) {
  uint32_t group;
  if (is_fill(p, group)) {
    fill_piece<TW>(p, group, s.present);
    return;
  }
  const uint32_t unit = __builtin_amdgcn_readfirstlane(group * (kThreads / kWave) + threadIdx.x / kWave);
  const uint32_t c = unit / p.col_tiles, tile = unit % p.col_tiles;
  if (c >= s.chunks) return;
  const int lane = lane_id();
  const int64_t col = (static_cast<int64_t>(tile) * kWave + lane) * VEC;
  const int64_t col_at = std::min(col, p.width - VEC);
  const auto* grad = static_cast<const typename TG::raw*>(p.grad) + col_at;
  const int64_t part_width = static_cast<int64_t>(p.col_tiles) * kWave * VEC;
  float* parts = s.parts + static_cast<int64_t>(c) * 2 * part_width + col_at;
  auto store_part = [](float* to, const float (&a)[VEC]) { __builtin_memcpy(to, a, sizeof(a)); };
  const uint64_t first = static_cast<uint64_t>(c) * s.chunk;
  const uint32_t end = static_cast<uint32_t>(std::min<uint64_t>(first + s.chunk, p.num_tokens));
  // whether the run being summed began before the chunk
  bool from_before = first > 0 && s.sorted[first - 1].x == s.sorted[first].x;
  bool pending = false;
  float acc[VEC] = {};
  for (uint64_t g = first; g < end; g += kWave) {
    const bool in = g + lane < end;
    const uint2 mine = in ? s.sorted[g + lane] : uint2{p.num_rows, 0};
    const uint32_t next = in && g + lane + 1 < p.num_tokens ? s.sorted[g + lane + 1].x : 0xFFFFFFFFu;
    const int count = __popcll(__ballot(mine.x < p.num_rows));  // positions without a row come last
    for (int j0 = 0; j0 < count; j0 += kRowsAhead) {
      Cols<TG, VEC> x[kRowsAhead];
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        const int j = std::min(j0 + u, count - 1);
        x[u].load_once(grad + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine.y), j)) * p.stride);
      }
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        const int j = j0 + u;
        if (j >= count) break;
        const uint32_t row = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine.x), j));
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = pending ? acc[e] + x[u][e] : x[u][e];
        pending = true;
        if (static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(next), j)) != row) {  // the run ends
          if (from_before) {
            store_part(parts, acc);
          } else {
            write_sum<TW, VEC>(p, row, col, col_at, acc);
          }
          from_before = pending = false;
        }
      }
    }
  }
  if (pending) {
    store_part(parts + (from_before ? 0 : part_width), acc);
  }
}

// Runs that reach over the end of the chunk they begin in.  A work-group of kJoinWaves waves looks
// at as many chunks and a tile of 4 * kWave columns.  A wave adds the parts of its own chunk's
// run where they are few; of a longer run every wave adds its share of the parts, one of
// kJoinWaves, and the waves' sums are added in their order.
constexpr int kJoinWaves = 16;

template <typename TW>
__device__ __forceinline__ void write_joined(const GradParams& p, uint32_t row, int64_t col, int n,
                                             const float (&acc)[4]) {
  if (n == 4) {
    write_sum<TW, 4>(p, row, col, col, acc);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e) {
      const float one[1] = {acc[e]};
      if (e < n) write_sum<TW, 1>(p, row, col + e, col + e, one);
    }
  }
}

template <typename TW>
__global__ __launch_bounds__(kJoinWaves* kWave) void grad_join_kernel(GradParams p, SumParams s, int64_t part_width,
                                                                      uint32_t tiles) {
  __shared__ float sums[kJoinWaves][4][kWave];
  __shared__ uint32_t lengths[kJoinWaves];
  const int wave = threadIdx.x / kWave, lane = lane_id();
  const uint32_t c0 = blockIdx.x / tiles * kJoinWaves, tile = blockIdx.x % tiles;
  const int64_t col = (static_cast<int64_t>(tile) * kWave + lane) * 4;
  const int n = static_cast<int>(std::min<int64_t>(4, p.width - col));  // below 1: no column
  // the number of chunks after c that the run at c's end reaches into, if it begins in c
  auto length_of = [&](uint32_t c) -> uint32_t {
    const uint64_t first = static_cast<uint64_t>(c) * s.chunk, end = first + s.chunk;
    if (end >= p.num_tokens) return 0;
    const uint32_t row = s.sorted[end].x;
    if (row >= p.num_rows || s.sorted[end - 1].x != row || (first > 0 && s.sorted[first - 1].x == row)) return 0;
    for (uint32_t count = 0;; count += kWave) {
      const uint64_t at = (static_cast<uint64_t>(c) + 1 + count + lane) * s.chunk;
      const uint64_t reached = __ballot(at < p.num_tokens && s.sorted[at].x == row);
      if (~reached != 0) return count + __ffsll(static_cast<unsigned long long>(~reached)) - 1;
    }
  };
  auto add = [&](uint32_t part, float (&acc)[4]) {
    Cols<F32, 4> x;
    x.load(reinterpret_cast<const uint32_t*>(s.parts + part * part_width + col));  // parts are whole tiles
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += x[e];
  };
  const uint32_t mine = c0 + wave < s.chunks ? length_of(c0 + wave) : 0;
  if (lane == 0) lengths[wave] = mine;
  if (mine > 0 && mine <= kJoinWaves && n > 0) {
    const uint32_t c = c0 + wave;
    float acc[4] = {};
    add(2 * c + 1, acc);
#pragma unroll 4
    for (uint32_t i = 1; i <= mine; ++i) add(2 * (c + i), acc);
    write_joined<TW>(p, s.sorted[(static_cast<uint64_t>(c) + 1) * s.chunk].x, col, n, acc);
  }
  __syncthreads();
  for (int w = 0; w < kJoinWaves; ++w) {
    const uint32_t length = lengths[w], c = c0 + w;
    if (length <= kJoinWaves) continue;
    float acc[4] = {};
    if (n > 0) {
#pragma unroll 4
      for (uint32_t i = wave; i <= length; i += kJoinWaves) add(i == 0 ? 2 * c + 1 : 2 * (c + i), acc);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave == 0) {
      for (int o = 1; o < kJoinWaves; ++o) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += sums[o][e][lane];
      }
      write_joined<TW>(p, s.sorted[(static_cast<uint64_t>(c) + 1) * s.chunk].x, col, n, acc);
    }
    __syncthreads();
  }
}

// How a call's tokens are sorted and summed.
struct GradPlan {
  int vec, passes;
  bool few, small, one;
  uint32_t col_tiles, tile, tiles, chunk, chunks;
  int64_t pairs, counts, present, parts, bytes;  // offsets into the workspace, and its size
};

GradPlan grad_plan(int64_t num_tokens, int64_t num_rows, int64_t width) {
  GradPlan g{};
  g.vec = width <= kWave ? 1 : width <= 2 * kWave ? 2 : width <= 4 * kWave ? 4 : 8;
  g.col_tiles = static_cast<uint32_t>((width + kWave * g.vec - 1) / (kWave * g.vec));
  g.few = num_tokens <= kFewTokens && num_tokens * num_tokens * g.col_tiles <= kFewReads;
  if (g.few) return g;
  int bits = 1;
  while (bits < 31 && (num_rows >> bits) != 0) ++bits;  // rows 0 .. num_rows, the last for none
  g.passes = (bits + kBits - 1) / kBits;
  g.small = num_tokens <= kSmallSort && g.passes > 1 && num_rows / kBins < kSmallGroups;
  g.one = !g.small && num_tokens <= kOneSort;
  const int64_t blocks = (num_tokens + kBlock - 1) / kBlock;
  g.tile = static_cast<uint32_t>((blocks + kMaxTiles - 1) / kMaxTiles * kBlock);
  g.tiles = static_cast<uint32_t>((num_tokens + g.tile - 1) / g.tile);
  int64_t chunk = kRowsAhead;  // 8192 waves, or as many as chunks of one load give
  while (num_tokens / chunk * g.col_tiles > 8192) chunk *= 2;
  g.chunk = static_cast<uint32_t>(chunk);
  g.chunks = static_cast<uint32_t>((num_tokens + chunk - 1) / chunk);
  auto take = [&](int64_t bytes) {
    const int64_t at = g.bytes;
    g.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  g.pairs = take((g.small || g.one ? 1 : 2) * num_tokens * 8);
  if (!g.small && !g.one) g.counts = take(static_cast<int64_t>(g.tiles) * kBins * 4);
  g.present = take(num_rows);
  g.parts = take(static_cast<int64_t>(g.chunks) * 2 * g.col_tiles * kWave * g.vec * 4);
  return g;
}

template <typename F>
void with_vec(int vec, F&& f) {
  switch (vec) {
    case 1: f(std::integral_constant<int, 1>{}); break;
    case 2: f(std::integral_constant<int, 2>{}); break;
    case 4: f(std::integral_constant<int, 4>{}); break;
    default: f(std::integral_constant<int, 8>{});
  }
}

int launch(const void* kernel, int64_t blocks, void** args, hipStream_t stream, int threads = kThreads) {
  const hipError_t err =
      hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(blocks)), dim3(threads), args, 0, stream);
  if (err != hipSuccess) return fail(TBE_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
  return TBE_OK;
}

bool fits(int64_t rows, int64_t width) { return width == 0 || rows <= (INT64_MAX >> 3) / width; }

}  // namespace
}  // namespace vocab
}  // namespace tbe

using namespace tbe;
using namespace tbe::vocab;

extern "C" int tbe_token_embedding(const TbeTokenEmbeddingArgs* a, void* hip_stream) {
  clear_error();
  if (!a) return fail(TBE_ERR_INVALID_ARG, "null args");
  if (!is_type(a->weight_dtype) || !is_type(a->output_dtype))
    return fail(TBE_ERR_INVALID_ARG, "weight and output must be float32, float16 or bfloat16 (types %d, %d)",
                a->weight_dtype, a->output_dtype);
  if (a->index_size != 4 && a->index_size != 8)
    return fail(TBE_ERR_INVALID_ARG, "token_ids must be int32 or int64 (%d bytes)", a->index_size);
  if (a->num_rows < 0 || a->width < 0 || a->num_tokens < 0 || a->weight_stride < a->width ||
      !fits(a->num_rows, a->weight_stride) || !fits(a->num_tokens, a->width))
    return fail(TBE_ERR_INVALID_ARG, "bad shape");
  if (a->num_tokens == 0 || a->width == 0) return TBE_OK;
  if ((!a->weight && a->num_rows > 0) || !a->token_ids || !a->output)
    return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  const int64_t elems = a->weight_dtype == TBE_TY_FP32 || a->output_dtype == TBE_TY_FP32 ? 4 : 8;
  const int64_t vecs = (a->width + elems - 1) / elems;
  if (vecs >= 1 << 30) return fail(TBE_ERR_UNSUPPORTED, "token_embedding rows too wide");
  LookupParams p{a->weight, a->token_ids,  a->output, a->weight_stride, a->num_rows,
                 a->width,  a->num_tokens, a->scale,  a->index_size,    FastDiv(static_cast<uint32_t>(vecs))};
  const bool once = a->num_tokens * a->width * (a->output_dtype == TBE_TY_FP32 ? 4 : 2) > kLookupCached;
  const int64_t per = kThreads * kLookupUnroll, groups = (a->num_tokens * vecs + per - 1) / per;
  int rc = TBE_OK;
  with_type(a->weight_dtype, [&](auto w) {
    with_type(a->output_dtype, [&](auto o) {
      const void* k = once ? reinterpret_cast<const void*>(lookup_kernel<decltype(w), decltype(o), true>)
                           : reinterpret_cast<const void*>(lookup_kernel<decltype(w), decltype(o), false>);
      for (int64_t first = 0; first < groups && rc == TBE_OK; first += kMaxBlocks) {
        void* args[] = {&p, &first};
        rc = launch(k, std::min(kMaxBlocks, groups - first), args, static_cast<hipStream_t>(hip_stream));
      }
    });
  });
  return rc;
}

extern "C" int64_t tbe_token_embedding_grad_workspace_bytes(int64_t num_tokens, int64_t num_rows, int64_t width) {
  if (num_tokens < 0 || num_tokens > INT32_MAX || num_rows < 0 || num_rows > INT32_MAX || width < 0 ||
      width > INT32_MAX || !fits(num_rows, width) || !fits(num_tokens, width))
    return -1;
  return num_rows == 0 || width == 0 ? 0 : grad_plan(num_tokens, num_rows, width).bytes;
}

extern "C" int tbe_token_embedding_grad(const TbeTokenEmbeddingGradArgs* a, void* hip_stream) {
  clear_error();
  if (!a) return fail(TBE_ERR_INVALID_ARG, "null args");
  if (!is_type(a->grad_dtype) || !is_type(a->weight_dtype))
    return fail(TBE_ERR_INVALID_ARG, "gradients must be float32, float16 or bfloat16 (types %d, %d)", a->grad_dtype,
                a->weight_dtype);
  if (a->index_size != 4 && a->index_size != 8)
    return fail(TBE_ERR_INVALID_ARG, "token_ids must be int32 or int64 (%d bytes)", a->index_size);
  const int64_t need = tbe_token_embedding_grad_workspace_bytes(a->num_tokens, a->num_rows, a->width);
  if (need < 0 || a->grad_stride < 0 || !fits(a->num_tokens, a->grad_stride))
    return fail(TBE_ERR_INVALID_ARG, "bad shape");
  if (a->num_rows == 0 || a->width == 0) return TBE_OK;
  if (!a->grad_weight || (a->num_tokens > 0 && (!a->grad_output || !a->token_ids)))
    return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  if (a->workspace_bytes < need || (need > 0 && (!a->workspace || reinterpret_cast<uintptr_t>(a->workspace) % 256 != 0)))
    return fail(TBE_ERR_INVALID_ARG, "a workspace of %lld bytes, 256-byte aligned, is needed",
                static_cast<long long>(need));
  const GradPlan g = grad_plan(a->num_tokens, a->num_rows, a->width);
  const int64_t row_bytes = a->width * (a->weight_dtype == TBE_TY_FP32 ? 4 : 2);
  GradParams p{};
  p.grad = a->grad_output;
  p.ids = a->token_ids;
  p.out = a->grad_weight;
  p.stride = a->grad_stride;
  p.padding = a->padding_idx;
  p.width = a->width;
  p.num_tokens = static_cast<uint32_t>(a->num_tokens);
  p.num_rows = static_cast<uint32_t>(a->num_rows);
  p.scale = a->scale;
  p.index_size = a->index_size;
  p.accumulate = a->accumulate;
  p.col_tiles = static_cast<int32_t>(g.col_tiles);
  p.row_vecs = FastDiv(static_cast<uint32_t>((row_bytes + 15) / 16));
  p.few_rows = static_cast<uint32_t>(std::min<int64_t>(kFewRows, std::max<int64_t>(1, kFewFill / row_bytes)));
  const int64_t vecs = a->num_rows * p.row_vecs.d;
  int64_t fills = 0;
  if (!a->accumulate) {
    p.fill_reps = 1;
    while ((fills = (vecs + kThreads * int64_t(p.fill_reps) - 1) / (kThreads * int64_t(p.fill_reps))) > kMaxBlocks / 2)
      p.fill_reps *= 2;
  }
  const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  int rc = TBE_OK;
  const int64_t units = g.few ? a->num_tokens * g.col_tiles
                              : (static_cast<int64_t>(g.chunks) * g.col_tiles + kThreads / kWave - 1) / (kThreads / kWave);
  const int64_t join_tiles = (a->width + 4 * kWave - 1) / (4 * kWave);
  const int64_t joins = (static_cast<int64_t>(g.chunks) + kJoinWaves - 1) / kJoinWaves * join_tiles;
  if (units + fills > kMaxBlocks || g.tiles + fills > kMaxBlocks || joins > kMaxBlocks / kJoinWaves)
    return fail(TBE_ERR_UNSUPPORTED, "token_embedding_grad shape too large for one launch");
  p.work_groups = static_cast<uint32_t>(units);
  p.fills = static_cast<uint32_t>(fills);
  if (g.few) {
    with_type(a->weight_dtype, [&](auto tw) {
      if (fills > 0 && (vecs * 16 >= kFewFillAll || a->num_tokens == 0)) {
        void* args[] = {&p};
        rc = launch(reinterpret_cast<const void*>(fill_kernel<decltype(tw)>), fills, args, stream);
        fills = 0;
      }
      p.fills = fills > 0 ? static_cast<uint32_t>((a->num_rows + p.few_rows - 1) / p.few_rows) : 0;
      if (rc != TBE_OK || a->num_tokens == 0) return;
      with_type(a->grad_dtype, [&](auto tg) {
        with_vec(g.vec, [&](auto v) {
          void* args[] = {&p};
          rc = launch(reinterpret_cast<const void*>(grad_few_kernel<decltype(tg), decltype(tw), decltype(v)::value>),
                      units + p.fills, args, stream);
        });
      });
    });
    return rc;
  }
  auto* ws = static_cast<uint8_t*>(a->workspace);
  uint2* pairs[2] = {reinterpret_cast<uint2*>(ws + g.pairs), reinterpret_cast<uint2*>(ws + g.pairs) + a->num_tokens};
  SortParams s{};
  const bool fill_all =
      (g.small || g.one) && !a->accumulate && (a->num_tokens * 4 <= a->num_rows || a->num_rows * row_bytes <= kFillBeside);
  s.present = a->accumulate || fill_all ? nullptr : ws + g.present;
  if (g.small || g.one) {
    s.out = pairs[0];
    // the last group's rows end with that of positions without one
    uint32_t sorters = g.one ? 1 : static_cast<uint32_t>(a->num_rows / kBins + 1);
    int32_t passes = g.passes;
    auto* zeros = static_cast<uint8_t*>(a->grad_weight);
    int64_t zero_bytes = a->num_rows * row_bytes;
    int64_t groups = 0;  // that fill
    if (fill_all) {
      groups = std::min<int64_t>(kMaxBlocks / 8, (zero_bytes + 16 * kSortThreads - 1) / (16 * kSortThreads));
      p.fills = 0;
    }
    void* by_one[] = {&p, &s, &passes, &zeros, &zero_bytes};
    void* by_rows[] = {&p, &s, &sorters, &zeros, &zero_bytes};
    rc = launch(g.one ? reinterpret_cast<const void*>(sort_one_kernel) : reinterpret_cast<const void*>(sort_small_kernel),
                sorters + groups, g.one ? by_one : by_rows, stream, kSortThreads);
  } else {
    s.counts = reinterpret_cast<uint32_t*>(ws + g.counts);
    s.tile = g.tile;
    s.tiles = g.tiles;
    for (int pass = 0; pass < g.passes && rc == TBE_OK; ++pass) {
      s.in = pairs[(pass + 1) & 1];
      s.out = pairs[pass & 1];
      s.shift = pass * kBits;
      int64_t zero_vecs = pass == 0 && s.present ? (a->num_rows + 15) / 16 : 0;
      void* count_args[] = {&p, &s, &zero_vecs};
      rc = launch(reinterpret_cast<const void*>(sort_count_kernel),
                  std::max<int64_t>(g.tiles, std::min<int64_t>(1024, zero_vecs / (4 * kThreads))), count_args, stream);
      if (rc != TBE_OK) break;
      // rows are marked in the first pass
      const bool fill = pass > 0 && pass + 1 == g.passes && p.fills > 0;
      with_type(a->weight_dtype, [&](auto tw) {
        void* args[] = {&p, &s};
        rc = launch(reinterpret_cast<const void*>(sort_pass_kernel<decltype(tw)>), g.tiles + (fill ? fills : 0), args,
                    stream);
      });
      if (fill) p.fills = 0;
    }
  }
  if (rc != TBE_OK) return rc;
  SumParams sum{s.out, ws + g.present, reinterpret_cast<float*>(ws + g.parts), g.chunk, g.chunks};
  with_type(a->grad_dtype, [&](auto tg) {
    with_type(a->weight_dtype, [&](auto tw) {
      with_vec(g.vec, [&](auto v) {
        void* args[] = {&p, &sum};
        rc = launch(reinterpret_cast<const void*>(grad_sum_kernel<decltype(tg), decltype(tw), decltype(v)::value>),
                    units + p.fills, args, stream);
      });
      if (rc != TBE_OK) return;
      int64_t part_width = static_cast<int64_t>(g.col_tiles) * kWave * g.vec;
      uint32_t tiles = static_cast<uint32_t>(join_tiles);
      void* args[] = {&p, &sum, &part_width, &tiles};
      rc = launch(reinterpret_cast<const void*>(grad_join_kernel<decltype(tw)>), joins, args, stream, kJoinWaves * kWave);
    });
  });
  return rc;
}
