// vocab_logits.hip — gfx950 kernels and C ABI of the operators over rows of logits
// (include/tbe_vocab_ops.h): log probabilities of given tokens with entropy and the top
// alternatives, the loss against a teacher's top logits, and their gradients.
//
// With m = max x, e_j = exp((x_j - m) / T), s = sum e:
//   log p_j = (x_j - m) / T - log s        H = log s - sum e_j (x_j - m) / (T s)
// A forward pass reads every logit once, a gradient reads and writes each once; about ten
// operations per logit.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "tbe_internal.h"
#include "tbe_nbit.h"
#include "tbe_vocab_ops.h"
#include "vocab_device.h"

namespace tbe {
namespace vocab {
namespace {

constexpr int kThreads = 256;                    // of a work-group, where nothing else is said
constexpr int kUnroll = 4;                       // 16-byte vectors a thread has in flight
constexpr int kListed = TBE_VOCAB_MAX_LISTED;
constexpr int kMaxParts = 64;                    // of one row
constexpr int64_t kMaxThreads = 0xFFFFFFFFLL;     // a launch holds fewer than 2^32
constexpr float kLn2 = 0.693147180559945309f;

static_assert(kListed <= kThreads, "one thread per listed token");

// A row from its first 16-byte boundary: nvec vectors, and the elements before and after them.
template <typename T>
struct Row {
  const typename T::raw* p;
  int32_t vocab, head, nvec, extra;
  __device__ Row(const void* logits, int64_t stride, int64_t row, int32_t v) {
    p = static_cast<const typename T::raw*>(logits) + row * stride;
    vocab = v;
    const uint32_t past = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
    head = std::min<int32_t>(v, ((16 - past) & 15) / sizeof(typename T::raw));
    nvec = (v - head) / kElems<T>;
    extra = v - nvec * kElems<T>;
  }
  // the first vector of a part of the row
  __device__ int32_t begin(int32_t part, int32_t parts) const {
    return static_cast<int32_t>(static_cast<int64_t>(nvec) * part / parts);
  }
  __device__ int32_t index(int32_t vec) const { return head + vec * kElems<T>; }
  // the i-th element outside the vectors
  __device__ int32_t extra_index(int32_t i) const { return i < head ? i : vocab - extra + i; }
};

// y(x) = log2(e) (x - m) / T for a reference m >= x (not -inf).
// Near 0, one fused multiply-add per logit: with c = log2(e) / T and M = m c rounded, fma(x, c, -M)
// is (x - m) c but for its own last rounding and that of M, which is the same for every x and taken
// out of sums by `rest`, at most 1/8.  From |m| c = 2^22 on (rows masked by a finite value, very low
// temperatures) M's rounding would reach whole powers of two: there x - m is taken first, exact
// for the x near m that count, and nothing is left to take out.
struct Scale {
  float c, off, M, rest;  // 2^y is exp((x - m) / T) 2^rest
  __device__ Scale(float m, float factor) : c(factor) {
    const bool far = !(fabsf(m) * factor < 4194304.f);
    off = far ? m : 0.f;
    M = far ? 0.f : m * factor;
    rest = far ? 0.f : fmaf(m, factor, -M);
  }
  __device__ float operator()(float x) const { return past_off(x - off); }
  __device__ float past_off(float x) const { return fmaf(x, c, -M); }  // of x - off
  // Calls f with a function from logits to their y: without the offset where it is 0, as almost always.
  template <typename F>
  __device__ __forceinline__ void with(F f) const {
    if (off == 0.f) {
      f([*this](float x) { return past_off(x); });
    } else {
      f([*this](float x) { return (*this)(x); });
    }
  }
};

// Maximum m, s = sum exp((x - m) / T) and t = sum exp((x - m) / T) y, y = log2(e) (x - m) / T, over the
// logits so far, in 32 bits.  A NaN among the x leaves m alone and makes s NaN; x of -inf adds nothing.
struct Stats {
  float m, s, t;

  __device__ static Stats none() { return {-INFINITY, 0.f, 0.f}; }
  // Moves the maximum to nm > m, by which y falls by delta.
  __device__ void raise(float nm, float delta) {
    const float r = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(-delta);
    t = r == 0.f ? 0.f : r * (t - delta * s);
    s *= r;  // 0 * NaN stays NaN
    m = nm;
  }
  // Over a wave, or the first N lanes of every N; every lane gets the same bits.
  template <int N>
  __device__ void join_lanes(float c) {
    const float most = lanes_max<N>(m);
    if (most > m) raise(most, (most - m) * c);
    s = lanes_sum<N>(s);
    t = lanes_sum<N>(t);
  }
  __device__ bool empty() const { return m == -INFINITY && s == 0.f; }  // no token is possible
  __device__ float log_s() const { return empty() ? 0.f : __builtin_amdgcn_logf(s) * kLn2; }
  __device__ float entropy() const { return empty() ? 0.f : (__builtin_amdgcn_logf(s) - t / s) * kLn2; }
};

// Statistics of the logits that one thread meets, on the scale of their maximum until settle().  The
// maximum moves seldom after the first vectors: a wave looks whether any lane's does.
struct Running : Stats {
  float factor;
  Scale scale;
  bool far = false;  // whether a lane of the wave has a scale with an offset
  __device__ explicit Running(float c) : Stats(Stats::none()), factor(c), scale(0.f, c) {}  // 2^y of -inf is 0
  template <int N, bool kEnt>
  __device__ __forceinline__ void absorb(float (&x)[N], float top) {
    if (__ballot(top > m) != 0) {
      if (top > m) {
        const Scale to(top, factor);
        raise(top, fmaf(to.off - scale.off, factor, to.M - scale.M));  // from scale to scale, rests and all
        scale = to;
      }
      far = __ballot(scale.off != 0.f) != 0;
    }
    if (far) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] -= scale.off;
    }
    // Summed apart first: small terms one by one into a sum that has met the maximum lose more (rows
    // of 200000 fp32, temperature 0.7: gradients 8.7e-7 off those in 64 bits, so 1.2e-7; no slower).
    float near_s = 0.f, near_t = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float y = scale.past_off(x[i]);
      const float e = __builtin_amdgcn_exp2f(y);
      near_s += e;
      if constexpr (kEnt) near_t = fmaf(e, fmaxf(y, -FLT_MAX), near_t);  // -inf adds 0, not 0 * inf
    }
    s += near_s;
    if constexpr (kEnt) t += near_t;
  }
  // Takes the scale's rest out, after the last logit.
  __device__ __forceinline__ void settle() {
    if (m == -INFINITY) return;
    const float rest = Scale(m, factor).rest, r = __builtin_amdgcn_exp2f(-rest);
    t = r * (t - rest * s);
    s *= r;
  }
};

// ---------------------------------------------------------------- top k

// Logits as whole numbers of the same order: NaN last, -0 and +0 equal.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x != x ? 0xFFFFFFFFu : u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
// The order just below o; that of -0 is no logit's, and -0 compares equal to +0.
__device__ __forceinline__ uint32_t below(uint32_t o) { return o == 0x80000000u ? o - 2 : o - 1; }
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == 0xFFFFFFFFu ? NAN : __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}

template <int J, typename V>
__device__ __forceinline__ void exchange(V& v, bool keep_max) {
  const V o = lane_xor<J>(v);
  v = (v > o) == keep_max ? v : o;
}
// Sorts a sequence that rises and then falls (or the reverse) into blocks of 2J lanes; up: rising.
template <int J, typename V>
__device__ __forceinline__ void bitonic(V& v, bool up) {
  exchange<J>(v, ((threadIdx.x & J) != 0) == up);
  if constexpr (J > 1) bitonic<J / 2>(v, up);
}
template <typename V>
__device__ __forceinline__ void sort_rising(V& v) {
  const int l = lane_id();
  bitonic<1>(v, (l & 2) == 0);
  bitonic<2>(v, (l & 4) == 0);
  bitonic<4>(v, (l & 8) == 0);
  bitonic<8>(v, (l & 16) == 0);
  bitonic<16>(v, (l & 32) == 0);
  bitonic<32>(v, true);
}
// The 64 largest of a falling list and a rising one, falling.
__device__ __forceinline__ uint64_t merge_lists(uint64_t falling, uint64_t rising) {
  uint64_t v = falling > rising ? falling : rising;
  bitonic<32>(v, false);
  return v;
}

constexpr int kTopBuffer = kWave * 8 + kWave;  // a vector of every lane, and what was left before

// The 64 largest (logit, lowest index) keys a wave has seen, one per lane, falling.  Logits
// above the k-th are gathered in LDS, 64 are made keys, sorted and merged at a time.
// A logit is left out when it is <= eff.  A wave meets its logits in rising order of index
// from one step (of all its lanes' vectors) to the next, so between steps one equal to the
// k-th can be left out; inside a step, and against the other waves' k-th, it cannot.
struct TopK {
  uint64_t list = 0;  // 0: no logit
  float eff = NAN;    // no logit is <= NaN
  uint2* buf;         // LDS: kTopBuffer logits and their indices, of this wave
  uint32_t* counter;  // LDS: how many
  uint32_t* kth;      // LDS: the greatest k-th of the work-group's waves
  uint32_t* shares;   // LDS: a bound from every wave
  int k, waves;

  __device__ static float bound(uint32_t o) { return o == 0 ? NAN : o >= 0xFF800000u ? INFINITY : value_of(o); }
  __device__ uint32_t own() const {
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(list >> 32), k - 1));
  }
  __device__ void limit(bool strict) {
    uint32_t o = own();
    if (o != 0 && !strict) o = below(o);
    const uint32_t other = std::max(__hip_atomic_load(kth, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP),
                                    lanes_min(__hip_atomic_load(&shares[lane_id() & (waves - 1)], __ATOMIC_RELAXED,
                                                                __HIP_MEMORY_SCOPE_WORKGROUP)));
    // a k-th of -inf elsewhere says nothing: -inf of a lower index may still come
    eff = bound(std::max(o, other >= 0x00800000u ? below(other) : 0u));
  }
  __device__ static uint32_t lanes_min(uint32_t v) {
    v = std::min(v, lane_xor<1>(v));
    v = std::min(v, lane_xor<2>(v));
    v = std::min(v, lane_xor<4>(v));
    return std::min(v, lane_xor<8>(v));
  }
  // Bounds from the maxima that the lanes have met so far (each a logit of its own): the k-th of
  // this wave's is not above the row's k-th, nor is, where every wave's share of the k
  // greatest is its ceil(k / waves), the least of the waves' last ones.
  __device__ void refresh(float best) {
    uint32_t o = order_of(best);
    sort_rising(o);
    const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(o), kWave - k));
    const int share = (k + waves - 1) / waves;
    const uint32_t part = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(o), kWave - share));
    if (lane_id() == 0) {
      atomicMax(kth, at);
      __hip_atomic_store(&shares[threadIdx.x / kWave], part, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    wave_fence();
  }
  // Keys [from, to) of the buffer, at most 64, into the list.
  __device__ void merge(int from, int to) {
    uint64_t v = 0;
    if (from + lane_id() < to) {
      const uint2 found = buf[from + lane_id()];
      v = static_cast<uint64_t>(order_of(__uint_as_float(found.x))) << 32 | (0xFFFFFFFFu - found.y);
    }
    sort_rising(v);
    list = merge_lists(list, v);
    if (lane_id() == 0) atomicMax(kth, own());
    wave_fence();
  }
  // This lane's logit x at idx; the lanes of a wave call it apart.  At most 8 times, then settle().
  __device__ void add(float x, uint32_t idx) {
    if (x <= eff) return;
    buf[atomicAdd(counter, 1u)] = uint2{__float_as_uint(x), idx};
  }
  __device__ void settle(int most) {
    wave_fence();
    int count = __builtin_amdgcn_readfirstlane(static_cast<int>(*counter));
    if (count < most) return;
    do {
      const int from = std::max(0, count - kWave);
      merge(from, count);
      count = from;
    } while (count >= most);
    if (lane_id() == 0) *counter = count;
    wave_fence();
    limit(false);
  }
};

// ---------------------------------------------------------------- one pass over a row

template <int N>
__device__ __forceinline__ float max_of(const float* x) {
  float top = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
  return top;
}

// Keeps the compiler from holding a vector's unpacked elements in registers from one use to the next.
__device__ __forceinline__ void reread(Vec16& v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(v.w[i]));
}

// Vectors [v0, v1) of the row, and the elements outside the vectors if `ends`.
template <int kSize, typename T, bool kEnt, bool kTop>
__device__ __forceinline__ void row_pass(const Row<T>& row, int32_t v0, int32_t v1, bool ends, Running& st,
                                         TopK& top) {
  constexpr int E = kElems<T>, kGroup = kTop ? 2 : 4;  // vectors summed at a time
  int step = 0;
  for (int32_t b = v0; b < v1; b += kSize * kUnroll) {
    Vec16 w[kUnroll];
    const int32_t i0 = b + static_cast<int32_t>(threadIdx.x);
    if (b + kSize * kUnroll <= v1) {  // all but the last step
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) w[u] = load16(row.p + row.index(i0) + u * (kSize * E));
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int32_t i = i0 + u * kSize;
        w[u] = i < v1 ? load16(row.p + row.index(i)) : Vec16{{T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf}};
      }
    }
    float best[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u += kGroup) {
      float x[kGroup * E], most = -INFINITY;
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        unpack<T>(w[u + g], x + g * E);
        best[u + g] = max_of<E>(x + g * E);
        most = g == 0 ? best[u] : fmaxf(most, best[u + g]);
      }
      st.absorb<kGroup * E, kEnt>(x, most);
    }
    if constexpr (kTop) {
      const float most = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
      if (step == 0) {
        top.refresh(st.m);
        __syncthreads();  // every wave has its first bound
      } else if ((step & (step - 1)) == 0 && (step & 0xAAAAAAAAu) != 0) {  // steps 2, 8, 32, ...
        top.refresh(st.m);
      }
      ++step;
      // the maxima leave NaN out, the sum does not
      if (__ballot(st.s != st.s || !(most <= top.eff)) != 0) {
        top.limit(true);  // the bounds may have risen
        const bool nan = st.s != st.s;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          if (i0 + u * kSize < v1 && (nan || !(best[u] <= top.eff))) {  // few lanes, one candidate each
            float x[E];
            reread(w[u]);
            unpack<T>(w[u], x);
            const uint32_t at = row.index(i0 + u * kSize);
#pragma unroll
            for (int e = 0; e < E; ++e) top.add(x[e], at + e);
          }
          top.settle(kWave);
        }
      }
    }
  }
  if (ends && threadIdx.x < kWave) {  // at most 14 elements, by the first wave, out of order
    const bool in = static_cast<int32_t>(threadIdx.x) < row.extra;
    const int32_t i = in ? row.extra_index(threadIdx.x) : 0;
    const float logit = in ? to_f32<T>(row.p[i]) : -INFINITY;
    float x[1] = {logit};
    st.absorb<1, kEnt>(x, logit);
    if constexpr (kTop) {
      top.limit(false);
      if (in) top.add(logit, i);
    }
  }
  if constexpr (kTop) top.settle(1);
  st.settle();
}

template <int kSize>
struct GroupShared {
  static constexpr int kWaves = kSize / kWave;
  Stats stats[kWaves];
  float sums[2][kWaves];
};
template <int kSize>
struct TopShared {
  static constexpr int kWaves = kSize / kWave;
  union {
    uint2 buf[kWaves][kTopBuffer];
    uint64_t lists[kWaves][kWave];  // once no wave gathers any more
  };
  uint32_t counters[kWaves];
  uint32_t kth, shares[kWaves];
  __device__ void begin(TopK& top, int k) {
    top.buf = buf[threadIdx.x / kWave];
    top.counter = &counters[threadIdx.x / kWave];
    top.kth = &kth;
    top.shares = shares;
    top.k = k;
    top.waves = kWaves;
    if (lane_id() == 0) *top.counter = shares[threadIdx.x / kWave] = 0;
    if (threadIdx.x == 0) kth = 0;
    __syncthreads();
  }
  // Joins the waves' lists into the first wave's.  After a barrier.
  __device__ void join(TopK& top) {
    const int w = threadIdx.x / kWave;
    for (int step = 1; step < kWaves; step *= 2) {
      if ((w & (2 * step - 1)) == step) lists[w][lane_id()] = top.list;
      __syncthreads();
      if ((w & (2 * step - 1)) == 0) top.list = merge_lists(top.list, lists[w + step][kWave - 1 - lane_id()]);
    }
  }
};

// Joins the waves' statistics; every thread gets the result.
template <int kSize>
__device__ __forceinline__ void join_group(Stats& st, float c, GroupShared<kSize>& sh) {
  constexpr int kWaves = GroupShared<kSize>::kWaves;
  st.join_lanes<kWave>(c);
  if (lane_id() == 0) sh.stats[threadIdx.x / kWave] = st;
  __syncthreads();
  st = sh.stats[threadIdx.x % kWaves];
  st.join_lanes<kWaves>(c);
}

// Sums of two values over the work-group.
template <int kSize>
__device__ __forceinline__ void group_sum(float& a, float& b, GroupShared<kSize>& sh) {
  constexpr int kWaves = GroupShared<kSize>::kWaves;
  a = lanes_sum<kWave>(a);
  b = lanes_sum<kWave>(b);
  __syncthreads();
  if (lane_id() == 0) {
    sh.sums[0][threadIdx.x / kWave] = a;
    sh.sums[1][threadIdx.x / kWave] = b;
  }
  __syncthreads();
  a = lanes_sum<kWaves>(sh.sums[0][threadIdx.x % kWaves]);
  b = lanes_sum<kWaves>(sh.sums[1][threadIdx.x % kWaves]);
}
template <int kSize>
__device__ __forceinline__ float group_sum(float a, GroupShared<kSize>& sh) {
  float none = 0.f;
  group_sum(a, none, sh);
  return a;
}
template <int kSize>
__device__ __forceinline__ float group_max(float v, GroupShared<kSize>& sh) {
  constexpr int kWaves = GroupShared<kSize>::kWaves;
  v = lanes_max<kWave>(v);
  __syncthreads();
  if (lane_id() == 0) sh.sums[0][threadIdx.x / kWave] = v;
  __syncthreads();
  return lanes_max<kWaves>(sh.sums[0][threadIdx.x % kWaves]);
}

// Where a work-group's part of a row is written when a row has several.
struct Parts {
  float4* stats;    // [rows][parts]
  uint64_t* lists;  // [rows][parts][kWave]
  int32_t parts;
};

__device__ __forceinline__ int64_t load_id(const void* ids, int32_t index_size, int64_t i) {
  return index_size == 8 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
}

// ---------------------------------------------------------------- log probabilities

struct LogprobsParams {
  const void* __restrict__ logits;
  const void* __restrict__ tokens;
  float* __restrict__ logprobs;
  float* __restrict__ entropy;
  float* __restrict__ top_logprobs;
  int64_t* __restrict__ top_tokens;
  float* __restrict__ stats;
  int64_t stride;
  int32_t vocab, given, index_size, top_k;
  float t, c;  // T, log2(e) / T
};

// A thread's given token: whether there is one, whether it is of the vocabulary, its logit.
// Read before the pass over the row, whose end would wait for it.
struct Given {
  bool some, ok;
  float x;
};

template <typename T>
__device__ __forceinline__ Given load_given(const LogprobsParams& p, const Row<T>& row, int64_t i) {
  Given g{static_cast<int32_t>(threadIdx.x) < p.given, false, 0.f};
  if (g.some) {
    const int64_t id = load_id(p.tokens, p.index_size, i * p.given + threadIdx.x);
    g.ok = id >= 0 && id < p.vocab;
    if (g.ok) g.x = to_f32<T>(row.p[id]);
  }
  return g;
}

// What follows from the whole row's statistics and list.
__device__ __forceinline__ void finish_row(const LogprobsParams& p, const Given& given, int64_t i, const Stats& st,
                                           uint64_t list) {
  const bool empty = st.empty();
  const float log_s = st.log_s();
  if (threadIdx.x == 0) {
    p.entropy[i] = st.entropy();
    p.stats[2 * i] = st.m;
    p.stats[2 * i + 1] = st.s;
  }
  if (given.some) {
    const float lp = empty ? -INFINITY : (given.x - st.m) / p.t - log_s;
    p.logprobs[i * p.given + threadIdx.x] = given.ok ? lp : 0.f;
  }
  if (static_cast<int32_t>(threadIdx.x) < p.top_k) {  // the first wave's list
    const float x = value_of(static_cast<uint32_t>(list >> 32));
    p.top_tokens[i * p.top_k + threadIdx.x] = 0xFFFFFFFFu - static_cast<uint32_t>(list);
    p.top_logprobs[i * p.top_k + threadIdx.x] = empty ? -INFINITY : (x - st.m) / p.t - log_s;
  }
}

// A work-group per row, or per part of a row (then logprobs_join_kernel finishes the row).  One pass
// over the logits, bound by HBM without a top list (2048 rows of 131072 bf16 95 us, 5.6 TB/s) and by
// its instructions with one (top 20 117 us, top 64 128 us).
template <int kSize, typename T, bool kTop>
__global__ __launch_bounds__(kSize) void logprobs_kernel(LogprobsParams p, Parts parts, int64_t first) {
  __shared__ GroupShared<kSize> sh;
  __shared__ TopShared<kTop ? kSize : kWave> lists;
  const int32_t part = blockIdx.x % parts.parts;
  const int64_t i = first + blockIdx.x / parts.parts;
  const Row<T> row(p.logits, p.stride, i, p.vocab);
  Given given{};
  if (parts.parts == 1) given = load_given(p, row, i);
  Running st(p.c);
  TopK top;
  if constexpr (kTop) lists.begin(top, p.top_k);
  row_pass<kSize, T, true, kTop>(row, row.begin(part, parts.parts), row.begin(part + 1, parts.parts),
                                 part + 1 == parts.parts, st, top);
  join_group(st, p.c, sh);
  if constexpr (kTop) lists.join(top);
  if (parts.parts == 1) {
    finish_row(p, given, i, st, top.list);
    return;
  }
  const int64_t at = i * parts.parts + part;
  if (threadIdx.x == 0) parts.stats[at] = float4{st.m, st.s, st.t, 0.f};
  if constexpr (kTop) {
    if (threadIdx.x < kWave) parts.lists[at * kWave + threadIdx.x] = top.list;
  }
}

// The parts' statistics, joined in an order of their own; every thread gets the result.
template <int kSize>
__device__ __forceinline__ Stats join_parts(const Parts& parts, int64_t i, float c, GroupShared<kSize>& sh) {
  static_assert(kMaxParts <= kSize, "a thread per part");
  Stats st = Stats::none();
  if (static_cast<int32_t>(threadIdx.x) < parts.parts) {
    const float4 v = parts.stats[i * parts.parts + threadIdx.x];
    st.m = v.x;
    st.s = v.y;
    st.t = v.z;
  }
  join_group(st, c, sh);
  return st;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_join_kernel(LogprobsParams p, Parts parts, int64_t first) {
  __shared__ GroupShared<kThreads> sh;
  __shared__ TopShared<kThreads> lists;
  const int64_t i = first + blockIdx.x;
  const Given given = load_given(p, Row<T>(p.logits, p.stride, i, p.vocab), i);
  TopK top;
  if (p.top_k > 0) {
    for (int32_t q = threadIdx.x / kWave; q < parts.parts; q += kThreads / kWave)
      top.list = merge_lists(top.list, parts.lists[(i * parts.parts + q) * kWave + kWave - 1 - lane_id()]);
  }
  const Stats st = join_parts(parts, i, p.c, sh);
  if (p.top_k > 0) lists.join(top);
  finish_row(p, given, i, st, top.list);
}

// ---------------------------------------------------------------- gradients

// What a part of a row writes: vectors [v0, v1), which hold tokens of [from, to), and, the last
// part, the elements outside the vectors.
template <typename T>
struct Range {
  int32_t v0, v1, from, to;
  bool ends;
  __device__ Range(const Row<T>& row, int32_t part, int32_t parts)
      : v0(row.begin(part, parts)), v1(row.begin(part + 1, parts)), ends(part + 1 == parts) {
    from = row.index(v0);
    to = row.index(v1);
  }
  __device__ bool holds(const Row<T>& row, int32_t id) const {
    return (id >= from && id < to) || (ends && (id < row.head || id >= row.index(row.nvec)));
  }
};

// Writes f(x) of every logit of the range.
template <int kSize, typename T, typename F>
__device__ __forceinline__ void map_row(const Row<T>& row, typename T::raw* out, const Range<T>& range, F f) {
  constexpr int E = kElems<T>;
  // last first: the end of the row is what was read last
  constexpr int kStep = kSize * kUnroll;
  for (int32_t b = range.v0 + (range.v1 - range.v0 + kStep - 1) / kStep * kStep - kStep; b >= range.v0; b -= kStep) {
    Vec16 w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t i = b + u * kSize + static_cast<int32_t>(threadIdx.x);
      w[u] = i < range.v1 ? load16_once(row.p + row.index(i)) : Vec16{};
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int32_t i = b + u * kSize + static_cast<int32_t>(threadIdx.x);
      float x[E];
      unpack<T>(w[u], x);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = f(x[e]);
      if (i < range.v1) store16_once(out + row.index(i), pack<T>(x));
    }
  }
  if (range.ends && static_cast<int32_t>(threadIdx.x) < row.extra) {
    const int32_t i = row.extra_index(threadIdx.x);
    out[i] = from_f32<T>(f(to_f32<T>(row.p[i])));
  }
}

// Writes f(y) of every logit of the range.
template <int kSize, typename T, typename F>
__device__ __forceinline__ void map_logits(const Row<T>& row, typename T::raw* out, const Range<T>& range,
                                           const Scale& scale, F f) {
  scale.with([&](auto y) { map_row<kSize>(row, out, range, [&](float x) { return f(y(x)); }); });
}

template <int kSize, typename T>
__device__ __forceinline__ void zero_row(const Row<T>& row, typename T::raw* out, const Range<T>& range) {
  for (int32_t i = range.v0 + threadIdx.x; i < range.v1; i += kSize) store16_once(out + row.index(i), Vec16{});
  if (range.ends && static_cast<int32_t>(threadIdx.x) < row.extra) out[row.extra_index(threadIdx.x)] = 0;
}

// Tokens of a row whose gradient has a term of its own: out = f(y) + the sum of the token's terms,
// in the order of the list.  Written after map_logits by the wave that wrote the token's vector,
// past a fence of that wave, so that the term is what stays.
struct Terms {
  int32_t ids[kListed];  // -1: none, or an earlier entry has it
  float sums[kListed], xs[kListed];

  // Threads 0 .. n - 1 hold one entry each (-1: none): token, term and logit.  Before a barrier of
  // the caller's.  A list of one wave's length is that wave's own matter.
  __device__ void set(int32_t id, float term, float x, int32_t n) {
    constexpr int32_t kAtOnce = 16;
    const int32_t at = static_cast<int32_t>(threadIdx.x), padded = (n + kAtOnce - 1) / kAtOnce * kAtOnce;
    auto written = [n] {
      if (n <= kWave) {
        wave_fence();
      } else {
        __syncthreads();
      }
    };
    if (at < padded) {
      ids[at] = at < n ? id : -1;
      sums[at] = term;
    }
    written();
    bool mine = at < n && id >= 0;
    float sum = term;
    if (mine) {
      int32_t same = 0, before = 0;
      for (int32_t k0 = 0; k0 < n; k0 += kAtOnce) {
#pragma unroll
        for (int32_t j = 0; j < kAtOnce; ++j) {
          const int32_t hit = ids[k0 + j] == id;
          same += hit;
          before += hit & (k0 + j < at);
        }
      }
      if (same > 1) {  // the token is listed more than once: the first entry sums them
        mine = before == 0;
        sum = 0.f;
        for (int32_t k = at; k < n; ++k) sum += ids[k] == id ? sums[k] : 0.f;
      }
    }
    written();
    if (at < n) {
      ids[at] = mine ? id : -1;
      sums[at] = sum;
      xs[at] = x;
    }
  }
  // `origin`: the vector that thread 0 wrote first.
  template <int kSize, typename T, typename F>
  __device__ void write(const Row<T>& row, typename T::raw* out, const Range<T>& range, int32_t origin, int32_t n,
                        const Scale& scale, F f) const {
    wave_fence();
    for (int32_t k = lane_id(); k < n; k += kWave) {
      const int32_t id = ids[k];
      if (id < 0 || !range.holds(row, id)) continue;
      const uint32_t vec = static_cast<uint32_t>(id - row.head) / kElems<T>;
      const bool outside = id < row.head || vec >= static_cast<uint32_t>(row.nvec);  // the first wave's
      const uint32_t wave = outside ? 0 : (vec - origin) % kSize / kWave;
      if (wave == threadIdx.x / kWave) out[id] = from_f32<T>(f(scale(xs[k])) + sums[k]);
    }
  }
};

// What 2^y is multiplied by to give `by` times the probability, s = sum exp((x - m) / T).  The
// forward pass leaves s and not its logarithm, whose last bit is 2^-21 of a probability.
__device__ __forceinline__ float grad_factor(float by, const Scale& scale, float s) {
  return by / s * __builtin_amdgcn_exp2f(-scale.rest);
}

struct LogprobsGradParams {
  const void* __restrict__ logits;
  const void* __restrict__ tokens;
  const float* __restrict__ grad_logprobs;
  const float* __restrict__ grad_entropy;
  const float* __restrict__ entropy;
  const float* __restrict__ stats;
  void* __restrict__ out;
  int64_t stride;
  int32_t vocab, given, index_size;
  float inv_t, c;
};

// Reads and writes every logit once, at the rate of a copy (4096 rows of 65536 bf16 222 us, 4.8 TB/s;
// after the forward pass 188).  The last rows come first: they are what a forward pass shortly before
// read last, and what the memory-side cache still holds (both passes 317 -> 286 us).
template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_grad_kernel(LogprobsGradParams p, int32_t parts, int64_t first) {
  const uint32_t group = gridDim.x - 1 - blockIdx.x;
  __shared__ GroupShared<kThreads> sh;
  __shared__ Terms terms;
  const int64_t i = first + group / parts;
  const Row<T> row(p.logits, p.stride, i, p.vocab);
  const Range<T> range(row, group % parts, parts);
  auto* out = static_cast<typename T::raw*>(p.out) + i * p.vocab;
  const float m = p.stats[2 * i], s = p.stats[2 * i + 1];
  if (m == -INFINITY && s == 0.f) {  // no token is possible
    zero_row<kThreads>(row, out, range);
    return;
  }
  int32_t id = -1;
  float g = 0.f, x = 0.f;
  if (p.grad_logprobs && static_cast<int32_t>(threadIdx.x) < p.given) {
    const int64_t t = load_id(p.tokens, p.index_size, i * p.given + threadIdx.x);
    if (t >= 0 && t < p.vocab) {
      id = static_cast<int32_t>(t);
      g = p.grad_logprobs[i * p.given + threadIdx.x] * p.inv_t;
      x = to_f32<T>(row.p[t]);
    }
  }
  terms.set(id, g, x, p.given);
  const float gh = p.grad_entropy ? p.grad_entropy[i] * p.inv_t : 0.f;
  const float base = group_sum(g, sh) + (gh != 0.f ? gh * p.entropy[i] : 0.f);
  // -p (gh log p + base), p = 2^y k, log p = (y + log2 k) ln 2
  const Scale scale(m, p.c);
  const float log2_k = -__builtin_amdgcn_logf(s) - scale.rest, k = grad_factor(-1.f, scale, s);
  const float by_y = k * gh * kLn2, by_1 = k * fmaf(gh * kLn2, log2_k, base);
  auto f = [&](float y) {
    return __builtin_amdgcn_exp2f(y) * fmaf(by_y, fmaxf(y, -1000.f), by_1);  // 2^-1000 is 0
  };
  map_logits<kThreads>(row, out, range, scale, f);
  terms.write<kThreads>(row, out, range, range.v0, p.given, scale, f);
}

// ---------------------------------------------------------------- distillation

struct DistillParams {
  const void* __restrict__ logits;
  const void* __restrict__ tokens;
  const void* __restrict__ values;
  const float* __restrict__ weights;
  float* __restrict__ loss;
  float* __restrict__ stats;
  void* __restrict__ out;
  int64_t stride;
  int32_t vocab, top, index_size, teacher_dtype, renormalize;
  float t, inv_t, c;
};

// Thread k's entry of the teacher's list: its token (-1: none), q and log q.
struct Entry {
  int32_t id = -1;
  float q = 0.f, log_q = -INFINITY, x = 0.f;
};

// What a thread reads of the list.
struct RawEntry {
  int32_t id = -1;
  float value = -INFINITY, x = 0.f;  // the teacher's, the student's logit
};

template <typename T>
__device__ __forceinline__ RawEntry load_entry(const DistillParams& p, const Row<T>& row, int64_t i) {
  RawEntry r;
  if (static_cast<int32_t>(threadIdx.x) < p.top) {
    const int64_t at = i * p.top + threadIdx.x;
    const int64_t id = load_id(p.tokens, p.index_size, at);
    const float y = p.teacher_dtype == TBE_TY_FP32   ? to_f32<F32>(static_cast<const uint32_t*>(p.values)[at])
                    : p.teacher_dtype == TBE_TY_FP16 ? to_f32<F16>(static_cast<const uint16_t*>(p.values)[at])
                                                     : to_f32<BF16>(static_cast<const uint16_t*>(p.values)[at]);
    if (id >= 0 && id < p.vocab) {
      r.id = static_cast<int32_t>(id);
      r.value = y;
      r.x = to_f32<T>(row.p[id]);
    }
  }
  return r;
}

template <int kSize>
__device__ __forceinline__ Entry teacher_entry(const DistillParams& p, const RawEntry& raw, GroupShared<kSize>& sh) {
  Entry r;
  r.id = raw.id;
  r.x = raw.x;
  const float y = raw.value;
  if (p.renormalize) {
    const bool one_wave = p.top <= kWave;  // then the others' entries are none
    const float top = one_wave ? lanes_max<kWave>(y) : group_max(y, sh);
    const float d = y == -INFINITY ? -INFINITY : (y - top) * p.inv_t;
    const float e = expf(d);
    const float total = one_wave ? lanes_sum<kWave>(e) : group_sum(e, sh);
    if (total != 0.f) {
      r.q = e / total;
      r.log_q = d - logf(total);
    }
  } else {
    r.q = expf(y);
    r.log_q = y;
  }
  return r;
}

__device__ __forceinline__ float row_weight(const DistillParams& p, int64_t i) {
  return p.weights ? p.weights[i] : 1.f;
}

// A thread's term of T sum q (log q - log p): log p, a difference of logits by T, may leave the range
// where T log p does not (listed tokens that a low value masks, low temperatures).
__device__ __forceinline__ float loss_term(const Entry& t, const Stats& st, float log_s, float temperature) {
  if (t.id < 0 || t.q == 0.f) return 0.f;
  const float d = st.empty() ? -INFINITY : t.x - st.m;
  return t.q * fmaf(t.log_q + log_s, temperature, -d);
}

__device__ __forceinline__ void store_row(const DistillParams& p, int64_t i, float loss, float m, float s) {
  if (threadIdx.x != 0) return;
  p.loss[i] = loss;
  p.stats[2 * i] = m;
  p.stats[2 * i + 1] = s;
}

template <int kSize>
__device__ __forceinline__ void finish_loss(const DistillParams& p, int64_t i, float weight, const Entry& t,
                                            const Stats& st, GroupShared<kSize>& sh) {
  const float log_s = st.log_s();
  const float loss = group_sum(loss_term(t, st, log_s, p.t), sh);
  store_row(p, i, weight * (p.t * loss), st.m, st.s);
}

// A work-group per row, or per part of a row (then distill_join_kernel finishes the row).
template <int kSize, typename T>
__global__ __launch_bounds__(kSize) void distill_loss_kernel(DistillParams p, Parts parts, int64_t first) {
  __shared__ GroupShared<kSize> sh;
  const int32_t part = blockIdx.x % parts.parts;
  const int64_t i = first + blockIdx.x / parts.parts;
  const float weight = row_weight(p, i);
  if (weight == 0.f) {
    if (parts.parts == 1) store_row(p, i, 0.f, -INFINITY, 0.f);
    return;
  }
  const Row<T> row(p.logits, p.stride, i, p.vocab);
  RawEntry raw;
  if (parts.parts == 1) raw = load_entry(p, row, i);
  Running st(p.c);
  TopK none;
  row_pass<kSize, T, false, false>(row, row.begin(part, parts.parts), row.begin(part + 1, parts.parts),
                                   part + 1 == parts.parts, st, none);
  join_group(st, p.c, sh);
  if (parts.parts == 1) {
    finish_loss(p, i, weight, teacher_entry(p, raw, sh), st, sh);
  } else if (threadIdx.x == 0) {
    parts.stats[i * parts.parts + part] = float4{st.m, st.s, 0.f, 0.f};
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join_kernel(DistillParams p, Parts parts, int64_t first) {
  __shared__ GroupShared<kThreads> sh;
  const int64_t i = first + blockIdx.x;
  const float weight = row_weight(p, i);
  if (weight == 0.f) {
    store_row(p, i, 0.f, -INFINITY, 0.f);
    return;
  }
  const RawEntry raw = load_entry(p, Row<T>(p.logits, p.stride, i, p.vocab), i);
  const Stats st = join_parts(parts, i, p.c, sh);
  finish_loss(p, i, weight, teacher_entry(p, raw, sh), st, sh);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_grad_kernel(DistillParams p, int32_t parts, int64_t first) {
  const uint32_t group = gridDim.x - 1 - blockIdx.x;  // as logprobs_grad_kernel
  __shared__ GroupShared<kThreads> sh;
  __shared__ Terms terms;
  const int64_t i = first + group / parts;
  const float weight = row_weight(p, i);
  const Row<T> row(p.logits, p.stride, i, p.vocab);
  const Range<T> range(row, group % parts, parts);
  auto* out = static_cast<typename T::raw*>(p.out) + i * p.vocab;
  const float m = p.stats[2 * i], s = p.stats[2 * i + 1];
  if (weight == 0.f || (m == -INFINITY && s == 0.f)) {
    zero_row<kThreads>(row, out, range);
    return;
  }
  const Entry t = teacher_entry(p, load_entry(p, row, i), sh);
  const float wt = weight * p.t;
  terms.set(t.q != 0.f ? t.id : -1, -wt * t.q, t.x, p.top);
  const float total = group_sum(t.q, sh);
  if (total == 0.f) {  // nothing to learn, also from a row that is no numbers
    zero_row<kThreads>(row, out, range);
    return;
  }
  const Scale scale(m, p.c);
  const float a = grad_factor(wt * total, scale, s);
  auto f = [&](float y) { return a * __builtin_amdgcn_exp2f(y); };
  map_logits<kThreads>(row, out, range, scale, f);
  terms.write<kThreads>(row, out, range, range.v0, p.top, scale, f);
}

// Loss and gradient of a row by one work-group that keeps the row's first kSize * kHeld vectors in
// registers between the two; the rest of a longer row is read a second time, last vectors first,
// while the caches still hold them.  Bound by HBM: 8192 rows of 256 KiB, a tenth of them not
// read, 737 us (5.5 TB/s; two kernels that each read the logits 1224 us).  The gradient is stored
// and the rest read the second time non-temporally (999 -> 930 us, 774 -> 757 us), so that they
// leave the logits in the caches.
template <int kSize, int kHeld, typename T>
__global__ __launch_bounds__(kSize) void distill_step_kernel(DistillParams p, int64_t first) {
  constexpr int E = kElems<T>;
  __shared__ GroupShared<kSize> sh;
  __shared__ Terms terms;
  const int64_t i = first + blockIdx.x;
  const float weight = row_weight(p, i);
  const Row<T> row(p.logits, p.stride, i, p.vocab);
  Range<T> range(row, 0, 1);
  auto* out = static_cast<typename T::raw*>(p.out) + i * p.vocab;
  if (weight == 0.f) {
    store_row(p, i, 0.f, -INFINITY, 0.f);
    zero_row<kSize>(row, out, range);
    return;
  }
  const RawEntry raw = load_entry(p, row, i);  // before the row, to be there before it
  Vec16 w[kHeld];
#pragma unroll
  for (int r = 0; r < kHeld; ++r) {
    const int32_t v = r * kSize + static_cast<int32_t>(threadIdx.x);
    w[r] = v < row.nvec ? load16(row.p + row.index(v)) : Vec16{{T::kNegInf, T::kNegInf, T::kNegInf, T::kNegInf}};
  }
  const Entry t = teacher_entry(p, raw, sh);  // while the row comes
  const float wt = weight * p.t;
  terms.set(t.q != 0.f ? t.id : -1, -wt * t.q, t.x, p.top);
  Running st(p.c);
#pragma unroll
  for (int r = 0; r < kHeld; r += 2) {
    float x[2 * E];
#pragma unroll
    for (int g = 0; g < 2; ++g) unpack<T>(w[r + g], x + g * E);
    st.absorb<2 * E, false>(x, max_of<2 * E>(x));
  }
  TopK none;
  const int32_t held = std::min(row.nvec, kSize * kHeld);
  row_pass<kSize, T, false, false>(row, held, row.nvec, true, st, none);
  join_group(st, p.c, sh);
  const float m = st.m, log_s = st.log_s();
  float loss = loss_term(t, st, log_s, p.t), total = t.q;
  group_sum(loss, total, sh);
  store_row(p, i, weight * (p.t * loss), m, st.s);
  if (st.empty() || total == 0.f) {  // no student or no teacher
    zero_row<kSize>(row, out, range);
    return;
  }
  const Scale scale(m, p.c);
  const float a = grad_factor(wt * total, scale, st.s);
  auto f = [&](float y) { return a * __builtin_amdgcn_exp2f(y); };
  scale.with([&](auto y) {
#pragma unroll
    for (int r = 0; r < kHeld; ++r) {
      const int32_t v = r * kSize + static_cast<int32_t>(threadIdx.x);
      float x[E];
      reread(w[r]);
      unpack<T>(w[r], x);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = f(y(x[e]));
      if (v < row.nvec) store16_once(out + row.index(v), pack<T>(x));
    }
  });
  range.v0 = held;
  map_logits<kSize>(row, out, range, scale, f);
  terms.write<kSize>(row, out, range, 0, p.top, scale, f);  // `held` is a multiple of kSize, or the whole row
}

// ---------------------------------------------------------------- host side

// `groups` work-groups per row.
template <typename P>
int launch_rows(const void* kernel, int64_t rows, int64_t groups, int threads, P& params, void* more,
                hipStream_t stream) {
  const int64_t most = kMaxThreads / threads / groups;
  for (int64_t first = 0; first < rows; first += most) {
    void* args[3] = {&params, more ? more : static_cast<void*>(&first), &first};
    const hipError_t err = hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(std::min(most, rows - first) * groups)),
                                           dim3(threads), args, 0, stream);
    if (err != hipSuccess) return fail(TBE_ERR_LAUNCH, "kernel launch failed: %s", hipGetErrorString(err));
  }
  return TBE_OK;
}

// Parts of a row and threads of a work-group for a pass over the logits.
struct RowPlan {
  int32_t parts;
  int threads;
};

// Wide work-groups keep the GPU busy with few rows; 300 of them and more share a CU, which two of 512 threads
// can.  us, top 20, 1024 / 512 / 256 threads: 64 x 32768 bf16 11.7 / 12.1 / 15.4; 300 x 131072 44.5 / 36.8 /
// 43.0; 1000 x 131072 - / 69.1 / 61.6.
// A few long rows are cut into parts, of at least the 32 KiB that 512 threads load at once, which a second
// launch of about 3 us joins: 1 x 131072 bf16, top 20, 8 parts 13.2, 4 of 1024 threads 14.7, one of 256 32.4.
// That launch pays for shorter rows only with a top list, whose instructions bound the pass, and few rows
// (fp32, one work-group of 1024 / parts): top 20 1 x 50000 15.0 / 11.7, 24 x 32768 11.8 / 11.1, 128 x 40000 13.7
// / 14.5; no list 24 x 32768 6.9 / 9.9, 24 x 100003 fp16 10.9 / 9.7.
// Up to 320 long rows, which as quarters of 256 threads are 1280 work-groups, the 5 that every CU holds at once,
// are quartered too if lists are asked for: else a CU has one long row or two.  One part of 512 threads / four of
// 256, the two sides of each edge (no list, 300 x 100003 fp16: 16.8 / 18.4):
//   bf16, top 5, 300 rows   65536 tokens 22.1 / 21.4   81920 25.1 / 25.9    98304 28.1 / 26.0   131072 33.8 / 29.6
//         131072 tokens     225 rows 26.6 / 26.3       256 27.1 / 26.6      320 34.1 / 29.8     328 34.1 / 35.3
//         98304 tokens      225 rows 22.2 / 23.1       256 22.4 / 23.3      257 26.2 / 24.9     320 28.3 / 26.3
//   fp32, top 5, 300 rows   49152 tokens 21.8 / 21.9   65536 26.1 / 24.9    100003, top 64 39.9 / 35.2
//         65536 tokens      225 rows 22.5 / 22.2       320 26.2 / 25.8      328 26.4 / 27.5     384 27.3 / 30.1
// Lists of 64 gain more: 225 x 131072 bf16 32.8 / 30.1, fp32 41.4 / 36.3.
RowPlan row_plan(int64_t rows, int64_t vocab, int32_t dtype, bool lists) {
  const int64_t quartered = dtype == TBE_TY_FP32 ? 65536 : rows > 256 ? 98304 : 131072;
  if (lists && rows >= 224 && rows <= 320 && vocab >= quartered) return {4, 256};
  if (rows >= 512) return {1, 256};
  if (rows >= 224) return {1, 512};
  const int64_t one_step = (32 << 10) / (dtype == TBE_TY_FP32 ? 4 : 2);
  const int64_t parts = std::min<int64_t>({kMaxParts, 512 / std::max<int64_t>(rows, 1), vocab / one_step});
  if (parts >= 4 && (vocab > 65536 || (lists && rows <= 64))) return {static_cast<int32_t>(parts), 512};
  return {1, 1024};
}
// Calls f with the number of threads.
template <typename F>
void with_threads(int threads, F&& f) {
  switch (threads) {
    case 256: f(std::integral_constant<int, 256>{}); break;
    case 512: f(std::integral_constant<int, 512>{}); break;
    default: f(std::integral_constant<int, 1024>{});
  }
}
int32_t grad_parts(int64_t rows, int64_t vocab) {
  return static_cast<int32_t>(
      std::max<int64_t>(1, std::min<int64_t>({kMaxParts, 1024 / std::max<int64_t>(rows, 1), vocab / 8192})));
}
int64_t parts_bytes(int64_t rows, int64_t vocab, bool lists) {
  const RowPlan r = row_plan(rows, vocab, TBE_TY_FP32, lists);  // no type has more parts
  return r.parts == 1 ? 0 : rows * r.parts * (16 + (lists ? 8 * kWave : 0));
}
Parts parts_of(void* workspace, int64_t rows, const RowPlan& r) {
  auto* stats = static_cast<float4*>(workspace);
  return {stats, reinterpret_cast<uint64_t*>(stats + rows * r.parts), r.parts};
}

// log2(e) / T, rounded once.
float factor_of(float temperature) { return static_cast<float>(1.4426950408889634 / temperature); }

// The checks that every entry point makes of its rows of logits and its lists.
int check_rows(int64_t rows, int64_t vocab, int64_t stride, int32_t dtype, float temperature, int32_t index_size) {
  if (!is_type(dtype)) return fail(TBE_ERR_INVALID_ARG, "logits must be float32, float16 or bfloat16 (type %d)", dtype);
  if (index_size != 4 && index_size != 8)
    return fail(TBE_ERR_INVALID_ARG, "tokens must be int32 or int64 (%d bytes)", index_size);
  if (rows < 0 || vocab < 1 || vocab > INT32_MAX || stride < 0 || rows > (INT64_MAX >> 12) / std::max(vocab, stride))
    return fail(TBE_ERR_INVALID_ARG, "bad shape");
  if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(factor_of(temperature)))
    return fail(TBE_ERR_INVALID_ARG, "temperature must be positive and finite");
  return TBE_OK;
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
  if (bytes < need || (need > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)))
    return fail(TBE_ERR_INVALID_ARG, "a workspace of %lld bytes, 256-byte aligned, is needed",
                static_cast<long long>(need));
  return TBE_OK;
}

int check_distill(const TbeTopkDistillArgs* a, bool loss) {
  if (!a) return fail(TBE_ERR_INVALID_ARG, "null args");
  if (const int rc = check_rows(a->num_rows, a->vocab, a->logits_stride, a->logits_dtype, a->temperature,
                                a->index_size))
    return rc;
  if (a->top < 1 || a->top > kListed)
    return fail(TBE_ERR_INVALID_ARG, "a row lists 1 to %d teacher tokens (%d)", kListed, a->top);
  if (!is_type(a->teacher_dtype))
    return fail(TBE_ERR_INVALID_ARG, "teacher_values must be float32, float16 or bfloat16 (type %d)",
                a->teacher_dtype);
  if (a->num_rows > 0 && (!a->logits || !a->teacher_tokens || !a->teacher_values || !a->stats))
    return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  return loss ? check_workspace(a->workspace, a->workspace_bytes, parts_bytes(a->num_rows, a->vocab, false)) : TBE_OK;
}

DistillParams distill_params(const TbeTopkDistillArgs* a) {
  return {a->logits,     a->teacher_tokens, a->teacher_values, a->row_weights, a->loss,
          a->stats,      a->grad_logits,    a->logits_stride,  static_cast<int32_t>(a->vocab),
          a->top,        a->index_size,     a->teacher_dtype,  a->renormalize, a->temperature,
          1.f / a->temperature, factor_of(a->temperature)};
}

}  // namespace
}  // namespace vocab
}  // namespace tbe

using namespace tbe;
using namespace tbe::vocab;

extern "C" int64_t tbe_token_logprobs_workspace_bytes(int64_t num_rows, int64_t vocab, int32_t top_k) {
  if (num_rows < 0 || vocab < 1 || vocab > INT32_MAX || top_k < 0 || top_k > TBE_VOCAB_MAX_TOP_K) return -1;
  return parts_bytes(num_rows, vocab, top_k > 0);
}

extern "C" int tbe_token_logprobs(const TbeTokenLogprobsArgs* a, void* hip_stream) {
  clear_error();
  if (!a) return fail(TBE_ERR_INVALID_ARG, "null args");
  if (const int rc = check_rows(a->num_rows, a->vocab, a->logits_stride, a->logits_dtype, a->temperature,
                                a->index_size))
    return rc;
  if (a->given < 0 || a->given > kListed)
    return fail(TBE_ERR_INVALID_ARG, "a row gives at most %d tokens (%d)", kListed, a->given);
  if (a->top_k < 0 || a->top_k > TBE_VOCAB_MAX_TOP_K || a->top_k > a->vocab)
    return fail(TBE_ERR_INVALID_ARG, "top_k must be between 0 and min(%d, vocab) (%d)", TBE_VOCAB_MAX_TOP_K, a->top_k);
  if (a->num_rows == 0) return TBE_OK;
  if (!a->logits || !a->entropy || !a->stats || (a->given > 0 && (!a->tokens || !a->logprobs)) ||
      (a->top_k > 0 && (!a->top_logprobs || !a->top_tokens)))
    return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  LogprobsParams p{a->logits, a->tokens, a->logprobs, a->entropy, a->top_logprobs, a->top_tokens, a->stats,
                   a->logits_stride, static_cast<int32_t>(a->vocab), a->given, a->index_size, a->top_k,
                   a->temperature, factor_of(a->temperature)};
  if (const int rc = check_workspace(a->workspace, a->workspace_bytes,
                                     tbe_token_logprobs_workspace_bytes(a->num_rows, a->vocab, a->top_k)))
    return rc;
  const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  const RowPlan plan = row_plan(a->num_rows, a->vocab, a->logits_dtype, a->top_k > 0);
  Parts parts = parts_of(a->workspace, a->num_rows, plan);
  int rc = TBE_OK;
  with_type(a->logits_dtype, [&](auto t) {
    using T = decltype(t);
    const void* k = nullptr;
    with_threads(plan.threads, [&](auto n) {
      k = a->top_k > 0 ? reinterpret_cast<const void*>(logprobs_kernel<decltype(n)::value, T, true>)
                       : reinterpret_cast<const void*>(logprobs_kernel<decltype(n)::value, T, false>);
    });
    rc = launch_rows(k, a->num_rows, plan.parts, plan.threads, p, &parts, stream);
    if (rc == TBE_OK && plan.parts > 1)
      rc = launch_rows(reinterpret_cast<const void*>(logprobs_join_kernel<T>), a->num_rows, 1, kThreads, p, &parts,
                       stream);
  });
  return rc;
}

extern "C" int tbe_token_logprobs_grad(const TbeTokenLogprobsGradArgs* a, void* hip_stream) {
  clear_error();
  if (!a) return fail(TBE_ERR_INVALID_ARG, "null args");
  if (const int rc = check_rows(a->num_rows, a->vocab, a->logits_stride, a->logits_dtype, a->temperature,
                                a->index_size))
    return rc;
  if (a->given < 0 || a->given > kListed)
    return fail(TBE_ERR_INVALID_ARG, "a row gives at most %d tokens (%d)", kListed, a->given);
  if (a->num_rows == 0) return TBE_OK;
  if (!a->logits || !a->stats || !a->grad_logits || (a->given > 0 && a->grad_logprobs && !a->tokens) ||
      (a->grad_entropy && !a->entropy))
    return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  LogprobsGradParams p{a->logits, a->tokens, a->grad_logprobs, a->grad_entropy, a->entropy, a->stats, a->grad_logits,
                       a->logits_stride, static_cast<int32_t>(a->vocab), a->given, a->index_size,
                       1.f / a->temperature, factor_of(a->temperature)};
  int32_t parts = grad_parts(a->num_rows, a->vocab);
  int rc = TBE_OK;
  with_type(a->logits_dtype, [&](auto t) {
    rc = launch_rows(reinterpret_cast<const void*>(logprobs_grad_kernel<decltype(t)>), a->num_rows, parts, kThreads, p,
                     &parts, static_cast<hipStream_t>(hip_stream));
  });
  return rc;
}

extern "C" int64_t tbe_topk_distill_workspace_bytes(int64_t num_rows, int64_t vocab) {
  if (num_rows < 0 || vocab < 1 || vocab > INT32_MAX) return -1;
  return parts_bytes(num_rows, vocab, false);
}

namespace tbe {
namespace vocab {
namespace {

int distill_loss(const TbeTopkDistillArgs* a, DistillParams& p, hipStream_t stream) {
  const RowPlan plan = row_plan(a->num_rows, a->vocab, a->logits_dtype, false);
  Parts parts = parts_of(a->workspace, a->num_rows, plan);
  int rc = TBE_OK;
  with_type(a->logits_dtype, [&](auto t) {
    using T = decltype(t);
    const void* k = nullptr;
    with_threads(plan.threads, [&](auto n) {
      k = reinterpret_cast<const void*>(distill_loss_kernel<decltype(n)::value, T>);
    });
    rc = launch_rows(k, a->num_rows, plan.parts, plan.threads, p, &parts, stream);
    if (rc == TBE_OK && plan.parts > 1)
      rc = launch_rows(reinterpret_cast<const void*>(distill_join_kernel<T>), a->num_rows, 1, kThreads, p, &parts,
                       stream);
  });
  return rc;
}

int distill_grad(const TbeTopkDistillArgs* a, DistillParams& p, hipStream_t stream) {
  int32_t parts = grad_parts(a->num_rows, a->vocab);
  int rc = TBE_OK;
  with_type(a->logits_dtype, [&](auto t) {
    rc = launch_rows(reinterpret_cast<const void*>(distill_grad_kernel<decltype(t)>), a->num_rows, parts, kThreads, p,
                     &parts, stream);
  });
  return rc;
}

}  // namespace
}  // namespace vocab
}  // namespace tbe

extern "C" int tbe_topk_distill_loss(const TbeTopkDistillArgs* a, void* hip_stream) {
  clear_error();
  if (const int rc = check_distill(a, true)) return rc;
  if (a->num_rows == 0) return TBE_OK;
  if (!a->loss) return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  DistillParams p = distill_params(a);
  return distill_loss(a, p, static_cast<hipStream_t>(hip_stream));
}

extern "C" int tbe_topk_distill_grad(const TbeTopkDistillArgs* a, void* hip_stream) {
  clear_error();
  if (const int rc = check_distill(a, false)) return rc;
  if (a->num_rows == 0) return TBE_OK;
  if (!a->grad_logits) return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  DistillParams p = distill_params(a);
  return distill_grad(a, p, static_cast<hipStream_t>(hip_stream));
}

extern "C" int tbe_topk_distill_step(const TbeTopkDistillArgs* a, void* hip_stream) {
  clear_error();
  if (const int rc = check_distill(a, true)) return rc;
  if (a->num_rows == 0) return TBE_OK;
  if (!a->loss || !a->grad_logits) return fail(TBE_ERR_INVALID_ARG, "null pointer argument");
  const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
  DistillParams p = distill_params(a);
  // Few long rows: one work-group a row leaves the GPU idle, two passes over parts of rows do not.
  // How many rows are few goes with their tokens, whatever the type.  us, two passes / one, bf16 and fp32:
  //   73728 tokens     8 rows 14.4 / 14.2, 14.1 / 15.3    40 15.8 / 14.8, 18.0 / 15.9
  //   98304           32 15.2 / 16.3, 18.3 / 18.9         64 18.3 / 16.5, 24.1 / 20.5
  //   131072          48 18.2 / 20.0, 23.9 / 24.7         80 24.6 / 20.4, 32.4 / 28.8
  //   262144          96 39.4 / 40.5, 61.0 / 68.8        144 51.1 / 46.6, 84.3 / 83.4
  //   524288         144 90.3 / 94.8, 164 / 179          192 112 / 107, 217 / 207
  if (a->vocab >= 81920 && a->num_rows <= std::min<int64_t>(160, a->vocab / 2560)) {
    const int rc = distill_loss(a, p, stream);
    return rc != TBE_OK ? rc : distill_grad(a, p, stream);
  }
  int rc = TBE_OK;
  with_type(a->logits_dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t vecs = a->vocab / kElems<T>;
    const void* k;
    int threads;
    auto take = [&](auto size, auto held) {
      threads = decltype(size)::value;
      k = reinterpret_cast<const void*>(distill_step_kernel<decltype(size)::value, decltype(held)::value, T>);
    };
    // The smallest work-group whose registers hold the row, while it has a thread per listed
    // token; a longer row goes half of it, or what fits of it, through registers.  All of a
    // 256 KiB row in the registers of 1024 threads (16 vectors each) was slower than half of it:
    // nothing is loaded while the whole of it is summed (8192 rows 932 us, half 814 us).
    // us, rows of 8 KiB / 16 / 32 / 64 / 128 / 256, about 0.4 GB (the first three) and 0.8 GB:
    //   64 x 8 threads x vectors 194 / 194 / 200, 128 x 8 208 / 167 / 169, 256 x 8 296 / 177 / 155 / 617 / 654 / 755,
    //   512 x 8 759 / 408 / 237 / 606 / 597 / 683, 512 x 16 - / - / - / 720 / 594 / 618,
    //   1024 x 8 - / - / - / 802 / 696 / 612
    if (vecs <= 64 * 8 && a->top <= 64) {
      take(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{});
    } else if (vecs <= 128 * 8 && a->top <= 128) {
      take(std::integral_constant<int, 128>{}, std::integral_constant<int, 8>{});
    } else if (vecs <= 256 * 8) {
      take(std::integral_constant<int, 256>{}, std::integral_constant<int, 8>{});
    } else if (vecs <= 512 * 8) {
      take(std::integral_constant<int, 512>{}, std::integral_constant<int, 8>{});
    } else if (vecs <= 512 * 16) {
      take(std::integral_constant<int, 512>{}, std::integral_constant<int, 16>{});
    } else {
      take(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
    }
    rc = launch_rows(k, a->num_rows, 1, threads, p, nullptr, stream);
  });
  return rc;
}
