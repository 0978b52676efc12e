// vocab_device.h — device helpers shared by the vocabulary operators (vocab_embedding.hip,
// vocab_logits.hip): element types, 16-byte vectors, exchanges between the lanes of a wave.
#ifndef TBE_VOCAB_DEVICE_H
#define TBE_VOCAB_DEVICE_H

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "tbe_nbit.h"

namespace tbe {
namespace vocab {

constexpr int kWave = 64;

struct F32 {
  using raw = uint32_t;
  static constexpr uint32_t kNegInf = 0xFF800000u;  // of a 32-bit word
};
struct F16 {
  using raw = uint16_t;
  static constexpr uint32_t kNegInf = 0xFC00FC00u;
};
struct BF16 {
  using raw = uint16_t;
  static constexpr uint32_t kNegInf = 0xFF80FF80u;
};

// Elements of a 16-byte vector.
template <typename T>
constexpr int kElems = 16 / static_cast<int>(sizeof(typename T::raw));

struct Vec16 {
  uint32_t w[4];
};

// 16 bytes at any alignment of the element.
__device__ __forceinline__ Vec16 load16(const void* p) {
  Vec16 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void store16(void* p, const Vec16& v) { __builtin_memcpy(p, &v, 16); }

// The same for what is read for the last time, or written once and not read here.
__device__ __forceinline__ Vec16 load16_once(const void* p) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  const Words w = __builtin_nontemporal_load(reinterpret_cast<const Words*>(p));
  Vec16 v;
  __builtin_memcpy(&v, &w, 16);
  return v;
}
__device__ __forceinline__ void store16_once(void* p, const Vec16& v) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  Words w;
  __builtin_memcpy(&w, &v, 16);
  __builtin_nontemporal_store(w, reinterpret_cast<Words*>(p));
}

template <typename T>
__device__ __forceinline__ float to_f32(typename T::raw r) {
  if constexpr (sizeof(r) == 4) {
    return __uint_as_float(r);
  } else if constexpr (T::kNegInf == BF16::kNegInf) {
    return __uint_as_float(static_cast<uint32_t>(r) << 16);
  } else {
    return static_cast<float>(__builtin_bit_cast(_Float16, r));
  }
}

// Round to nearest, ties to even; NaN stays NaN.
template <typename T>
__device__ __forceinline__ typename T::raw from_f32(float f) {
  if constexpr (sizeof(typename T::raw) == 4) {
    return __float_as_uint(f);
  } else if constexpr (T::kNegInf == BF16::kNegInf) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(f));
  } else {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(f));
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const Vec16& v, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kElems<T> == 4) {
      x[i] = __uint_as_float(v.w[i]);
    } else {
      x[2 * i] = to_f32<T>(static_cast<uint16_t>(v.w[i]));
      x[2 * i + 1] = to_f32<T>(static_cast<uint16_t>(v.w[i] >> 16));
    }
  }
}

template <typename T>
__device__ __forceinline__ Vec16 pack(const float* x) {
  Vec16 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kElems<T> == 4) {
      v.w[i] = __float_as_uint(x[i]);
    } else if constexpr (T::kNegInf == BF16::kNegInf) {  // two at a time
      typedef float F2 __attribute__((ext_vector_type(2)));
      typedef __bf16 B2 __attribute__((ext_vector_type(2)));
      v.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((F2{x[2 * i], x[2 * i + 1]}), B2));
    } else {
      v.w[i] = static_cast<uint32_t>(from_f32<T>(x[2 * i])) |
               static_cast<uint32_t>(from_f32<T>(x[2 * i + 1])) << 16;
    }
  }
  return v;
}

__device__ __forceinline__ int lane_id() { return static_cast<int>(threadIdx.x) & (kWave - 1); }

// The value of the lane whose number differs in bit J (1, 2, 4, 8, 16 or 32), without LDS.
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  const int i = static_cast<int>(v);
  if constexpr (J == 1) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(i, 0xB1, 0xF, 0xF, true));  // quad_perm 1,0,3,2
  } else if constexpr (J == 2) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(i, 0x4E, 0xF, 0xF, true));  // quad_perm 2,3,0,1
  } else if constexpr (J == 4) {  // mirrored in eights, then in fours
    const int m = __builtin_amdgcn_mov_dpp(i, 0x141, 0xF, 0xF, true);
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(m, 0x1B, 0xF, 0xF, true));
  } else if constexpr (J == 8) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(i, 0x128, 0xF, 0xF, true));  // row_ror:8
  } else if constexpr (J == 16) {  // rows 1 and 0, 3 and 2 swapped between two copies
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? r[0] : r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? r[0] : r[1];
  }
}
template <int J>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<J>(__float_as_uint(v)));
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return static_cast<uint64_t>(lane_xor<J>(static_cast<uint32_t>(v >> 32))) << 32 |
         lane_xor<J>(static_cast<uint32_t>(v));
}

// Orders the accesses of one wave to LDS and memory, of all its lanes (its instructions run in
// order; this stops the compiler).
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Over the first N lanes of every N (a power of two); every lane gets the same bits.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (N > 1) v += lane_xor<1>(v);
  if constexpr (N > 2) v += lane_xor<2>(v);
  if constexpr (N > 4) v += lane_xor<4>(v);
  if constexpr (N > 8) v += lane_xor<8>(v);
  if constexpr (N > 16) v += lane_xor<16>(v);
  if constexpr (N > 32) v += lane_xor<32>(v);
  return v;
}
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (N > 1) v = fmaxf(v, lane_xor<1>(v));
  if constexpr (N > 2) v = fmaxf(v, lane_xor<2>(v));
  if constexpr (N > 4) v = fmaxf(v, lane_xor<4>(v));
  if constexpr (N > 8) v = fmaxf(v, lane_xor<8>(v));
  if constexpr (N > 16) v = fmaxf(v, lane_xor<16>(v));
  if constexpr (N > 32) v = fmaxf(v, lane_xor<32>(v));
  return v;
}

// Host: calls f with the element type of a TBE_TY_* code; false for a code that has none.
template <typename F>
bool with_type(int32_t ty, F&& f) {
  switch (ty) {
    case TBE_TY_FP32: f(F32{}); return true;
    case TBE_TY_FP16: f(F16{}); return true;
    case TBE_TY_BF16: f(BF16{}); return true;
    default: return false;
  }
}
inline bool is_type(int32_t ty) {
  return with_type(ty, [](auto) {});
}

}  // namespace vocab
}  // namespace tbe

#endif  // TBE_VOCAB_DEVICE_H
