// Element types of the operators that take fp32, bf16 or fp16 tensors: loads widen to fp32, stores
// round once (to nearest even).
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace mx {

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct F32 {
  using store_t = float;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ float load(float v) { return v; }
  static __device__ __forceinline__ float store(float v) { return v; }
};
struct BF16 {
  using store_t = uint16_t;
  static constexpr uint32_t kNegInf = 0xff80u;
  static __device__ __forceinline__ float load(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t store(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
  }
};
struct F16 {
  using store_t = uint16_t;
  static constexpr uint32_t kNegInf = 0xfc00u;
  static __device__ __forceinline__ float load(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ uint16_t store(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

// one element of a tensor whose type is known at run time (rarely read operands)
__device__ __forceinline__ float load_any(const void* p, int64_t i, int type) {
  if (type == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  return type == kBF16 ? BF16::load(v) : F16::load(v);
}

// 16 bytes at any address: global memory takes them in one access whatever their alignment
struct __attribute__((packed, aligned(1))) Bytes16 {
  uint32_t v[4];
};

// 16 bytes of a row: 4 fp32 or 8 16-bit elements
template <class T>
struct Piece {
  static constexpr int kN = 16 / sizeof(typename T::store_t);
  uint32_t v[4];
  // elements i .. i + kN - 1 of p, `fill` (the element's bits) where they reach n
  __device__ __forceinline__ void load(const typename T::store_t* p, int64_t i, int64_t n, uint32_t fill) {
    if (i + kN <= n) {
      const Bytes16 b = *reinterpret_cast<const Bytes16*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = b.v[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (kN == 4) {
          v[j] = i + j < n ? __builtin_bit_cast(uint32_t, p[i + j]) : fill;
        } else {
          const uint32_t lo = i + 2 * j < n ? p[i + 2 * j] : fill, hi = i + 2 * j + 1 < n ? p[i + 2 * j + 1] : fill;
          v[j] = lo | hi << 16;
        }
      }
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (kN == 4) return T::load(__builtin_bit_cast(float, v[e]));
    else return T::load((uint16_t)(e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu));
  }
};

#define MX_BY_TYPE(type, T, ...)                                    \
  do {                                                              \
    if ((type) == ::mx::kF32) { using T = ::mx::F32; __VA_ARGS__; } \
    else if ((type) == ::mx::kBF16) { using T = ::mx::BF16; __VA_ARGS__; } \
    else if ((type) == ::mx::kF16) { using T = ::mx::F16; __VA_ARGS__; }   \
    else throw std::runtime_error("mxddp check failed: element type must be fp32, bf16 or fp16"); \
  } while (0)

}  // namespace mx
