// 16-byte vectors of f32 / f16 / bf16 storage, decoded exactly to f32 and
// rounded once (nearest even, NaN kept) on the way back.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "quixicore_hip.h"

namespace qc {
namespace storage {

template <int TYPE>
struct Storage {   // the two 16-bit types
  typedef uint16_t raw;
  static constexpr int per16 = 8;   // elements of 16 bytes
};
template <>
struct Storage<QC_STORAGE_F32> {
  typedef uint32_t raw;
  static constexpr int per16 = 4;
};

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int TYPE>
__device__ __forceinline__ float decode(typename Storage<TYPE>::raw b) {
  if constexpr (TYPE == QC_STORAGE_F32) return __uint_as_float(b);
  else if constexpr (TYPE == QC_STORAGE_F16) return static_cast<float>(__builtin_bit_cast(_Float16, b));
  else return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

// The value as it stands in f32.  A conversion to f16 that the compiler sees beside the
// product it takes becomes one instruction without the f32 rounding between, in some of the
// places that use it and not in others.
__device__ __forceinline__ float in_f32(float v) {
  asm("" : "+v"(v));
  return v;
}

template <int TYPE>
__device__ __forceinline__ typename Storage<TYPE>::raw encode(float v) {
  if constexpr (TYPE == QC_STORAGE_F32) return __float_as_uint(v);
  else if constexpr (TYPE == QC_STORAGE_F16)
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(in_f32(v)));
  else return __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

// Two values as one dword of a 16-bit type.
template <int TYPE>
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  static_assert(TYPE != QC_STORAGE_F32, "16-bit types");
  const f32x2 v = {in_f32(a), in_f32(b)};
  if constexpr (TYPE == QC_STORAGE_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

// The Storage<TYPE>::per16 values of 16 bytes.
template <int TYPE>
__device__ __forceinline__ void decode16(const u32x4& w, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TYPE == QC_STORAGE_F32) {
      v[i] = __uint_as_float(w[i]);
    } else {
      v[2 * i] = decode<TYPE>(static_cast<uint16_t>(w[i]));
      v[2 * i + 1] = decode<TYPE>(static_cast<uint16_t>(w[i] >> 16));
    }
  }
}

template <int TYPE>
__device__ __forceinline__ u32x4 encode16(const float* v) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (TYPE == QC_STORAGE_F32) w[i] = __float_as_uint(v[i]);
    else w[i] = encode2<TYPE>(v[2 * i], v[2 * i + 1]);
  }
  return w;
}

}  // namespace storage
}  // namespace qc
