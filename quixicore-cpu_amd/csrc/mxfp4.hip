// MXFP4 on gfx950: blocks of 32 values as 4-bit floats (sign, two exponent
// bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) under a power of two.
//
// Of a block, e = clamp(floor(log2 max|x|) - 2, -127, 127) (-127 for a block of
// zeros), stored as the byte e + 127; element x becomes the code of
// x * 2^-e rounded to nearest, ties to the even code, and at most 6.  The
// product with 2^-e is exact in f32 wherever it does not round to zero, so the
// codes are those of the real quotient.
#include <algorithm>

#include "qc_device.h"
#include "qc_internal.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

constexpr int kThreads = 256;

// Power of two 2^e, -127 <= e <= 127, exactly.
__device__ __forceinline__ float pow2(int e) {
  return __int_as_float(e == -127 ? 0x00400000 : (e + 127) << 23);
}

// Largest of a value over the four lanes of a quad.
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, dpp_f32<0xB1>(v));
  return fmaxf(v, dpp_f32<0x4E>(v));
}

// Four lanes a block, eight values each.  v_cvt_scalef32_pk_fp4_f32 rounds to nearest
// even and saturates at 6; its scale stays 1, the power of two is a product before it
// that is exact.  Bound by memory: 14336 x 4096 f32 (235 MB read, 31 written) 65 us with a
// thread per block and the rounding written out, 48 here (5.5 TB/s).  VEC: x rows allow 16-byte
// loads.
template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* __restrict__ x,
                                                            long long stride,
                                                            uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales,
                                                            long long rows, long long blocks,
                                                            int* status) {
  typedef typename Storage<TYPE>::raw raw;
  constexpr int V = Storage<TYPE>::per16;
  const long long step = static_cast<long long>(gridDim.x) * kThreads, quads = 4 * blocks;
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < rows * quads;
       i += step) {
    const long long r = i / quads, q = i - r * quads;
    const raw* src = static_cast<const raw*>(x) + r * stride + 8 * q;
    float v[8];
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 8; j += V)
        decode16<TYPE>(__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + j)), v + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = decode<TYPE>(src[j]);
    }
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad = bad || !isfinite(v[j]);
      top = fmaxf(top, fabsf(v[j]));
    }
    top = quad_max(bad ? INFINITY : top);
    if (top == INFINITY) {
      *status = QC_INVALID_ARGUMENT;
      continue;
    }
    int e = -127;
    if (top > 0.f) {
      (void)frexpf(top, &e);
      e = max(e - 3, -127);
    }
    const float inv = pow2(-e);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0] * inv, v[1] * inv, 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2] * inv, v[3] * inv, 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4] * inv, v[5] * inv, 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6] * inv, v[7] * inv, 1.0f, 3);
    reinterpret_cast<uint32_t*>(codes)[i] = w;
    if ((q & 3) == 0) scales[i >> 2] = static_cast<uint8_t>(e + 127);
  }
}

// A thread per eight values: 14336 x 4096 to f32 (31 MB read, 235 written) 55 us with a byte
// of codes a thread, 39 here (6.8 TB/s).
template <int TYPE, bool VEC>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales,
                                                              void* __restrict__ out,
                                                              long long count) {
  typedef typename Storage<TYPE>::raw raw;
  constexpr int V = Storage<TYPE>::per16;
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < count;
       i += step) {
    const int sb = scales[i >> 2];
    const float d = sb == 255 ? __uint_as_float(0x7FC00000u) : pow2(sb - 127);
    const uint32_t c = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes) + i);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f32x2 e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
    const f32x2 f = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    const float v[8] = {a[0] * d, a[1] * d, b[0] * d, b[1] * d, e[0] * d, e[1] * d, f[0] * d, f[1] * d};
    raw* o = static_cast<raw*>(out) + 8 * i;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < 8; j += V) *reinterpret_cast<u32x4*>(o + j) = encode16<TYPE>(v + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = encode<TYPE>(v[j]);
    }
  }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void mxfp4_nonfinite(const void* __restrict__ x,
                                                            long long stride, long long rows,
                                                            long long dim, int* flag) {
  typedef typename Storage<TYPE>::raw raw;
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < rows * dim;
       i += step) {
    const long long r = i / dim;
    if (!isfinite(decode<TYPE>(static_cast<const raw*>(x)[r * stride + i - r * dim])))
      *flag = QC_INVALID_ARGUMENT;
  }
}

int grid_for(long long items) {
  return static_cast<int>(std::min<long long>((items + kThreads - 1) / kThreads, 1 << 20));
}

}  // namespace

hipError_t launch_mxfp4_nonfinite(const void* x, int type, long long stride, long long rows,
                                  long long dim, int* flag, hipStream_t s) {
  const int grid = static_cast<int>(std::min<long long>((rows * dim + kThreads - 1) / kThreads, 4096));
  switch (type) {
    case QC_STORAGE_F32:
      mxfp4_nonfinite<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(x, stride, rows, dim, flag);
      break;
    case QC_STORAGE_F16:
      mxfp4_nonfinite<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(x, stride, rows, dim, flag);
      break;
    default:
      mxfp4_nonfinite<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(x, stride, rows, dim, flag);
  }
  return hipGetLastError();
}

namespace {

template <int TYPE>
void run_quantize(const void* x, long long stride, uint8_t* codes, uint8_t* scales, long long rows,
                  long long blocks, int* status, hipStream_t s) {
  const int grid = grid_for(4 * rows * blocks);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && stride % Storage<TYPE>::per16 == 0;
  if (vec) quantize_kernel<TYPE, true><<<grid, kThreads, 0, s>>>(x, stride, codes, scales, rows, blocks, status);
  else quantize_kernel<TYPE, false><<<grid, kThreads, 0, s>>>(x, stride, codes, scales, rows, blocks, status);
}

template <int TYPE>
void run_dequantize(const uint8_t* codes, const uint8_t* scales, void* out, long long count, hipStream_t s) {
  const int grid = grid_for(count);
  if (reinterpret_cast<uintptr_t>(out) % 16 == 0)
    dequantize_kernel<TYPE, true><<<grid, kThreads, 0, s>>>(codes, scales, out, count);
  else
    dequantize_kernel<TYPE, false><<<grid, kThreads, 0, s>>>(codes, scales, out, count);
}

}  // namespace

hipError_t launch_quantize_mxfp4(const void* x, int type, long long stride, uint8_t* codes,
                                 uint8_t* scales, long long rows, long long dim, int* status,
                                 hipStream_t s) {
  switch (type) {
    case QC_STORAGE_F32: run_quantize<QC_STORAGE_F32>(x, stride, codes, scales, rows, dim / 32, status, s); break;
    case QC_STORAGE_F16: run_quantize<QC_STORAGE_F16>(x, stride, codes, scales, rows, dim / 32, status, s); break;
    default: run_quantize<QC_STORAGE_BF16>(x, stride, codes, scales, rows, dim / 32, status, s);
  }
  return hipGetLastError();
}

hipError_t launch_dequantize_mxfp4(const uint8_t* codes, const uint8_t* scales, void* out, int type,
                                   long long rows, long long dim, hipStream_t s) {
  const long long count = rows * (dim / 8);
  switch (type) {
    case QC_STORAGE_F32: run_dequantize<QC_STORAGE_F32>(codes, scales, out, count, s); break;
    case QC_STORAGE_F16: run_dequantize<QC_STORAGE_F16>(codes, scales, out, count, s); break;
    default: run_dequantize<QC_STORAGE_BF16>(codes, scales, out, count, s);
  }
  return hipGetLastError();
}

}  // namespace qc
