// MXFP4 on gfx950: blocks of 32 values as 4-bit floats (sign, two exponent
// bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) under a power of two.
//
// Of a block, e = clamp(floor(log2 max|x|) - 2, -127, 127) (-127 for a block of
// zeros), stored as the byte e + 127; element x becomes the code of
// x * 2^-e rounded to nearest, ties to the even code, and at most 6.  The
// product with 2^-e is exact in f32 wherever it does not round to zero, so the
// codes are those of the real quotient.
#include <algorithm>

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

__device__ __forceinline__ uint32_t e2m1(float v) {
  const float a = fabsf(v);
  const uint32_t code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) +
                        (a >= 3.5f) + (a > 5.0f);
  return code | (__float_as_uint(v) >> 31 << 3);
}

__device__ __forceinline__ float e2m1_value(uint32_t code) {
  const uint32_t m = code & 7;
  const float a = m < 2 ? 0.5f * m : __uint_as_float((126 + (m >> 1)) << 23 | (m & 1) << 22);
  return code & 8 ? -a : a;
}

// One thread per block of 32.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const void* __restrict__ x,
                                                            long long stride,
                                                            uint8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ scales,
                                                            long long rows, long long blocks,
                                                            int* status) {
  typedef typename Storage<TYPE>::raw raw;
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < rows * blocks;
       i += step) {
    const long long r = i / blocks, b = i - r * blocks;
    const raw* src = static_cast<const raw*>(x) + r * stride + 32 * b;
    float v[32], top = 0.f;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      v[j] = decode<TYPE>(src[j]);
      bad = bad || !isfinite(v[j]);
      top = fmaxf(top, fabsf(v[j]));
    }
    if (bad) {
      *status = QC_INVALID_ARGUMENT;
      continue;
    }
    int e = -127;
    if (top > 0.f) {
      (void)frexpf(top, &e);
      e = max(e - 3, -127);
    }
    const float inv = pow2(-e);
    u32x4 w;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      w[q] = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[q] |= e2m1(v[8 * q + j] * inv) << (4 * j);
    }
    uint8_t* out = codes + 16 * i;
#pragma unroll
    for (int q = 0; q < 16; ++q) out[q] = static_cast<uint8_t>(w[q / 4] >> (8 * (q % 4)));
    scales[i] = static_cast<uint8_t>(e + 127);
  }
}

template <int TYPE>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales,
                                                              void* __restrict__ out,
                                                              long long count) {
  typedef typename Storage<TYPE>::raw raw;
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < count;
       i += step) {
    const int sb = scales[i >> 4];
    const float d = sb == 255 ? __uint_as_float(0x7FC00000u) : pow2(sb - 127);
    const uint32_t c = codes[i];
    static_cast<raw*>(out)[2 * i] = encode<TYPE>(e2m1_value(c & 15) * d);
    static_cast<raw*>(out)[2 * i + 1] = encode<TYPE>(e2m1_value(c >> 4) * d);
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

hipError_t launch_quantize_mxfp4(const void* x, int type, long long stride, uint8_t* codes,
                                 uint8_t* scales, long long rows, long long dim, int* status,
                                 hipStream_t s) {
  const int grid = grid_for(rows * (dim / 32));
  switch (type) {
    case QC_STORAGE_F32:
      quantize_kernel<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(x, stride, codes, scales, rows, dim / 32, status);
      break;
    case QC_STORAGE_F16:
      quantize_kernel<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(x, stride, codes, scales, rows, dim / 32, status);
      break;
    default:
      quantize_kernel<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(x, stride, codes, scales, rows, dim / 32, status);
  }
  return hipGetLastError();
}

hipError_t launch_dequantize_mxfp4(const uint8_t* codes, const uint8_t* scales, void* out, int type,
                                   long long rows, long long dim, hipStream_t s) {
  const long long count = rows * dim / 2;
  const int grid = grid_for(count);
  switch (type) {
    case QC_STORAGE_F32:
      dequantize_kernel<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(codes, scales, out, count);
      break;
    case QC_STORAGE_F16:
      dequantize_kernel<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(codes, scales, out, count);
      break;
    default:
      dequantize_kernel<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(codes, scales, out, count);
  }
  return hipGetLastError();
}

}  // namespace qc
