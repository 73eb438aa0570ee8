// Rotary positions on gfx950: tables of cosines and sines for contexts of any
// scaling, and the rotation of many tokens' heads by them.
//
// Pair i of a head's first R = rotary_dim elements, (a, b), at position p:
//   a' = a cos(p w_i) - b sin(p w_i),  b' = b cos(p w_i) + a sin(p w_i)
// with (a, b) = elements (i, i + R/2) in the half layout, (2 i, 2 i + 1) in the
// interleaved one, w_i = base^(-2 i / R) before scaling.  Products and sums are
// rounded to f32 one by one, as the single-token seam's are, then once to the
// output's type.
#include <algorithm>

#include "qc_internal.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

constexpr int kThreads = 256;

struct RopeArgs {
  const void* x;
  void* y;
  long long xt, xh, yt, yh;      // elements between tokens and between heads
  const float* cosine;
  const float* sine;
  const int* positions;
  int max_position;
  int heads, rotary, head_dim;
  int tokens;
  int* status;
};

// One thread per token, head and chunk of V pairs (V elements past the rotated
// part, which are copied where y is another array than x).
template <int TYPE, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a, int chunks, int rot_chunks) {
  typedef typename Storage<TYPE>::raw raw;
  const uint32_t per_token = static_cast<uint32_t>(a.heads) * chunks;
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t token = id / per_token;
  if (token >= static_cast<uint32_t>(a.tokens)) return;
  const uint32_t rest = id - token * per_token;
  const int head = rest / chunks, chunk = rest - head * chunks;
  const int p = a.positions[token];
  if (p == -1) return;
  if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.max_position)) {
    if (rest == 0) *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const raw* x = static_cast<const raw*>(a.x) + token * a.xt + head * a.xh;
  raw* y = static_cast<raw*>(a.y) + token * a.yt + head * a.yh;
  if (chunk >= rot_chunks) {
    const int d = a.rotary + (chunk - rot_chunks) * V;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (d + j < a.head_dim) y[d + j] = x[d + j];
    return;
  }
  const int half = a.rotary / 2, i0 = chunk * V;
  const float* c = a.cosine + static_cast<long long>(p) * half;
  const float* s = a.sine + static_cast<long long>(p) * half;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int i = i0 + j;
    if (i >= half) return;
    const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : i + half;
    const float u = decode<TYPE>(x[ia]), v = decode<TYPE>(x[ib]);
    y[ia] = encode<TYPE>(u * c[i] - v * s[i]);
    y[ib] = encode<TYPE>(v * c[i] + u * s[i]);
  }
}

// Any position outside [-1, max_position): *flag = 3.
__global__ __launch_bounds__(kThreads) void rope_check(const int* __restrict__ positions,
                                                       int tokens, int max_position, int* flag) {
  for (int t = blockIdx.x * kThreads + threadIdx.x; t < tokens; t += gridDim.x * kThreads)
    if (positions[t] < -1 || positions[t] >= max_position) *flag = QC_INVALID_ARGUMENT;
}

template <int TYPE>
hipError_t rope_typed(const RopeArgs& a, bool interleaved, bool copy, hipStream_t s) {
  constexpr int V = 4;
  const int rot_chunks = (a.rotary / 2 + V - 1) / V;
  const int chunks = rot_chunks + (copy ? (a.head_dim - a.rotary + V - 1) / V : 0);
  const long long per_token = static_cast<long long>(a.heads) * chunks;
  // ids are 32-bit: slices of tokens
  const long long slice = std::max<long long>(1, (1LL << 30) / per_token);
  for (long long t0 = 0; t0 < a.tokens; t0 += slice) {
    RopeArgs b = a;
    b.tokens = static_cast<int>(std::min(slice, a.tokens - t0));
    b.x = static_cast<const typename Storage<TYPE>::raw*>(a.x) + t0 * a.xt;
    b.y = static_cast<typename Storage<TYPE>::raw*>(a.y) + t0 * a.yt;
    b.positions = a.positions + t0;
    const unsigned grid = static_cast<unsigned>((b.tokens * per_token + kThreads - 1) / kThreads);
    if (interleaved) rope_kernel<TYPE, V, true><<<grid, kThreads, 0, s>>>(b, chunks, rot_chunks);
    else rope_kernel<TYPE, V, false><<<grid, kThreads, 0, s>>>(b, chunks, rot_chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Table rows: the angle p w_i in 64 bits (f32 holds the angle of position 10^5
// to 0.008 only), its cosine and sine times the magnitude rounded once.
__global__ __launch_bounds__(kThreads) void rope_table_kernel(float* __restrict__ cosine,
                                                              float* __restrict__ sine,
                                                              long long first, long long count,
                                                              int half, RopeFrequencies f) {
  const long long step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long k = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; k < count * half;
       k += step) {
    const long long p = k / half;
    double sn, cs;
    sincos(static_cast<double>(first + p) * f.w[k - p * half], &sn, &cs);
    cosine[k] = static_cast<float>(f.magnitude * cs);
    sine[k] = static_cast<float>(f.magnitude * sn);
  }
}

}  // namespace

hipError_t launch_rope(const RopeLaunch& r, int* status, hipStream_t s) {
  RopeArgs a;
  a.x = r.x;
  a.y = r.y;
  a.xt = r.x_token;
  a.xh = r.x_head;
  a.yt = r.y_token;
  a.yh = r.y_head;
  a.cosine = r.cosine;
  a.sine = r.sine;
  a.positions = r.positions;
  a.max_position = static_cast<int>(r.max_position);
  a.heads = static_cast<int>(r.heads);
  a.rotary = static_cast<int>(r.rotary);
  a.head_dim = static_cast<int>(r.head_dim);
  a.tokens = static_cast<int>(r.tokens);
  a.status = status;
  const bool copy = r.x != r.y && r.rotary < r.head_dim;
  switch (r.type) {
    case QC_STORAGE_F32: return rope_typed<QC_STORAGE_F32>(a, r.interleaved, copy, s);
    case QC_STORAGE_F16: return rope_typed<QC_STORAGE_F16>(a, r.interleaved, copy, s);
    default: return rope_typed<QC_STORAGE_BF16>(a, r.interleaved, copy, s);
  }
}

hipError_t launch_rope_check(const int* positions, long long tokens, long long max_position,
                             int* flag, hipStream_t s) {
  const int grid = static_cast<int>(std::min<long long>((tokens + kThreads - 1) / kThreads, 1024));
  rope_check<<<grid, kThreads, 0, s>>>(positions, static_cast<int>(tokens),
                                       static_cast<int>(max_position), flag);
  return hipGetLastError();
}

hipError_t launch_rope_table(float* cosine, float* sine, long long first, long long count,
                             int half, const RopeFrequencies& f, hipStream_t s) {
  const long long work = count * half;
  const int grid = static_cast<int>(std::min<long long>((work + kThreads - 1) / kThreads, 1 << 16));
  rope_table_kernel<<<grid, kThreads, 0, s>>>(cosine, sine, first, count, half, f);
  return hipGetLastError();
}

}  // namespace qc
