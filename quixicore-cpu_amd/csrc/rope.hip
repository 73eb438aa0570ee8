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

// Position of a token and whether its heads are rotated: not at -1 (padding) and
// not where there is no table row (an error).
__device__ __forceinline__ bool position_of(const RopeArgs& a, uint32_t token, bool tell, int& p) {
  p = a.positions[token];
  if (static_cast<unsigned>(p) < static_cast<unsigned>(a.max_position)) return true;
  if (p != -1 && tell) *a.status = QC_INVALID_ARGUMENT;
  return false;
}

// One thread per token, head and V pairs (V elements past the rotated part, which
// are copied where y is another array than x): any strides and alignment.
template <int TYPE, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_any(RopeArgs a, int chunks, int rot_chunks) {
  typedef typename Storage<TYPE>::raw raw;
  const uint32_t per_token = static_cast<uint32_t>(a.heads) * chunks;
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t token = id / per_token;
  if (token >= static_cast<uint32_t>(a.tokens)) return;
  const uint32_t rest = id - token * per_token;
  const int head = rest / chunks, chunk = rest - head * chunks;
  int p;
  if (!position_of(a, token, rest == 0, p)) return;
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

// The same in 16-byte accesses (every chunk of V = 16 bytes' elements aligned, V
// dividing rotary / 2, or rotary if interleaved, and the part that is copied): a
// thread holds one chunk's cosines and sines for H heads.  The half layout's chunk is V
// pairs in two vectors, the interleaved one's V / 2 pairs in one.
//
// Bound by memory: 8192 x 40 heads of 128 f32, 64 rotated (336 MB), 124 us as
// rope_any with V = 4, 66 here (5.1 TB/s).  H = 4 takes a quarter of the table reads (they
// are 2 to 4 times a head's bytes, from L1 and L2) and keeps 4 to 8 loads in flight; with few
// tokens its threads are too few to fill the chip and H = 1 is the faster (16 tokens: a
// launch's time either way).
template <int TYPE, bool INTERLEAVED, int H>
__global__ __launch_bounds__(kThreads) void rope_wide(RopeArgs a, int chunks, int rot_chunks) {
  typedef typename Storage<TYPE>::raw raw;
  constexpr int V = Storage<TYPE>::per16;
  constexpr int P = INTERLEAVED ? V / 2 : V;      // pairs of a chunk
  constexpr int N = INTERLEAVED ? 1 : 2;          // vectors of it
  const int groups = (a.heads + H - 1) / H;
  const uint32_t per_token = static_cast<uint32_t>(groups) * chunks;
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t token = id / per_token;
  if (token >= static_cast<uint32_t>(a.tokens)) return;
  const uint32_t rest = id - token * per_token;
  const int group = rest / chunks, chunk = rest - group * chunks;
  int p;
  if (!position_of(a, token, rest == 0, p)) return;
  const int h0 = group * H;
  const raw* x = static_cast<const raw*>(a.x) + token * a.xt + h0 * a.xh;
  raw* y = static_cast<raw*>(a.y) + token * a.yt + h0 * a.yh;
  const bool copy = chunk >= rot_chunks;
  const int d = copy ? a.rotary + (chunk - rot_chunks) * V : chunk * V;
  const int half = a.rotary / 2;
  const int gap = copy ? 0 : half;                // half layout: the second vector's distance
  u32x4 w[H][N];
#pragma unroll
  for (int h = 0; h < H; ++h)
    if (h0 + h < a.heads) {
#pragma unroll
      for (int n = 0; n < N; ++n) w[h][n] = *reinterpret_cast<const u32x4*>(x + h * a.xh + d + n * gap);
    }
  if (copy) {
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (h0 + h < a.heads) *reinterpret_cast<u32x4*>(y + h * a.yh + d) = w[h][0];
    return;
  }
  const long long row = static_cast<long long>(p) * half + chunk * P;
  float c[P], s[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    c[i] = a.cosine[row + i];
    s[i] = a.sine[row + i];
  }
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (h0 + h >= a.heads) break;
    float v[N][V], o[N][V];
#pragma unroll
    for (int n = 0; n < N; ++n) decode16<TYPE>(w[h][n], v[n]);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      if constexpr (INTERLEAVED) {
        o[0][2 * i] = v[0][2 * i] * c[i] - v[0][2 * i + 1] * s[i];
        o[0][2 * i + 1] = v[0][2 * i + 1] * c[i] + v[0][2 * i] * s[i];
      } else {
        o[0][i] = v[0][i] * c[i] - v[N - 1][i] * s[i];
        o[N - 1][i] = v[N - 1][i] * c[i] + v[0][i] * s[i];
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
      *reinterpret_cast<u32x4*>(y + h * a.yh + d + n * gap) = encode16<TYPE>(o[n]);
  }
}

// Any position outside [-1, max_position): *flag = 3.
__global__ __launch_bounds__(kThreads) void rope_check(const int* __restrict__ positions,
                                                       int tokens, int max_position, int* flag) {
  for (int t = blockIdx.x * kThreads + threadIdx.x; t < tokens; t += gridDim.x * kThreads)
    if (positions[t] < -1 || positions[t] >= max_position) *flag = QC_INVALID_ARGUMENT;
}

template <int TYPE, bool INTERLEAVED>
hipError_t rope_typed(const RopeArgs& a, bool copy, hipStream_t s) {
  constexpr int V = Storage<TYPE>::per16, kAny = 4;
  const int pairs = a.rotary / 2;
  const auto whole = [](long long n) { return n % V == 0; };
  const bool wide = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.y)) & 15) == 0 &&
                    whole(a.xt) && whole(a.xh) && whole(a.yt) && whole(a.yh) &&
                    whole(INTERLEAVED ? a.rotary : pairs) && (!copy || whole(a.head_dim - a.rotary));
  const int per = wide ? (INTERLEAVED ? V / 2 : V) : kAny;
  const int rot_chunks = (pairs + per - 1) / per;
  const int tail = wide ? V : kAny;
  const int chunks = rot_chunks + (copy ? (a.head_dim - a.rotary + tail - 1) / tail : 0);
  const bool four = wide && static_cast<long long>(a.tokens) * a.heads * chunks >= 4LL * 1024 * device_cu_count();
  const int groups = four ? (a.heads + 3) / 4 : a.heads;
  const long long per_token = static_cast<long long>(groups) * chunks;
  // ids are 32-bit: slices of tokens
  const long long slice = std::max<long long>(1, (1LL << 30) / per_token);
  for (long long t0 = 0; t0 < a.tokens; t0 += slice) {
    RopeArgs b = a;
    b.tokens = static_cast<int>(std::min(slice, a.tokens - t0));
    b.x = static_cast<const typename Storage<TYPE>::raw*>(a.x) + t0 * a.xt;
    b.y = static_cast<typename Storage<TYPE>::raw*>(a.y) + t0 * a.yt;
    b.positions = a.positions + t0;
    const unsigned grid = static_cast<unsigned>((b.tokens * per_token + kThreads - 1) / kThreads);
    if (four) rope_wide<TYPE, INTERLEAVED, 4><<<grid, kThreads, 0, s>>>(b, chunks, rot_chunks);
    else if (wide) rope_wide<TYPE, INTERLEAVED, 1><<<grid, kThreads, 0, s>>>(b, chunks, rot_chunks);
    else rope_any<TYPE, kAny, INTERLEAVED><<<grid, kThreads, 0, s>>>(b, chunks, rot_chunks);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int TYPE>
hipError_t rope_layout(const RopeArgs& a, bool interleaved, bool copy, hipStream_t s) {
  return interleaved ? rope_typed<TYPE, true>(a, copy, s) : rope_typed<TYPE, false>(a, copy, s);
}

// Table rows: the angle p w_i in 64 bits (f32 holds the angle of position 10^5
// to 0.008 only), its cosine and sine times the magnitude rounded once.  A thread
// takes kRun positions of a pair: the first from sincos, the others turned on by (cos w,
// sin w), each turn within 2^-52.  131072 positions of 32 pairs: 22 us with a sincos
// each, 9 so: 3 for the launch and the two sincos before the first store, then 34 MB at 5.8 TB/s.
constexpr int kRun = 16;
__global__ __launch_bounds__(kThreads) void rope_table_kernel(float* __restrict__ cosine,
                                                              float* __restrict__ sine,
                                                              long long first, long long count,
                                                              int half, RopeFrequencies f) {
  const long long runs = (count + kRun - 1) / kRun, step = static_cast<long long>(gridDim.x) * kThreads;
  for (long long k = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; k < runs * half;
       k += step) {
    const long long p0 = k / half * kRun;
    const int i = static_cast<int>(k % half);
    const double w = f.w[i];
    double sn, cs, dsn, dcs;
    sincos(static_cast<double>(first + p0) * w, &sn, &cs);
    sincos(w, &dsn, &dcs);
    const int n = static_cast<int>(count - p0 < kRun ? count - p0 : kRun);
    for (int j = 0; j < n; ++j) {
      const long long at = (p0 + j) * half + i;
      cosine[at] = static_cast<float>(f.magnitude * cs);
      sine[at] = static_cast<float>(f.magnitude * sn);
      const double c = cs;
      cs = c * dcs - sn * dsn;
      sn = sn * dcs + c * dsn;
    }
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
    case QC_STORAGE_F32: return rope_layout<QC_STORAGE_F32>(a, r.interleaved, copy, s);
    case QC_STORAGE_F16: return rope_layout<QC_STORAGE_F16>(a, r.interleaved, copy, s);
    default: return rope_layout<QC_STORAGE_BF16>(a, r.interleaved, copy, s);
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
  const long long work = (count + kRun - 1) / kRun * half;
  const int grid = static_cast<int>(std::min<long long>((work + kThreads - 1) / kThreads, 1 << 16));
  rope_table_kernel<<<grid, kThreads, 0, s>>>(cosine, sine, first, count, half, f);
  return hipGetLastError();
}

}  // namespace qc
