// The 8-bit key/value cache on gfx950: pages of tokens, per page and head an
// int8 matrix [page_tokens][head_dim] and one f32 scale; an element is
// code * scale.
//
// Append.  A page's scale only grows while the page fills: with the new tokens'
// largest magnitude t, s' = max(s, t * c), c the f32 nearest 1 / 127 (s = 0 where the page holds no
// tokens before the new ones; s' below 2^-126 counts as 0), the codes there
// become rint(code * (s / s')) and the new ones clamp(rint(x * (1 / s')), -127,
// 127), ties to even, each step rounded to f32.  So a call's codes are
// defined bit for bit, and a page that is filled token by token has been rounded
// at most once for each growth of its scale.
#include <algorithm>

#include "qc_kv8.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

constexpr int kThreads = 256;

struct Rows {
  const void* p;
  long long stride;   // elements between tokens
};

// What a workgroup of a grid over (sequence, touched page, head, K or V) works on:
// the page's new tokens, positions [lo, hi) of a page that starts at p0.  slots: pages
// of a sequence in the grid, 0 where those there are are listed (8192 new tokens beside
// 255 sequences of one, 8 heads of 128, pages of 16: append 452 us padded, 21 listed, gather 1290,
// 38).
struct Place {
  int which, head;
  int lo, hi, p0;
  int row;                 // token row of position lo
  long long unit;          // page * kv_heads + head; -1 where the page id is out of range
};

__device__ __forceinline__ bool place_of(const Kv8Args& a, int slots, Place& w) {
  int id = blockIdx.x;
  w.which = id & 1;
  id >>= 1;
  const int rest = id / a.kv_heads;
  w.head = id - rest * a.kv_heads;
  int q, slot, first, rows, kv;
  if (slots > 0) {
    q = rest / slots;
    slot = rest - q * slots;
  } else {
    Kv8Listed l;
    const bool found = kv8_find(a, rest, l, [&](int rows, int kv) {
      if (rows > kv) *a.status = QC_INVALID_ARGUMENT;
      return rows > kv ? 0 : ((kv - 1) >> a.page_shift) - ((kv - rows) >> a.page_shift) + 1;
    });
    if (!found) return false;
    q = l.seq;
    slot = l.at;
  }
  if (!kv8_sequence(a, q, first, rows, kv)) return false;
  const int begin = kv - rows;               // position of the first new token
  if (begin < 0) {
    *a.status = QC_INVALID_ARGUMENT;
    return false;
  }
  const int column = (begin >> a.page_shift) + slot;
  w.p0 = column << a.page_shift;
  w.lo = max(begin, w.p0);
  w.hi = min(kv, w.p0 + a.page_tokens);
  if (w.lo >= w.hi) return false;
  const int page = a.table[static_cast<long long>(q) * a.columns + column];
  const bool in = static_cast<unsigned>(page) < static_cast<unsigned>(a.pages);
  if (!in) *a.status = QC_INVALID_ARGUMENT;
  w.row = first + w.lo - begin;
  w.unit = in ? static_cast<long long>(page) * a.kv_heads + w.head : -1;
  return true;
}

__device__ __forceinline__ int code_of(float v) {
  return static_cast<int>(fminf(fmaxf(rintf(v), -127.f), 127.f));
}

// Chunks of V elements (VEC: 16 bytes of a row, aligned); the first kHeld of a thread
// stay in registers between the maximum and the codes, the others are read again
// (from L2).  A page and head is a chain of dependent reads (lengths, page id, rows, scale)
// with little data behind it, so many small workgroups: 64 threads where a page's
// head is at most 4096 elements.  7152 tokens of 8 heads of 128, f16, pages of 16 (29 MB of rows
// read, 15 of codes written): 39 us with an element a thread, 14.8 here: 3.0 TB/s, 1.7 times what the bytes
// take at a copy's rate, for that chain and the VALU (busy two thirds of the time).
constexpr int kHeld = 8;
template <int TYPE, int NT, bool VEC>
__global__ __launch_bounds__(NT) void append_kernel(Kv8Args a, Rows k, Rows v, int slots) {
  typedef typename Storage<TYPE>::raw raw;
  constexpr int V = VEC ? Storage<TYPE>::per16 : 4;
  __shared__ float stop[NT / 64];
  Place w;
  if (!place_of(a, slots, w) || w.unit < 0) return;
  const Rows src = w.which ? v : k;
  int8_t* codes = (w.which ? a.v_codes : a.k_codes) + w.unit * a.page_tokens * a.head_dim;
  float* scale_at = (w.which ? a.v_scales : a.k_scales) + w.unit;
  const raw* x = static_cast<const raw*>(src.p) + w.row * src.stride +
                 static_cast<long long>(w.head) * a.head_dim;
  const float before = w.lo > w.p0 ? *scale_at : 0.f;
  const int per_row = a.head_dim / V, n = (w.hi - w.lo) * per_row;
  auto load = [&](int i, float* f) {
    const int t = i / per_row;
    const raw* p = x + t * src.stride + (i - t * per_row) * V;
    if constexpr (VEC) {
      decode16<TYPE>(*reinterpret_cast<const u32x4*>(p), f);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = decode<TYPE>(p[j]);
    }
  };
  float held[kHeld][V], top = 0.f;
  auto see = [&](const float* f) {
#pragma unroll
    for (int j = 0; j < V; ++j) top = isfinite(f[j]) ? fmaxf(top, fabsf(f[j])) : INFINITY;
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = threadIdx.x + h * NT;
    if (i < n) load(i, held[h]);
  }
#pragma unroll
  for (int h = 0; h < kHeld; ++h)
    if (static_cast<int>(threadIdx.x) + h * NT < n) see(held[h]);
  for (int i = threadIdx.x + kHeld * NT; i < n; i += NT) {
    float f[V];
    load(i, f);
    see(f);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if constexpr (NT > 64) {
    if ((threadIdx.x & 63) == 0) stop[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) top = fmaxf(top, stop[i]);
  }
  if (top == INFINITY || !isfinite(before)) {
    if (threadIdx.x == 0) *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  float scale = fmaxf(before, top * (1.0f / 127.0f));
  if (scale < 1.17549435e-38f) scale = 0.f;
  const float inv = scale > 0.f ? 1.0f / scale : 0.f;
  const float ratio = scale > 0.f ? before / scale : 0.f;
  if (w.lo > w.p0 && ratio != 1.0f) {
    uint32_t* old = reinterpret_cast<uint32_t*>(codes);
    const int m = (w.lo - w.p0) * a.head_dim / 4;
    for (int i = threadIdx.x; i < m; i += NT) {
      const uint32_t c = old[i];
      uint32_t o = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o |= (code_of(static_cast<float>(static_cast<int8_t>(c >> (8 * j))) * ratio) & 0xFF) << (8 * j);
      old[i] = o;
    }
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + (w.lo - w.p0) * a.head_dim);
  auto put = [&](int i, const float* f) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      uint32_t o = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) o |= (code_of(f[4 * j + e] * inv) & 0xFF) << (8 * e);
      out[i * (V / 4) + j] = o;
    }
  };
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = threadIdx.x + h * NT;
    if (i < n) put(i, held[h]);
  }
  for (int i = threadIdx.x + kHeld * NT; i < n; i += NT) {
    float f[V];
    load(i, f);
    put(i, f);
  }
  // every wave has read the scale before: at the latest by the barrier above
  if (threadIdx.x == 0) *scale_at = scale;
}

// Which of the 64 token rows from t0 on belong to no sequence that has its tokens in the cache.
__device__ __forceinline__ uint64_t rows_of_none(const Kv8Args& a, int t0) {
  const int n = min(64, a.tokens - t0);
  uint64_t taken = n < 64 ? ~0ull << n : 0;
  for (int i = threadIdx.x & 63; i < a.seqs; i += 64) {
    int first, rows, kv;
    if (!kv8_sequence(a, i, first, rows, kv) || rows > kv) continue;
    const int lo = max(first - t0, 0), hi = min(first + rows - t0, 64);
    if (lo < hi) taken |= (~0ull >> (64 - (hi - lo))) << lo;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    taken |= static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(taken), o));
  return ~taken;
}

template <int TYPE, int NT, bool VEC>
__device__ __forceinline__ void zero_row(typename Storage<TYPE>::raw* p, int n) {
  constexpr int V = VEC ? Storage<TYPE>::per16 : 1;
  for (int i = threadIdx.x * V; i < n; i += NT * V) {
    if constexpr (VEC) *reinterpret_cast<u32x4*>(p + i) = u32x4{0, 0, 0, 0};
    else p[i] = 0;
  }
}

// The same places read back: code * scale, rounded once; eight codes a thread and step, kHeld
// loads ahead of the stores.  7152 tokens of 8 heads of 128 to f16, pages of 16 (15 MB read, 30
// written): 17 us with four codes and a load a step and 256 threads, 10.8 here (4.1 TB/s).
// rest: workgroups from it on, two for each 64 token rows (K and V), set those to zero that no
// sequence has; 0 where such rows stay as they are.  (A fill of all rows before the call: 6 us more, and
// as many of the host's.)
template <int TYPE, int NT, bool VEC>
__global__ __launch_bounds__(NT) void gather_kernel(Kv8Args a, void* k, void* v, long long k_stride,
                                                    long long v_stride, int slots, unsigned rest) {
  typedef typename Storage<TYPE>::raw raw;
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  if (rest > 0 && blockIdx.x >= rest) {
    const int which = (blockIdx.x - rest) & 1, t0 = (blockIdx.x - rest) / 2 * 64;
    uint64_t empty = rows_of_none(a, t0);
    raw* rows = static_cast<raw*>(which ? v : k);
    for (; empty != 0; empty &= empty - 1) {
      const int t = t0 + __ffsll(static_cast<unsigned long long>(empty)) - 1;
      zero_row<TYPE, NT, VEC>(rows + t * (which ? v_stride : k_stride), a.kv_heads * a.head_dim);
    }
    return;
  }
  Place w;
  if (!place_of(a, slots, w)) return;
  const long long stride = w.which ? v_stride : k_stride;
  raw* out = static_cast<raw*>(w.which ? v : k) + w.row * stride +
             static_cast<long long>(w.head) * a.head_dim;
  if (w.unit >= 0) {
    const u32x2* codes = reinterpret_cast<const u32x2*>(
        (w.which ? a.v_codes : a.k_codes) + (w.unit * a.page_tokens + w.lo - w.p0) * a.head_dim);
    const float scale = (w.which ? a.v_scales : a.k_scales)[w.unit];
    // looked at in the loop, where the codes are on their way (ahead of them: 0.2 us a call)
    float s = scale;
    const int per_row = a.head_dim / 8, n = (w.hi - w.lo) * per_row;
    for (int i0 = threadIdx.x; i0 < n; i0 += kHeld * NT) {
      u32x2 held[kHeld];
#pragma unroll
      for (int h = 0; h < kHeld; ++h)
        if (i0 + h * NT < n) held[h] = codes[i0 + h * NT];
      asm volatile("" : "+s"(s));
      if (!isfinite(s)) break;
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int i = i0 + h * NT;
        if (i >= n) break;
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          f[j] = static_cast<float>(static_cast<int8_t>(held[h][j >> 2] >> (8 * (j & 3)))) * s;
        const int t = i / per_row;
        raw* o = out + t * stride + (i - t * per_row) * 8;
        if constexpr (VEC) {
#pragma unroll
          for (int j = 0; j < 8; j += Storage<TYPE>::per16) *reinterpret_cast<u32x4*>(o + j) = encode16<TYPE>(f + j);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = encode<TYPE>(f[j]);
        }
      }
    }
    if (isfinite(scale)) return;
    if (threadIdx.x == 0) *a.status = QC_INVALID_ARGUMENT;
  }
  // a page that is not there, or without a scale
  if (rest == 0) return;
  for (int t = 0; t < w.hi - w.lo; ++t) zero_row<TYPE, NT, VEC>(out + t * stride, a.head_dim);
}

// The figures, table entries and scales that a call goes by: append and gather touch the new
// tokens' pages, attention those that its queries see (window: see qc_hip_kv8_attention).
// An append goes by the scales of pages that hold tokens before the new ones, the others by all.
__global__ __launch_bounds__(kThreads) void kv8_check(Kv8Args a, Kv8Call call, int window) {
  const int q = blockIdx.x;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  if (rows == 0) return;
  const bool attention = call == Kv8Call::kAttention;
  if (!attention && rows > kv) *a.status = QC_INVALID_ARGUMENT;
  const int from = !attention ? max(kv - rows, 0) : window > 0 ? max(kv - rows + 1 - window, 0) : 0;
  for (int c = (from >> a.page_shift) + threadIdx.x; c < (kv + a.page_tokens - 1) >> a.page_shift;
       c += kThreads) {
    const int page = a.table[static_cast<long long>(q) * a.columns + c];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) {
      *a.status = QC_INVALID_ARGUMENT;
      continue;
    }
    if (call == Kv8Call::kAppend && c << a.page_shift >= kv - rows) continue;
    for (int h = 0; h < a.kv_heads; ++h) {
      const long long at = static_cast<long long>(page) * a.kv_heads + h;
      if (!isfinite(a.k_scales[at]) || !isfinite(a.v_scales[at])) *a.status = QC_INVALID_ARGUMENT;
    }
  }
}

// *flag = 3 where a row of the batch's sequences holds NaN or +-inf; `parts` workgroups a
// sequence for K and V each.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void kv8_nonfinite(Kv8Args a, Rows k, Rows v, int parts) {
  typedef typename Storage<TYPE>::raw raw;
  const int part = (blockIdx.x >> 1) % parts, q = (blockIdx.x >> 1) / parts;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  const Rows src = blockIdx.x & 1 ? v : k;
  const int row = a.kv_heads * a.head_dim;
  for (int t = part; t < rows; t += parts)
    for (int i = threadIdx.x; i < row; i += kThreads)
      if (!isfinite(decode<TYPE>(static_cast<const raw*>(src.p)[(first + t) * src.stride + i])))
        *a.status = QC_INVALID_ARGUMENT;
}

// Pages that max_new tokens in a row can touch.
int touched_slots(const Kv8Args& a) { return (a.max_new + a.page_tokens - 2) / a.page_tokens + 1; }

// Workgroups over the touched pages and heads; slots: what place_of takes.
unsigned touched_grid(const Kv8Args& a, int& slots) {
  slots = touched_slots(a);
  const long long padded = static_cast<long long>(slots) * a.seqs;
  const long long there = a.tokens / a.page_tokens + 2LL * std::min(a.seqs, a.tokens);   // at most
  const bool listed = kv8_listed(padded, there);
  if (listed) slots = 0;
  return static_cast<unsigned>(2 * a.kv_heads * (listed ? there : padded));
}

}  // namespace

Kv8Args kv8_args(const qc_kv8_cache& c, const qc_kv8_batch& b, int* status) {
  Kv8Args a;
  a.k_codes = c.k_codes;
  a.v_codes = c.v_codes;
  a.k_scales = c.k_scales;
  a.v_scales = c.v_scales;
  a.table = b.block_table;
  a.seq_start = b.seq_start;
  a.kv_len = b.kv_len;
  a.pages = static_cast<int>(c.pages);
  a.kv_heads = static_cast<int>(c.kv_heads);
  a.page_tokens = static_cast<int>(c.page_tokens);
  a.page_shift = __builtin_ctz(a.page_tokens);
  a.head_dim = static_cast<int>(c.head_dim);
  a.seqs = static_cast<int>(b.seqs);
  a.columns = static_cast<int>(b.columns);
  a.tokens = static_cast<int>(b.tokens);
  a.max_new = static_cast<int>(std::min(b.max_new, b.tokens));
  a.max_kv = static_cast<int>(b.max_kv);
  a.status = status;
  return a;
}

hipError_t launch_kv8_check(const qc_kv8_cache& c, const qc_kv8_batch& b, Kv8Call call, int window,
                            int* flag, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, flag);
  if (!kv8_grid_fits(a.seqs, kThreads)) return hipErrorInvalidValue;
  kv8_check<<<a.seqs, kThreads, 0, s>>>(a, call, window);
  return hipGetLastError();
}

hipError_t launch_kv8_nonfinite(const qc_kv8_cache& c, const qc_kv8_batch& b, const void* k,
                                long long k_stride, const void* v, long long v_stride, int type,
                                int* flag, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, flag);
  const Rows kr = {k, k_stride}, vr = {v, v_stride};
  // (of many sequences under a loose bound each takes its rows in more turns)
  const int parts = std::min(touched_slots(a), std::max(1, (1 << 18) / a.seqs));
  if (!kv8_grid_fits(2LL * parts * a.seqs, kThreads)) return hipErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(2LL * parts * a.seqs);
  switch (type) {
    case QC_STORAGE_F32: kv8_nonfinite<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a, kr, vr, parts); break;
    case QC_STORAGE_F16: kv8_nonfinite<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a, kr, vr, parts); break;
    default: kv8_nonfinite<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a, kr, vr, parts);
  }
  return hipGetLastError();
}

namespace {

// Rows of 16-byte chunks (the heads of a row are multiples of 16 elements apart).
bool wide_rows(const void* p, long long stride, int size) {
  return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride * size)) % 16 == 0;
}

template <int TYPE>
hipError_t run_append(const Kv8Args& a, const Rows& k, const Rows& v, hipStream_t s) {
  constexpr int size = TYPE == QC_STORAGE_F32 ? 4 : 2;
  int slots;
  const unsigned grid = touched_grid(a, slots);
  const bool vec = wide_rows(k.p, k.stride, size) && wide_rows(v.p, v.stride, size);
  const bool small = std::min(a.max_new, a.page_tokens) * a.head_dim <= 4096;
  if (!kv8_grid_fits(grid, vec && small ? 64 : 256)) return hipErrorInvalidValue;
  if (vec && small) append_kernel<TYPE, 64, true><<<grid, 64, 0, s>>>(a, k, v, slots);
  else if (vec) append_kernel<TYPE, 256, true><<<grid, 256, 0, s>>>(a, k, v, slots);
  else append_kernel<TYPE, 256, false><<<grid, 256, 0, s>>>(a, k, v, slots);
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_gather(const Kv8Args& a, void* k, void* v, long long k_stride, long long v_stride, bool zero_rest,
                      hipStream_t s) {
  constexpr int size = TYPE == QC_STORAGE_F32 ? 4 : 2;
  int slots;
  unsigned grid = touched_grid(a, slots);
  const unsigned rest = zero_rest ? grid : 0;
  if (zero_rest) grid += 2u * static_cast<unsigned>((a.tokens + 63LL) / 64);
  const bool vec = wide_rows(k, k_stride, size) && wide_rows(v, v_stride, size);
  const bool small = std::min(a.max_new, a.page_tokens) * a.head_dim <= 4096;
  if (!kv8_grid_fits(grid, vec && small ? 64 : 256)) return hipErrorInvalidValue;
  if (vec && small) gather_kernel<TYPE, 64, true><<<grid, 64, 0, s>>>(a, k, v, k_stride, v_stride, slots, rest);
  else if (vec) gather_kernel<TYPE, 256, true><<<grid, 256, 0, s>>>(a, k, v, k_stride, v_stride, slots, rest);
  else gather_kernel<TYPE, 256, false><<<grid, 256, 0, s>>>(a, k, v, k_stride, v_stride, slots, rest);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_append(const qc_kv8_cache& c, const qc_kv8_batch& b, const void* k,
                             long long k_stride, const void* v, long long v_stride, int type,
                             int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, status);
  const Rows kr = {k, k_stride}, vr = {v, v_stride};
  switch (type) {
    case QC_STORAGE_F32: return run_append<QC_STORAGE_F32>(a, kr, vr, s);
    case QC_STORAGE_F16: return run_append<QC_STORAGE_F16>(a, kr, vr, s);
    default: return run_append<QC_STORAGE_BF16>(a, kr, vr, s);
  }
}

hipError_t launch_kv8_gather(const qc_kv8_cache& c, const qc_kv8_batch& b, void* k,
                             long long k_stride, void* v, long long v_stride, int type, bool zero_rest,
                             int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, status);
  switch (type) {
    case QC_STORAGE_F32: return run_gather<QC_STORAGE_F32>(a, k, v, k_stride, v_stride, zero_rest, s);
    case QC_STORAGE_F16: return run_gather<QC_STORAGE_F16>(a, k, v, k_stride, v_stride, zero_rest, s);
    default: return run_gather<QC_STORAGE_BF16>(a, k, v, k_stride, v_stride, zero_rest, s);
  }
}

}  // namespace qc
