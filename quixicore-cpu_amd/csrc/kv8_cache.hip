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

// Workgroup (page slot, head, K or V) of a sequence: the page's new tokens.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void append_kernel(Kv8Args a, Rows k, Rows v, int slots) {
  typedef typename Storage<TYPE>::raw raw;
  __shared__ float stop[kThreads / 64];
  __shared__ int sbad[kThreads / 64];
  long long id = blockIdx.x;
  const int which = id & 1;
  id >>= 1;
  const int head = id % a.kv_heads;
  id /= a.kv_heads;
  const int slot = id % slots;
  const int q = id / slots;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  const int begin = kv - rows;               // position of the first new token
  if (begin < 0) {
    *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const int column = (begin >> a.page_shift) + slot;
  const int p0 = column << a.page_shift;     // the page's first position
  const int lo = max(begin, p0), hi = min(kv, p0 + a.page_tokens);
  if (lo >= hi) return;
  const int page = a.table[static_cast<long long>(q) * a.columns + column];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) {
    *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const Rows src = which ? v : k;
  const long long unit = static_cast<long long>(page) * a.kv_heads + head;
  int8_t* codes = (which ? a.v_codes : a.k_codes) + unit * a.page_tokens * a.head_dim;
  float* scale_at = (which ? a.v_scales : a.k_scales) + unit;
  const raw* x = static_cast<const raw*>(src.p) + (first + lo - begin) * src.stride +
                 static_cast<long long>(head) * a.head_dim;
  const int n = (hi - lo) * a.head_dim;
  float top = 0.f;
  int bad = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / a.head_dim;
    const float f = decode<TYPE>(x[t * src.stride + i - t * a.head_dim]);
    bad |= !isfinite(f);
    top = fmaxf(top, fabsf(f));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  bad = __any(bad);
  if ((threadIdx.x & 63) == 0) {
    stop[threadIdx.x >> 6] = top;
    sbad[threadIdx.x >> 6] = bad;
  }
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) {
    top = fmaxf(top, stop[w]);
    bad |= sbad[w];
  }
  if (bad) {
    if (threadIdx.x == 0) *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const float before = lo > p0 ? *scale_at : 0.f;
  if (!isfinite(before)) {
    if (threadIdx.x == 0) *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  float scale = fmaxf(before, top * (1.0f / 127.0f));
  if (scale < 1.17549435e-38f) scale = 0.f;
  const float inv = scale > 0.f ? 1.0f / scale : 0.f;
  const float ratio = scale > 0.f ? before / scale : 0.f;
  if (lo > p0 && ratio != 1.0f) {
    const int m = (lo - p0) * a.head_dim;
    for (int i = threadIdx.x; i < m; i += kThreads)
      codes[i] = static_cast<int8_t>(fminf(fmaxf(rintf(static_cast<float>(codes[i]) * ratio), -127.f), 127.f));
  }
  int8_t* out = codes + (lo - p0) * a.head_dim;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / a.head_dim;
    const float f = decode<TYPE>(x[t * src.stride + i - t * a.head_dim]);
    out[i] = static_cast<int8_t>(fminf(fmaxf(rintf(f * inv), -127.f), 127.f));
  }
  __syncthreads();                            // every wave has read the scale before
  if (threadIdx.x == 0) *scale_at = scale;
}

// The same places read back: code * scale, rounded once.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void gather_kernel(Kv8Args a, void* k, void* v,
                                                          long long k_stride, long long v_stride,
                                                          int slots) {
  typedef typename Storage<TYPE>::raw raw;
  long long id = blockIdx.x;
  const int which = id & 1;
  id >>= 1;
  const int head = id % a.kv_heads;
  id /= a.kv_heads;
  const int slot = id % slots;
  const int q = id / slots;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  const int begin = kv - rows;
  if (begin < 0) {
    *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const int column = (begin >> a.page_shift) + slot;
  const int p0 = column << a.page_shift;
  const int lo = max(begin, p0), hi = min(kv, p0 + a.page_tokens);
  if (lo >= hi) return;
  const int page = a.table[static_cast<long long>(q) * a.columns + column];
  if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) {
    *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const long long unit = static_cast<long long>(page) * a.kv_heads + head;
  const int8_t* codes = (which ? a.v_codes : a.k_codes) +
                        (unit * a.page_tokens + lo - p0) * a.head_dim;
  const float scale = (which ? a.v_scales : a.k_scales)[unit];
  const long long stride = which ? v_stride : k_stride;
  raw* out = static_cast<raw*>(which ? v : k) + (first + lo - begin) * stride +
             static_cast<long long>(head) * a.head_dim;
  const int n = (hi - lo) * a.head_dim;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int t = i / a.head_dim;
    out[t * stride + i - t * a.head_dim] = encode<TYPE>(static_cast<float>(codes[i]) * scale);
  }
}

// The figures and table entries that a call goes by.  from_new: it touches the
// new tokens' pages; else the pages that its queries see (window: see
// qc_hip_kv8_attention), and their scales are finite.
__global__ __launch_bounds__(kThreads) void kv8_check(Kv8Args a, bool from_new, int window) {
  const int q = blockIdx.x;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  if (rows == 0) return;
  if (from_new && rows > kv) *a.status = QC_INVALID_ARGUMENT;
  const int from = from_new ? max(kv - rows, 0) : window > 0 ? max(kv - rows + 1 - window, 0) : 0;
  for (int c = (from >> a.page_shift) + threadIdx.x; c < (kv + a.page_tokens - 1) >> a.page_shift;
       c += kThreads) {
    const int page = a.table[static_cast<long long>(q) * a.columns + c];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) {
      *a.status = QC_INVALID_ARGUMENT;
      continue;
    }
    if (from_new) continue;
    for (int h = 0; h < a.kv_heads; ++h) {
      const long long at = static_cast<long long>(page) * a.kv_heads + h;
      if (!isfinite(a.k_scales[at]) || !isfinite(a.v_scales[at])) *a.status = QC_INVALID_ARGUMENT;
    }
  }
}

// *flag = 3 where a row of the batch's sequences holds NaN or +-inf.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void kv8_nonfinite(Kv8Args a, Rows k, Rows v) {
  typedef typename Storage<TYPE>::raw raw;
  const int q = blockIdx.x >> 1;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  const Rows src = blockIdx.x & 1 ? v : k;
  const int row = a.kv_heads * a.head_dim;
  for (int t = 0; t < rows; ++t)
    for (int i = threadIdx.x; i < row; i += kThreads)
      if (!isfinite(decode<TYPE>(static_cast<const raw*>(src.p)[(first + t) * src.stride + i])))
        *a.status = QC_INVALID_ARGUMENT;
}

// Pages that max_new tokens in a row can touch.
int touched_slots(const Kv8Args& a) { return (a.max_new + a.page_tokens - 2) / a.page_tokens + 1; }

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
  a.max_new = static_cast<int>(b.max_new);
  a.max_kv = static_cast<int>(b.max_kv);
  a.status = status;
  return a;
}

hipError_t launch_kv8_check(const qc_kv8_cache& c, const qc_kv8_batch& b, bool from_new, int window,
                            int* flag, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, flag);
  kv8_check<<<a.seqs, kThreads, 0, s>>>(a, from_new, window);
  return hipGetLastError();
}

hipError_t launch_kv8_nonfinite(const qc_kv8_cache& c, const qc_kv8_batch& b, const void* k,
                                long long k_stride, const void* v, long long v_stride, int type,
                                int* flag, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, flag);
  const Rows kr = {k, k_stride}, vr = {v, v_stride};
  const unsigned grid = 2u * static_cast<unsigned>(a.seqs);
  switch (type) {
    case QC_STORAGE_F32: kv8_nonfinite<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a, kr, vr); break;
    case QC_STORAGE_F16: kv8_nonfinite<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a, kr, vr); break;
    default: kv8_nonfinite<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a, kr, vr);
  }
  return hipGetLastError();
}

hipError_t launch_kv8_append(const qc_kv8_cache& c, const qc_kv8_batch& b, const void* k,
                             long long k_stride, const void* v, long long v_stride, int type,
                             int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, status);
  const int slots = touched_slots(a);
  const unsigned grid = static_cast<unsigned>(2LL * a.kv_heads * slots * a.seqs);
  const Rows kr = {k, k_stride}, vr = {v, v_stride};
  switch (type) {
    case QC_STORAGE_F32: append_kernel<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a, kr, vr, slots); break;
    case QC_STORAGE_F16: append_kernel<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a, kr, vr, slots); break;
    default: append_kernel<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a, kr, vr, slots);
  }
  return hipGetLastError();
}

hipError_t launch_kv8_gather(const qc_kv8_cache& c, const qc_kv8_batch& b, void* k,
                             long long k_stride, void* v, long long v_stride, int type, int* status,
                             hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, status);
  const int slots = touched_slots(a);
  const unsigned grid = static_cast<unsigned>(2LL * a.kv_heads * slots * a.seqs);
  switch (type) {
    case QC_STORAGE_F32:
      gather_kernel<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a, k, v, k_stride, v_stride, slots);
      break;
    case QC_STORAGE_F16:
      gather_kernel<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a, k, v, k_stride, v_stride, slots);
      break;
    default:
      gather_kernel<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a, k, v, k_stride, v_stride, slots);
  }
  return hipGetLastError();
}

}  // namespace qc
