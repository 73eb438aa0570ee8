// The accepted ones of a sequence's drafted tokens close up in the 8-bit cache on gfx950.
//
// Of a sequence with c tokens before its n drafted ones, the drafted tokens p_0 < p_1 < .. <
// p_(m-1) stay: token p_a moves from position c + p_a to c + a.  A page and head that
// receives tokens of other pages takes the scale s' = the largest magnitude among its own
// scale and those pages'; codes that come under it, and those held, become rint(code * (s /
// s')), s the scale they had, ratio and product rounded to f32.  Without such tokens the codes move
// as they are.
#include "qc_kv8.h"

namespace qc {
namespace {

constexpr int kThreads = 256;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 16 codes times a ratio.
__device__ __forceinline__ u32x4 turned_codes(u32x4 w, float ratio) {
  if (ratio == 1.0f) return w;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t o = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float v = rintf(static_cast<float>(static_cast<int8_t>(w[i] >> (8 * j))) * ratio);
      o |= (static_cast<int>(fminf(fmaxf(v, -127.f), 127.f)) & 0xFF) << (8 * j);
    }
    w[i] = o;
  }
  return w;
}

// A workgroup takes a sequence's keys or values of a head and moves codes in place, page after page: the token that comes to
// position c + a was behind it, so what a page or a later one gives is read before it is written over.  (A path staged whole
// in LDS would need no order of pages; not built.)  CHECK: looks only.
//
// Bound by dependent reads and barriers, a page after the other, not by its bytes: 64 sequences, up to 59 tokens of 8
// heads of 128 over pages of 16 (5.1 MB) 12.3 us, 16 sequences of up to 3 tokens 5.1.  Path and page ids kept in LDS from the
// look at them change nothing (12.2), codes asked for before the scale that they come under little (11.7).
template <bool CHECK>
__global__ __launch_bounds__(kThreads) void keep_kernel(Kv8Args a, const int* __restrict__ kept,
                                                        long long columns, const int* __restrict__ counts,
                                                        int* __restrict__ new_len) {
  __shared__ float s_top[kThreads / 64];
  const int tid = threadIdx.x, which = blockIdx.x & 1;
  const int head = (blockIdx.x >> 1) % a.kv_heads, q = (blockIdx.x >> 1) / a.kv_heads;
  int first, rows, kv;
  if (!kv8_sequence(a, q, first, rows, kv)) return;
  const int begin = kv - rows, n = counts[q];
  if (begin < 0 || n < 0 || n > columns || n > rows) {
    if (tid == 0) *a.status = QC_INVALID_ARGUMENT;
    return;
  }
  const int* path = kept + q * columns;
  const int* table = a.table + static_cast<long long>(q) * a.columns;
  int8_t* codes = which ? a.v_codes : a.k_codes;
  float* scales = which ? a.v_scales : a.k_scales;
  auto unit = [&](int column) { return static_cast<long long>(table[column]) * a.kv_heads + head; };

  // the path, and the pages and scales of what moves; the first `still` tokens stay where they are
  int still = 0;
  bool bad = false, broken = false;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + tid;
    bool same = false;
    if (i < n) {
      const int p = path[i];
      const bool in = p > (i > 0 ? path[i - 1] : -1) && p < rows;
      bad = bad || !in;
      same = p == i;
      if (in && !same) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int column = (begin + (j ? p : i)) >> a.page_shift;
          const int page = table[column];
          if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) bad = true;
          else broken = broken || !isfinite(scales[static_cast<long long>(page) * a.kv_heads + head]);
        }
      }
    }
    still += __syncthreads_count(same);
  }
  bad = __syncthreads_or(bad);
  broken = __syncthreads_or(broken);
  if ((bad || broken) && tid == 0) *a.status = QC_INVALID_ARGUMENT;
  if (CHECK || bad) return;
  if (tid == 0 && (blockIdx.x >> 1) % a.kv_heads == 0 && which == 0) new_len[q] = begin + n;
  if (broken) return;

  const int per_row = a.head_dim / 16;
  for (int i = still; i < n;) {
    const int column = (begin + i) >> a.page_shift, p0 = column << a.page_shift;
    const int end = min(n, p0 + a.page_tokens - begin);   // tokens [i, end) come to this page
    const long long to = unit(column);
    const float held = scales[to];
    float top = -1.f;                                     // of pages that tokens come from, if any
    for (int j = i + tid; j < end; j += kThreads) {
      const int from = (begin + path[j]) >> a.page_shift;
      if (from != column) top = fmaxf(top, fabsf(scales[unit(from)]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((tid & 63) == 0) s_top[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, s_top[w]);
    const float scale = top < 0.f ? held : fmaxf(top, fabsf(held));
    auto ratio_of = [&](float s) { return s == scale ? 1.0f : scale != 0.f ? s / scale : 0.f; };
    u32x4* page = reinterpret_cast<u32x4*>(codes + to * a.page_tokens * a.head_dim);
    const float turn = ratio_of(held);
    if (turn != 1.0f)
      for (int j = tid; j < (begin + i - p0) * per_row; j += kThreads) page[j] = turned_codes(page[j], turn);
    for (int j0 = 0; j0 < (end - i) * per_row; j0 += kThreads) {
      const int j = j0 + tid, t = j / per_row;
      const bool in = j < (end - i) * per_row;
      u32x4 w = {0, 0, 0, 0};
      if (in) {
        const int at = begin + path[i + t], from = at >> a.page_shift;
        const long long u = unit(from);
        w = *reinterpret_cast<const u32x4*>(codes + (u * a.page_tokens + (at & (a.page_tokens - 1))) * a.head_dim +
                                            16 * (j - t * per_row));
        w = turned_codes(w, from == column ? turn : ratio_of(scales[u]));
      }
      __syncthreads();   // everyone's are read
      if (in) page[(begin + i - p0) * per_row + j] = w;
    }
    // the scale held is read by all before the barrier of the codes
    if (tid == 0 && scale != held) scales[to] = scale;
    i = end;
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_kv8_keep(const qc_kv8_cache& c, const qc_kv8_batch& b, const int* kept, long long kept_columns,
                           const int* kept_count, int* new_len, bool check, int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(c, b, status);
  const long long grid = 2LL * a.kv_heads * a.seqs;
  if (!kv8_grid_fits(grid, kThreads)) return hipErrorInvalidValue;
  const unsigned g = static_cast<unsigned>(grid);
  if (check) keep_kernel<true><<<g, kThreads, 0, s>>>(a, kept, kept_columns, kept_count, new_len);
  else keep_kernel<false><<<g, kThreads, 0, s>>>(a, kept, kept_columns, kept_count, new_len);
  return hipGetLastError();
}

}  // namespace qc
