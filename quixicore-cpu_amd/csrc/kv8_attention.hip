// Attention over the 8-bit key/value cache on gfx950.
//
// Query row (token i of a sequence of n new tokens and length L, head h) stands at
// position p = L - n + i and sees the keys j < L, with `causal` j <= p, with a
// window w also j > p - w.  out = sum_j softmax_j(scale q . k_j) v_j, in one pass over
// the keys: running maximum m and sum l of the exponentials, both f32, and the
// running sum of values, rescaled by exp(m_old - m_new) when m grows.  A row
// that sees no key is zeros.
#include "qc_kv8.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

constexpr int kThreads = 256;

// One wavefront per query row and head; a lane holds head_dim / 64 elements
// (rounded up), the wave walks over the keys.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void attention_simple(Kv8Args a, const void* qp,
                                                             long long q_stride, void* out,
                                                             long long out_stride, int heads,
                                                             float scale, int causal, int window) {
  typedef typename Storage<TYPE>::raw raw;
  const int lane = threadIdx.x & 63;
  const int s = blockIdx.y;
  int first, rows, kv;
  if (!kv8_sequence(a, s, first, rows, kv)) return;
  const long long item = static_cast<long long>(blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  const int i = static_cast<int>(item / heads), h = static_cast<int>(item % heads);
  if (i >= rows) return;
  const int kvh = h / (heads / a.kv_heads);
  const int pos = kv - rows + i;
  const int hi = causal ? min(kv, pos + 1) : kv;
  const int lo = window > 0 ? max(0, pos + 1 - window) : 0;
  const raw* q = static_cast<const raw*>(qp) + (first + i) * q_stride + static_cast<long long>(h) * a.head_dim;
  float qv[4], acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 64 * e;
    qv[e] = d < a.head_dim ? decode<TYPE>(q[d]) : 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = lo; j < hi; ++j) {
    const int page = a.table[static_cast<long long>(s) * a.columns + (j >> a.page_shift)];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pages)) {
      *a.status = QC_INVALID_ARGUMENT;
      continue;
    }
    const long long unit = static_cast<long long>(page) * a.kv_heads + kvh;
    const long long at = (unit * a.page_tokens + (j & (a.page_tokens - 1))) * a.head_dim;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      if (d < a.head_dim) dot = fmaf(qv[e], static_cast<float>(a.k_codes[at + d]), dot);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o);
    const float z = dot * (a.k_scales[unit] * scale);
    const float mn = fmaxf(m, z);
    const float alpha = expf(m - mn), p = expf(z - mn);
    l = l * alpha + p;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      const float v = d < a.head_dim ? static_cast<float>(a.v_codes[at + d]) * a.v_scales[unit] : 0.f;
      acc[e] = fmaf(p, v, acc[e] * alpha);
    }
    m = mn;
  }
  raw* y = static_cast<raw*>(out) + (first + i) * out_stride + static_cast<long long>(h) * a.head_dim;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 64 * e;
    if (d < a.head_dim) y[d] = encode<TYPE>(l == 0.f ? 0.f : acc[e] / l);
  }
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8Attention& r, int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(*r.cache, *r.batch, status);
  const long long items = static_cast<long long>(a.max_new) * r.heads;
  const dim3 grid(static_cast<unsigned>((items + kThreads / 64 - 1) / (kThreads / 64)), a.seqs);
  const int heads = static_cast<int>(r.heads), window = static_cast<int>(r.window);
  switch (r.type) {
    case QC_STORAGE_F32:
      attention_simple<QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a, r.q, r.q_stride, r.out, r.out_stride,
                                                                 heads, r.scale, r.causal, window);
      break;
    case QC_STORAGE_F16:
      attention_simple<QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a, r.q, r.q_stride, r.out, r.out_stride,
                                                                 heads, r.scale, r.causal, window);
      break;
    default:
      attention_simple<QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a, r.q, r.q_stride, r.out, r.out_stride,
                                                                  heads, r.scale, r.causal, window);
  }
  return hipGetLastError();
}

}  // namespace qc
