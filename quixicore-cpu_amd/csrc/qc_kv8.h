// Shared by the 8-bit key/value cache's kernels: kv8_cache.hip (append,
// gather, checks) and kv8_attention.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qc_internal.h"

namespace qc {

// A call's cache and batch with the limits the host checked: pages, heads,
// page_tokens (a power of two, 16..256), head_dim (a multiple of 16, 16..256), seqs,
// columns, tokens, max_new and max_kv positive and within int.
struct Kv8Args {
  int8_t* k_codes;
  int8_t* v_codes;
  float* k_scales;
  float* v_scales;
  const int* table;
  const int* seq_start;
  const int* kv_len;
  int pages, kv_heads, page_tokens, page_shift, head_dim;
  int seqs, columns, tokens, max_new, max_kv;
  int* status;
};

Kv8Args kv8_args(const qc_kv8_cache& c, const qc_kv8_batch& b, int* status);

#ifdef __HIPCC__
// Sequence q's rows [first, first + rows) of the batch's tokens and its length;
// false (and status 3) where the device's figures do not fit the call's: such a
// sequence is left alone.
__device__ __forceinline__ bool kv8_sequence(const Kv8Args& a, int q, int& first, int& rows, int& kv) {
  first = a.seq_start[q];
  const int end = a.seq_start[q + 1];
  kv = a.kv_len[q];
  rows = end - first;
  const bool ok = first >= 0 && end >= first && end <= a.tokens && rows <= a.max_new && kv >= 0 &&
                  kv <= a.max_kv;
  if (!ok) *a.status = QC_INVALID_ARGUMENT;
  return ok;
}
#endif

}  // namespace qc
