// Shared by the 8-bit key/value cache's kernels: kv8_cache.hip (append,
// gather, checks) and kv8_attention.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qc_internal.h"

namespace qc {

// A call's cache and batch with the limits the host checked: pages, heads,
// page_tokens (a power of two, 16..256), head_dim (a multiple of 16, 16..256), seqs,
// columns, tokens, max_new (at most tokens) and max_kv positive and within int.
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

// A launch's work-items are counted in 32 bits.
inline bool kv8_grid_fits(long long groups, int threads) {
  return groups >= 0 && groups <= static_cast<long long>(UINT32_MAX) / threads;
}

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

// Work of a ragged batch, listed.  A grid padded to the longest sequence's blocks is
// mostly empty workgroups where the others are shorter (and those between the ones with
// work leave them on few of the shader engines that a grid is dealt to in turn), so such a
// batch's grid is what its tokens allow at most, and a workgroup finds its place by a scan.
//
// With count(rows, kv) blocks of each sequence: the sequence that has the b-th
// of all, b's place in it and the number of sequences before it that have any.  Every lane of
// the wavefront takes part, with the same b.  The first workgroup looks at every sequence, so that
// a bad one is told of.
struct Kv8Listed {
  int seq, at, before;
};
template <class Count>
__device__ __forceinline__ bool kv8_find(const Kv8Args& a, int b, Kv8Listed& out, Count&& count) {
  b = __builtin_amdgcn_readfirstlane(b);
  const int lane = threadIdx.x & 63;
  bool found = false;
  int before = 0;
  for (int base = 0; base < a.seqs; base += 64) {
    int n = 0, first, rows, kv;
    if (base + lane < a.seqs && kv8_sequence(a, base + lane, first, rows, kv) && rows > 0) n = count(rows, kv);
    int sum = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(sum, o);
      if (lane >= o) sum += below;
    }
    const uint64_t past = __ballot(sum > b), some = __ballot(n > 0);
    if (past != 0 && !found) {
      const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
      out.seq = base + l;
      out.at = b - __builtin_amdgcn_readlane(sum - n, l);
      out.before = before + __popcll(some & ((1ull << l) - 1));
      found = out.at >= 0;
      if (blockIdx.x != 0) return found;
    }
    b -= __builtin_amdgcn_readlane(sum, 63);
    before += __popcll(some);
  }
  return found;
}
#endif

// Whether a batch of at most `there` blocks is listed: not where the padded grid is about as
// large, whose workgroups need no scan.
inline bool kv8_listed(long long padded, long long there) { return 2 * padded > 3 * there; }

}  // namespace qc
