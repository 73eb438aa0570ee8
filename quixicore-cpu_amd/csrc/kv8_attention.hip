// Attention over the 8-bit key/value cache on gfx950.
//
// Query row (token i of a sequence of n new tokens and length L, head h) stands at
// position p = L - n + i and sees the keys j < L, with `causal` j <= p, with a
// window w also j > p - w.  out = sum_j softmax_j(scale q . k_j) v_j, in one pass over
// the keys: running maximum m and sum l of the exponentials, both f32, and the
// running sum of values, rescaled by exp(m_old - m_new) when m grows.  A row
// that sees no key is zeros.
//
// Codes are exact in f16, so both products run on f16 MFMA with the codes themselves, and
// the scales of a page stay outside: a page's key scale multiplies its scores, its value
// scale the probabilities that meet its codes.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "qc_kv8.h"
#include "qc_lds_dma.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896340736f;

// The rows of one sequence and key head: row r is token r / group, head
// kv_head * group + r % group.
struct Unit {
  int first, rows, kv;   // the sequence's first token row, new tokens, length
  __device__ __forceinline__ int position(int token) const { return kv - rows + token; }
};

struct AttnArgs {
  const void* q;
  void* out;
  long long q_stride, out_stride;
  int heads, group;
  float scale;
  int causal, window;
  int vec;              // q and out rows allow 16-byte accesses
  float* part;          // [split][tokens * heads][head_dim], then statistics
  float* stats;         // [split][tokens * heads][2]: maximum (log2 units), sum
  int splits, chunk;    // key ranges, and tokens of one, at most
  int want, span;       // ranges to cut the keys into, at most; keys that a row block sees at most
  int per, row_blocks;  // rows of a row block, row blocks of a sequence's key head at most
  int rows_from, rows_to;   // sequences of [rows_from, rows_to) rows a key head are worked on
  int listed;           // what blocks are counted by: kPadded, kBlocks, kSequences
  int route;            // host: 0 by size, 1 / 2 one or two row tiles, 3 tiled
};

// How blocks are counted.  kPadded: every sequence has row_blocks of them.  kBlocks:
// only those there are.  kSequences: one for each sequence with rows in range.  us, 32 / 8
// heads of 128, bf16: 256 new tokens beside 127 sequences of one, 1000 to 2000 keys, 1907
// padded, 118 listed.
enum { kPadded, kBlocks, kSequences };

__device__ __forceinline__ bool find_listed(const Kv8Args& a, const AttnArgs& p, int b, Kv8Listed& out) {
  return kv8_find(a, b, out, [&](int rows, int) {
    const int all = rows * p.group;
    if (all < p.rows_from || all >= p.rows_to) return 0;
    return p.listed == kBlocks ? (all + p.per - 1) / p.per : 1;
  });
}

// What block `id` of a grid over row blocks is: the same for a whole wavefront where
// the grid is listed.
__device__ __forceinline__ bool block_of(const Kv8Args& a, const AttnArgs& p, int id, int& seq, int& kvh, int& rb) {
  if (p.listed == kPadded) {
    rb = id % p.row_blocks;
    id /= p.row_blocks;
    kvh = id % a.kv_heads;
    seq = id / a.kv_heads;
    return true;
  }
  kvh = id % a.kv_heads;
  Kv8Listed l;
  const bool found = find_listed(a, p, id / a.kv_heads, l);
  seq = l.seq;
  rb = l.at;
  return found;
}

// Keys [lo, hi) that rows of tokens t0..t1 (inclusive) see together.
__device__ __forceinline__ void seen_range(const AttnArgs& p, const Unit& u, int t0, int t1, int& lo,
                                           int& hi) {
  hi = p.causal ? min(u.kv, u.position(t1) + 1) : u.kv;
  lo = p.window > 0 ? max(0, u.position(t0) + 1 - p.window) : 0;
}

// The most keys of a sequence with rows; for all lanes.
__device__ __forceinline__ int longest(const Kv8Args& a) {
  int n = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < a.seqs; i += 64) {
    const int kv = a.kv_len[i];
    if (a.seq_start[i + 1] > a.seq_start[i] && kv <= a.max_kv) n = max(n, kv);
  }
  // lanes 1, 2, then 4 and 8 (mirrors) away, then the rows of 16
  n = max(n, __builtin_amdgcn_update_dpp(0, n, 0xB1, 0xF, 0xF, true));
  n = max(n, __builtin_amdgcn_update_dpp(0, n, 0x4E, 0xF, 0xF, true));
  n = max(n, __builtin_amdgcn_update_dpp(0, n, 0x141, 0xF, 0xF, true));
  n = max(n, __builtin_amdgcn_update_dpp(0, n, 0x140, 0xF, 0xF, true));
  const auto r = __builtin_amdgcn_permlane16_swap(n, n, false, false);
  n = max(static_cast<int>(r[0]), static_cast<int>(r[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(n, n, false, false);
  return __builtin_amdgcn_readfirstlane(max(static_cast<int>(h[0]), static_cast<int>(h[1])));
}

// Keys of a range, from the batch's longest sequence and not from the host's bound, which a captured step
// has far above its lengths (8 sequences of 16384 keys, 32 / 8 heads of 128, bound 131072: 192 us with
// ranges cut from the bound, 51 so, 49 with the bound at the length).  used: ranges that hold keys.  All
// keys are covered: n <= splits * chunk, want <= splits; `least` and chunk are multiples of `step`.  (Where the
// blocks alone fill the chip, want is 1 and ranges are cut for LDS only: nothing to look up.)
__device__ __forceinline__ int range_keys(const Kv8Args& a, const AttnArgs& p, int least, int step, int& used) {
  used = p.splits;
  if (p.chunk <= least || p.splits == 1 || p.want == 1) return p.chunk;
  const int n = min(longest(a), p.span);
  if (n == p.span) return p.chunk;
  const int keys = min(max(least, ((n + p.want - 1) / p.want + step - 1) / step * step), p.chunk);
  used = max(1, (n + keys - 1) / keys);
  return keys;
}

// Four signed bytes as f16: 0x6400 | u is 1024 + u for a byte u, and u = code + 128.
__device__ __forceinline__ void bytes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const f16x2 bias = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + bias);
  hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + bias);
}

// Rows r[0..3] of four bytes each -> t[c] = {r[0][c], r[1][c], r[2][c], r[3][c]}.
__device__ __forceinline__ void transpose4(const uint32_t (&r)[4], uint32_t (&t)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const uint32_t c = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  t[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
  t[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
  t[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
  t[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Largest of three (fmaxf would first quiet each value that an MFMA wrote).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

// Maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float lanes16_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes16_sum(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Power of two that takes a row whose largest magnitude is `top` to [2^14, 2^15):
// elements down to 2^-28 of it keep their 11 bits in f16.  inverse: its inverse, NaN
// for a row that is not finite.
__device__ __forceinline__ float row_scale(float top, float& inverse) {
  if (!(top <= 3.402823466e38f)) {
    inverse = __uint_as_float(0x7FC00000u);
    return 1.0f;
  }
  int e = -100;
  if (top > 0.f) {
    (void)frexpf(top, &e);
    e = max(e, -100);
  }
  inverse = ldexpf(1.0f, e - 15);
  return ldexpf(1.0f, 15 - e);
}

// A value that all lanes hold, in a scalar register.
__device__ __forceinline__ float uniform(float v) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// unit = m 2^e of a workgroup's largest value scale, m 0 or in [1/2, 1).
__device__ __forceinline__ float split_unit(float unit, int& e) {
  const float m = frexpf(unit, &e);
  e = __builtin_amdgcn_readfirstlane(e);
  return uniform(m);
}

// Elements d, .., d + 7 of a q row (zeros at and past head_dim, a multiple of 16).
template <int TYPE>
__device__ __forceinline__ void load8(const void* q, long long at, bool in, bool vec, float* v) {
  typedef typename Storage<TYPE>::raw raw;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (!in) return;
  const raw* p = static_cast<const raw*>(q) + at;
  if (vec) {
    decode16<TYPE>(*reinterpret_cast<const u32x4*>(p), v);
    if constexpr (TYPE == QC_STORAGE_F32) decode16<TYPE>(*reinterpret_cast<const u32x4*>(p + 4), v + 4);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = decode<TYPE>(p[j]);
  }
}

// N consecutive elements of an out row.
template <int TYPE, int N>
__device__ __forceinline__ void store_n(void* out, long long at, bool vec, const float* v) {
  typedef typename Storage<TYPE>::raw raw;
  raw* p = static_cast<raw*>(out) + at;
  if (!vec) {
#pragma unroll
    for (int j = 0; j < N; ++j) p[j] = encode<TYPE>(v[j]);
  } else if constexpr (TYPE == QC_STORAGE_F32) {
#pragma unroll
    for (int j = 0; j < N; j += 4) *reinterpret_cast<u32x4*>(p + j) = encode16<TYPE>(v + j);
  } else if constexpr (N == 4) {
    *reinterpret_cast<u32x2*>(p) = u32x2{encode2<TYPE>(v[0], v[1]), encode2<TYPE>(v[2], v[3])};
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 8) *reinterpret_cast<u32x4*>(p + j) = encode16<TYPE>(v + j);
  }
}

// ---- Few rows a key head: the cache straight from memory -----------------------
//
// Workgroup = a range of keys, RT tiles of 16 rows of a key head, a sequence.  Its
// waves take the range's steps of 32 keys in turn, each with statistics and sums of its
// own, and join at the end through LDS; several ranges join in a second launch.
//
// S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_16x16x32_f16, so that a lane's scores
// and sums belong to one row (lane & 15): with g = lane >> 4, register e of key tile t is
// key 16 t + 4 g + e, and the products' K order is free, so the lane's own eight
// probabilities are its operand of the second product.  K: lane loads 16 bytes of key
// lane & 15 at dimension 64 c + 16 g.  V: lane loads DP / 16 bytes of its eight
// keys at dimension (DP / 16) (lane & 15), transposed in registers.
//
// Bound by memory where the cache is long: 32 sequences of 4096 to 16384 keys, 32 / 8 heads of 128,
// bf16 (711 MB), 143 to 151 us by session, 4.7 to 5.0 TB/s, and 3 to 5 for the join; one of 600 keys, f32, 7.9 and
// 2.8: a launch, then figures, page id, codes and the waves' join, each waiting for the one
// before.  A single workgroup of 8 or 16 waves in place of ranges and their join is slower
// (500 keys, bf16: 13.7 us against 10.0).
constexpr int kWaves = 4;
constexpr int kMaxGroups = 1024;   // 16-key groups of a range

template <int DP, int RT, int TYPE>
__global__ __launch_bounds__(64 * kWaves, RT == 1 && DP <= 128 && TYPE != QC_STORAGE_F32 ? 4 : 1) void attention_direct(Kv8Args a, AttnArgs p) {
  constexpr int KC = DP / 64;                     // 16-byte chunks of a key a lane holds
  constexpr int KS = DP / 32;                     // MFMAs of 32 dimensions
  constexpr int VB = DP / 16;                     // bytes of a value a lane holds
  constexpr int VW = VB / 4;
  constexpr int NQ = TYPE == QC_STORAGE_F32 ? 2 : 1;   // f16 terms of q
  // And of the probabilities: one rounded to 11 bits weighs as much as an f16 output's own
  // rounding, and the second term costs little beside the loads.  A bf16 output's is 8 times as
  // coarse: a second term would change its error against 64 bits by less than 1% (single outputs take the
  // next bf16 step) and cost 2% of decoding (32 x 16384 keys, 154 -> 157 us), 8 to 15% of prompts of 16 to 100 tokens.
  constexpr int NP = TYPE == QC_STORAGE_BF16 ? 1 : 2;
  __shared__ int s_page[kMaxGroups];
  __shared__ float s_ks[kMaxGroups], s_vs[kMaxGroups];
  __shared__ float s_red[kWaves], s_m[kWaves][RT * 16], s_l[kWaves][RT * 16];
  __shared__ f32x4 s_o[kWaves / 2][RT][VB][64];

  const int lane = threadIdx.x & 63, row16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Range fastest, then row block, key head, sequence; ranges past every length after all of these.
  // With blocks enough to fill the chip and an even number of ranges the range is slowest: workgroups are dealt to the
  // 8 XCDs in turn, and short sequences' empty ranges would leave some idle (128 sequences of up to 6000 keys, heads of
  // 64, 2 ranges, 141 -> 110 us; 3 ranges spread by themselves: 64 x 4 row blocks, 11832 keys, 183 -> 200; with fewer
  // blocks 32 x 16384 keys 154 -> 162, and row blocks that share keys on several XCDs).
  int used;
  const int chunk = range_keys(a, p, 32 * kWaves, 32, used);
  const bool slowest = p.want == 1 && (p.splits & 1) == 0;
  int id = blockIdx.x / used, split = blockIdx.x - id * used;
  if (slowest || used < p.splits) {
    const int blocks = gridDim.x / p.splits, first = slowest ? 0 : blocks * used;   // of the workgroups in that order
    if (static_cast<int>(blockIdx.x) >= first) {
      const int more = (blockIdx.x - first) / blocks;
      split = (slowest ? 0 : used) + more;
      id = blockIdx.x - first - more * blocks;
    }
  }
  int seq, kvh, rb;
  if (!block_of(a, p, id, seq, kvh, rb)) return;
  // Where a unit's row blocks lie side by side, the last ones of an even number, which short sequences lack, would
  // always be the same XCDs': exchanged from unit to unit, within the power of two that divides the number (64
  // sequences of 4 to 16 tokens, 8 blocks each, 2000 keys, 129 -> 111 us).
  if (p.listed == kPadded && (slowest || p.splits == 1)) rb ^= (seq * a.kv_heads + kvh) & ((p.row_blocks & -p.row_blocks) - 1);
  Unit u;
  if (!kv8_sequence(a, seq, u.first, u.rows, u.kv) || u.rows * p.group >= p.rows_to) return;
  const int r0 = rb * RT * 16, r1 = min(r0 + RT * 16, u.rows * p.group);
  if (r0 >= r1) return;
  int lo, hi;
  seen_range(p, u, r0 / p.group, (r1 - 1) / p.group, lo, hi);
  const int base = lo & ~31;
  const int from = __builtin_amdgcn_readfirstlane(base + split * chunk);   // a multiple of 32
  const int to = __builtin_amdgcn_readfirstlane(min(hi, from + chunk));
  if (from >= to && p.splits > 1) {               // a range without keys
    for (int r = r0 + threadIdx.x; r < r1; r += 64 * kWaves) {
      const int token = r / p.group, head = kvh * p.group + r - token * p.group;
      float* st = p.stats + 2 * ((static_cast<long long>(split) * a.tokens + u.first + token) * p.heads + head);
      st[0] = -INFINITY;
      st[1] = 0.f;
    }
    return;
  }
  const int groups = max(0, (to - from + 15) >> 4);
  const int* table = a.table + static_cast<long long>(seq) * a.columns;
  // the page of 16 keys, -1 where no row sees one of them; ids out of range are told apart below
  auto page_of = [&](int tok) { return tok < to && tok + 15 >= lo ? table[tok >> a.page_shift] : -1; };

  // Codes of 32 keys from tok.  A group without a page reads page 0 and counts for nothing,
  // lanes past head_dim read dimension 0: q is zero there, and sums there are not stored.
  u32x4 kr[2][KC];
  uint32_t vr8[8][VW];
  const int k_lane = row16 * a.head_dim + (16 * g < a.head_dim ? 16 * g : 0);
  const int v_lane = 4 * g * a.head_dim + (VB * row16 < a.head_dim ? VB * row16 : 0);
  int k_off[KC];
#pragma unroll
  for (int c = 0; c < KC; ++c) k_off[c] = 64 * c + 16 * g < a.head_dim ? 64 * c : 0;
  auto code_at = [&](int tok, int id) {
    id = __builtin_amdgcn_readfirstlane(id);
    const int page = static_cast<unsigned>(id) < static_cast<unsigned>(a.pages) ? id : 0;
    return ((static_cast<long long>(page) * a.kv_heads + kvh) * a.page_tokens + (tok & (a.page_tokens - 1))) * a.head_dim;
  };
  auto load_k = [&](long long at0, long long at1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int8_t* kp = a.k_codes + (t ? at1 : at0);
#pragma unroll
      for (int c = 0; c < KC; ++c) kr[t][c] = *reinterpret_cast<const u32x4*>(kp + k_lane + k_off[c]);
    }
  };
  auto load_v = [&](long long at0, long long at1) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int8_t* vp = a.v_codes + (t ? at1 : at0);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int8_t* q = vp + v_lane + e * a.head_dim;
        if constexpr (VW == 1) {
          vr8[4 * t + e][0] = *reinterpret_cast<const uint32_t*>(q);
        } else if constexpr (VW == 2) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(q);
          vr8[4 * t + e][0] = x[0];
          vr8[4 * t + e][1] = x[1];
        } else {
          const u32x4 x = *reinterpret_cast<const u32x4*>(q);
#pragma unroll
          for (int w = 0; w < 4; ++w) vr8[4 * t + e][w] = x[w];
        }
      }
    }
  };
  // the wave's first keys are on their way before anything is waited for
  const int stride = 32 * kWaves, tok0 = from + 32 * wave;
  if (tok0 < to) {
    const long long at0 = code_at(tok0, page_of(tok0)), at1 = code_at(tok0 + 16, page_of(tok0 + 16));
    load_k(at0, at1);
    load_v(at0, at1);
  }

  // page ids and scales of the range's groups of 16 keys, and the largest value scale
  float unit = 0.f;
  for (int i = threadIdx.x; i < groups; i += 64 * kWaves) {
    int page = page_of(from + 16 * i);
    float ks = 0.f, vs = 0.f;
    if (from + 16 * i + 15 >= lo) {
      bool ok = false;
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.pages)) {
        const long long at = static_cast<long long>(page) * a.kv_heads + kvh;
        ks = a.k_scales[at];
        vs = a.v_scales[at];
        ok = isfinite(ks) && isfinite(vs);
      }
      if (!ok) {
        *a.status = QC_INVALID_ARGUMENT;
        page = -1;
        ks = vs = 0.f;
      }
    }
    s_page[i] = page;
    s_ks[i] = ks;
    s_vs[i] = vs;
    unit = fmaxf(unit, fabsf(vs));
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) unit = fmaxf(unit, __shfl_xor(unit, o));
  if (lane == 0) s_red[wave] = unit;

  // q's fragments: row row16 of tile t, dimensions 64 c + 16 g + 8 h + j
  f16x8 qf[RT][KS][NQ];
  float factor[RT];                               // score's scale in log2 units, over q's
  int row_lo[RT], row_hi[RT];                     // keys the lane's row sees
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + 16 * t + row16;
    const bool has = r < r1;
    const int token = (has ? r : r0) / p.group, head = kvh * p.group + (has ? r : r0) - token * p.group;
    const long long at = (u.first + token) * p.q_stride + static_cast<long long>(head) * a.head_dim;
    float v[KS][8], top = 0.f;
    bool nan = false;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
      load8<TYPE>(p.q, at + d, has && d < a.head_dim, p.vec, v[s]);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(v[s][j]));
        nan = nan || v[s][j] != v[s][j];
      }
    if (nan) top = INFINITY;
    top = lanes16_max(top);
    float inverse;
    const float up = row_scale(top, inverse);
    factor[t] = p.scale * kLog2e * inverse;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = in_f32(v[s][j] * up);
        qf[t][s][0][j] = static_cast<_Float16>(x);
        if constexpr (NQ == 2) qf[t][s][1][j] = static_cast<_Float16>(x - static_cast<float>(qf[t][s][0][j]));
      }
    row_hi[t] = has ? (p.causal ? min(u.kv, u.position(token) + 1) : u.kv) : 0;
    row_lo[t] = p.window > 0 ? u.position(token) + 1 - p.window : 0;
  }
  // keys that every row of the block sees (its rows past r1 count for nothing whatever they see)
  int all_hi = hi, all_lo = lo;
  if (p.causal) all_hi = min(u.kv, u.position(r0 / p.group) + 1);
  if (p.window > 0) all_lo = u.position((r1 - 1) / p.group) + 1 - p.window;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) unit = fmaxf(unit, s_red[w]);
  // Probabilities enter the second product as p * (value scale / unit) * 2^15, the power of two
  // in either scale taken out first: 2^15 / unit alone is infinite from 9.6e-35 down.
  int unit_e;
  const float unit_m = split_unit(unit, unit_e);
  const float per_unit = uniform(unit > 0.f ? 32768.0f / unit_m : 0.f);

  float m[RT], l[RT];
  f32x4 acc[RT][VB];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int k = 0; k < VB; ++k) acc[t][k] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  for (int tok = tok0; tok < to; tok += stride) {
    f32x4 s[RT][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint32_t w[4];
        bytes_to_f16(kr[t][ks >> 1][2 * (ks & 1)], w[0], w[1]);
        bytes_to_f16(kr[t][ks >> 1][2 * (ks & 1) + 1], w[2], w[3]);
        const f16x8 kf = __builtin_bit_cast(f16x8, u32x4{w[0], w[1], w[2], w[3]});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int q = 0; q < NQ; ++q)
            s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][ks][q], s[rt][t], 0, 0, 0);
      }
    }
    const int i = (tok - from) / 16;
    const int i1 = min(i + 1, groups - 1);
    // the next step's keys take the registers of these
    const bool more = tok + stride < to;
    long long at0 = 0, at1 = 0;
    if (more) {
      const int n = i + stride / 16;
      at0 = code_at(tok + stride, s_page[n]);
      at1 = code_at(tok + stride + 16, n + 1 < groups ? s_page[n + 1] : -1);
      load_k(at0, at1);
    }
    const float ks[2] = {s_ks[i], s_ks[i1]};
    const float vr[2] = {ldexpf(s_vs[i], -unit_e) * per_unit, ldexpf(s_vs[i1], -unit_e) * per_unit};
    const int page[2] = {s_page[i], s_page[i1]};
    const bool whole = __builtin_amdgcn_readfirstlane(tok >= all_lo && tok + 32 <= all_hi && tok + 32 <= to &&
                                                      page[0] >= 0 && page[1] >= 0);
    f16x8 pf[RT][NP];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float z[8];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float c = ks[t] * factor[rt];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[4 * t + e] = s[rt][t][e] * c;
      }
      if (!whole) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = tok + 16 * (e >> 2) + 4 * g + (e & 3);
          if (j < row_lo[rt] || j >= row_hi[rt] || page[e >> 2] < 0) z[e] = -INFINITY;
        }
      }
      float top = fmaxf(fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])), fmaxf(fmaxf(z[4], z[5]), fmaxf(z[6], z[7])));
      top = lanes16_max(top);
      const float mn = fmaxf(m[rt], top);
      const float ref = mn == -INFINITY ? 0.f : mn;   // nothing seen yet: all terms are 0
      if (__any(mn != m[rt])) {
        const float alpha = __builtin_amdgcn_exp2f(m[rt] - ref);
        l[rt] *= alpha;
#pragma unroll
        for (int k = 0; k < VB; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[rt][k][e] *= alpha;
        m[rt] = mn;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = __builtin_amdgcn_exp2f(z[e] - ref);
        l[rt] += pe;
        const float pv = in_f32(pe * vr[e >> 2]);
        pf[rt][0][e] = static_cast<_Float16>(pv);
        if constexpr (NP == 2) pf[rt][1][e] = static_cast<_Float16>(pv - static_cast<float>(pf[rt][0][e]));
      }
    }
#pragma unroll
    for (int w = 0; w < VW; ++w) {
      uint32_t x[2][4], y[2][4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[t][e] = vr8[4 * t + e][w];
        transpose4(x[t], y[t]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t f[4];
        bytes_to_f16(y[0][c], f[0], f[1]);
        bytes_to_f16(y[1][c], f[2], f[3]);
        const f16x8 vf = __builtin_bit_cast(f16x8, u32x4{f[0], f[1], f[2], f[3]});
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int q = 0; q < NP; ++q)
            acc[rt][4 * w + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt][q], acc[rt][4 * w + c], 0, 0, 0);
      }
    }
    if (more) load_v(at0, at1);
  }

  // join the waves: the common maximum, then the sums pairwise in a fixed order; unit 2^-15 with half
  // of its power of two here and the rest with 1 / l, so that neither factor underflows
  const int half_e = unit_e / 2;
  const float early = ldexpf(1.0f / 32768.0f, half_e), back = ldexpf(unit_m, unit_e - half_e);
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l[t] = lanes16_sum(l[t]);
    if (g == 0) {
      s_m[wave][16 * t + row16] = m[t];
      s_l[wave][16 * t + row16] = l[t];
    }
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    float all = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all = fmaxf(all, s_m[w][16 * t + row16]);
    const float ref = all == -INFINITY ? 0.f : all;
    const float mine = __builtin_amdgcn_exp2f(m[t] - ref) * early;
#pragma unroll
    for (int k = 0; k < VB; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][k][e] *= mine;
    l[t] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      l[t] += s_l[w][16 * t + row16] * __builtin_amdgcn_exp2f(s_m[w][16 * t + row16] - ref);
    m[t] = all;
  }
#pragma unroll
  for (int half = kWaves / 2; half > 0; half /= 2) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int k = 0; k < VB; ++k) s_o[wave - half][t][k][lane] = acc[t][k];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int k = 0; k < VB; ++k) acc[t][k] += s_o[wave][t][k][lane];
    }
    if (half > 1) __syncthreads();
  }
  if (wave > 0) return;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = r0 + 16 * t + row16;
    if (r >= r1) continue;
    const int token = r / p.group, head = kvh * p.group + r - token * p.group;
    const bool last = p.splits == 1;
    const float f = last ? (l[t] == 0.f ? 0.f : back / l[t]) : back;
    const long long row = static_cast<long long>(u.first + token) * p.heads + head;
    const long long part = (static_cast<long long>(split) * a.tokens * p.heads + row) * a.head_dim;
    if (!last && g == 0) {
      float* st = p.stats + 2 * (static_cast<long long>(split) * a.tokens * p.heads + row);
      st[0] = m[t];
      st[1] = l[t];
    }
    if (!last && l[t] == 0.f) continue;           // saw no key: the join takes nothing of it
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = VB * (4 * g + e);
      if (d >= a.head_dim) continue;
      float v[VB];
#pragma unroll
      for (int k = 0; k < VB; ++k) v[k] = acc[t][k][e] * f;
      if (last)
        store_n<TYPE, VB>(p.out, (u.first + token) * p.out_stride + static_cast<long long>(head) * a.head_dim + d,
                          p.vec, v);
      else
        store_n<QC_STORAGE_F32, VB>(p.part, part + d, true, v);
    }
  }
}

// ---- Many rows a key head: both operands through LDS ---------------------------
//
// With hundreds of rows a key head each key is used that often, so a first launch
// lays the codes out as f16 operands, exactly, once: per sequence and key head, for every 32
// keys the fragments of v_mfma_f32_32x32x16_f16, 1 KB each, in the order they
// are read.  K fragment s (16 dimensions): lane l key l & 31, dimensions 16 s + 8 (l >> 5)
// + j.  V fragment (t, k) (32 dimensions, 16 keys): lane l dimension 32 t + (l & 31), keys
// 16 k + 8 (j >> 2) + 4 (l >> 5) + (j & 3) -- the keys whose scores lane l of S^T = K Q^T
// holds in registers 8 k + j, so its probabilities are its operand of O^T = V^T P^T.
// Beside them the magnitudes of the key and value scales of each 16 keys (a negative scale
// turns its codes' signs); a key scale of -1 marks a group without a page.
// Workgroup barrier after which what the waves have read from LDS may be overwritten.
__device__ __forceinline__ void ring_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

struct Frags {
  _Float16* k;           // [units][cap / 32][DP / 16][512]
  _Float16* v;           // [units][cap / 32][DP / 32][2][512]
  float* ks;             // [units][cap / 16]
  float* vs;
  int cap;               // keys laid out per unit: a multiple of 64
  int unit0, units;      // the pass's units (sequence, of the listed ones, * kv_heads + key head)
};

template <int DP>
__global__ __launch_bounds__(256) void attention_layout(Kv8Args a, AttnArgs p, Frags f, int tiles) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = blockIdx.x % tiles, local = blockIdx.x / tiles;
  const int window = p.window;
  const int unit = f.unit0 + local, kvh = unit % a.kv_heads;
  int seq = unit / a.kv_heads, first, rows, kv;
  if (p.listed != kPadded) {
    Kv8Listed l;
    if (!find_listed(a, p, seq, l)) return;
    seq = l.seq;
  }
  if (!kv8_sequence(a, seq, first, rows, kv) || rows == 0) return;
  const int lo = window > 0 ? max(0, kv - rows + 1 - window) & ~63 : 0;
  const int tok = 32 * tile;
  if (tok < lo || tok >= ((kv + 63) & ~63)) return;
  const int8_t *kp[2], *vp[2];                    // codes of the tile's two groups of 16 keys
  bool k_neg[2], v_neg[2], v_zero[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = tok + 16 * i;
    kp[i] = vp[i] = nullptr;
    k_neg[i] = v_neg[i] = v_zero[i] = false;
    float ks = -1.f, vs = 0.f;
    if (t < kv && (window <= 0 || t + 15 >= kv - rows + 1 - window)) {   // some row sees one of them
      const int page = a.table[static_cast<long long>(seq) * a.columns + (t >> a.page_shift)];
      bool ok = false;
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.pages)) {
        const long long at = static_cast<long long>(page) * a.kv_heads + kvh;
        const float sk = a.k_scales[at], sv = a.v_scales[at];
        ok = isfinite(sk) && isfinite(sv);
        if (ok) {
          const long long off = (at * a.page_tokens + (t & (a.page_tokens - 1))) * a.head_dim;
          kp[i] = a.k_codes + off;
          vp[i] = a.v_codes + off;
          k_neg[i] = sk < 0.f;
          v_neg[i] = sv < 0.f;
          v_zero[i] = sv == 0.f;
          ks = fabsf(sk);
          vs = fabsf(sv);
        }
      }
      if (!ok && threadIdx.x == 0) *a.status = QC_INVALID_ARGUMENT;
    }
    if (threadIdx.x == 0) {
      const long long at = static_cast<long long>(local) * (f.cap / 16) + t / 16;
      f.ks[at] = ks;
      f.vs[at] = vs;
    }
  }
  const long long at32 = static_cast<long long>(local) * (f.cap / 32) + tile;
  constexpr int NF = DP / 16;                     // fragments of either kind
  for (int s = wave; s < NF; s += 4) {            // K
    const int key = lane & 31, d = 16 * s + 8 * (lane >> 5), i = key >> 4;
    u32x4 o = {0, 0, 0, 0};
    if (kp[i] != nullptr && d < a.head_dim) {
      const u32x2 b = *reinterpret_cast<const u32x2*>(kp[i] + (key & 15) * a.head_dim + d);
      uint32_t w[4];
      bytes_to_f16(b[0], w[0], w[1]);
      bytes_to_f16(b[1], w[2], w[3]);
      const uint32_t sign = k_neg[i] ? 0x80008000u : 0u;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = w[e] ^ sign;
    }
    *reinterpret_cast<u32x4*>(f.k + (at32 * NF + s) * 512 + 8 * lane) = o;
  }
  for (int s = wave; s < NF; s += 4) {            // V: fragment (t, k) = (s / 2, s % 2)
    const int i = s & 1, d = 32 * (s >> 1) + (lane & 31);
    f16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = static_cast<_Float16>(0.f);
    if (vp[i] != nullptr && !v_zero[i] && d < a.head_dim) {
      const int8_t* from = vp[i] + 4 * (lane >> 5) * a.head_dim + d;
      const int sign = v_neg[i] ? -1 : 1;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        o[j] = static_cast<_Float16>(sign * from[(8 * (j >> 2) + (j & 3)) * a.head_dim]);
    }
    *reinterpret_cast<u32x4*>(f.v + (at32 * NF + s) * 512 + 8 * lane) = __builtin_bit_cast(u32x4, o);
  }
}

// Workgroup: NW waves of 32 rows of a key head, a range of keys.  A step is 64 keys.
// A score's exponent is one fused multiply-add: with c the key scale times the row's
// factor and b = log2(value scale / largest one) + shift per 16 keys, p' = 2^(s c + b - m)
// is the probability as it meets the codes of V, and the sum takes p' 2^-b.  For 16-bit q p' is one
// f16, 11 bits.  That is as coarse as an f16 output, whose error against 64 bits it takes from 2.1e-4 to 2.8e-4 of the
// outputs' size (bf16: 1.66e-3 to 1.67e-3); a second term for f16 q, as the direct form has, costs 19 to 40% (8192
// tokens, heads of 128, 536 -> 747 us): half again the MFMAs of a loop that they bound.
// The shift is 11 there, and m follows the running maximum only once that is 4 above it (p' <= 2^15
// fits f16): of random rows, some maximum among 32 grows in most steps, and each growth
// rescales all sums.  p' keeps its 11 bits down to 2^-25 of the row's largest that way (with 7
// and 8, to 2^-21: a row whose largest meets a code of 0 showed it); f32 q, whose second
// term is 2^-11 smaller, takes 15 and 0.
//
// The exponentials of a step and its 32 MFMAs take about the same time, so they have to
// run beside each other, and waves that meet at a barrier every step do the same thing at
// the same time: a wave's own stream mixes them.  It computes the scores of step t + 1
// while step t's exponentials and value products go on, so K is a step ahead of V in the S
// LDS buffers each has.
//
// 8192 tokens, 32 / 8 heads of 128, bf16, causal (550 GFLOP): 510 to 550 us by session and 13 for the layout, 0.98 to
// 1.05 PFLOP/s of both (a plain f16 product of 8192^3 reaches 1.1 to 1.3).  MFMAs and VALU are each busy
// half of the SIMDs' cycles and the clock is at 1.9 GHz: what bounds it is issue and power.
// Priorities by wave or phase change nothing or cost 4%.
// 16-key groups of a range: what LDS holds beside the buffers. (Each range of a prompt's keys
// takes its rows' sums in memory: 17 GB for 131072 tokens of 32 heads in ranges of 16384.)
template <int DP>
constexpr int kTiledGroups = DP == 256 ? 1024 : 4096;
constexpr int kTiledLeast = 1024;   // keys of a range, where there are as many

template <int DP, int NW, int TYPE>
__global__ __launch_bounds__(64 * NW, NW / 4) void attention_tiled(Kv8Args a, AttnArgs p, Frags f) {
  constexpr int NF = DP / 16, DT = DP / 32;
  constexpr int NQ = TYPE == QC_STORAGE_F32 ? 2 : 1;
  constexpr int kBytes = 2 * NF * 1024;           // 64 keys of K, or of V
  constexpr int LOADS = kBytes / 1024 / NW;       // a wave's loads of 1 KB of either a step
  constexpr int S = 2;                            // buffers (three: 582 -> 605 us)
  static_assert(kBytes % (1024 * NW) == 0, "whole loads");
  __shared__ __attribute__((aligned(1024))) uint8_t s_k[S * kBytes], s_v[S * kBytes];
  __shared__ f32x4 s_c[kTiledGroups<DP> / 4], s_b[kTiledGroups<DP> / 4], s_inv[kTiledGroups<DP> / 4];
  __shared__ float s_unit[NW];
  __shared__ int s_bad[NW];

  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // unit (listed: key head) fastest: with workgroups dealt to the XCDs in turn, a head's
  // blocks share an L2; the longest rows (last blocks) first
  int id = blockIdx.x, local, split, rb, seq;
  Unit u;
  if (p.listed == kPadded) {
    const int units = gridDim.x / (p.splits * p.row_blocks);
    local = id % units;
    id /= units;
    split = id % p.splits;
    rb = p.row_blocks - 1 - id / p.splits;
    seq = (f.unit0 + local) / a.kv_heads;
    if (!kv8_sequence(a, seq, u.first, u.rows, u.kv)) return;
  } else {
    local = id % a.kv_heads;
    id /= a.kv_heads;
    split = id % p.splits;
    Kv8Listed l;
    if (!find_listed(a, p, id / p.splits, l)) return;
    seq = l.seq;
    local += l.before * a.kv_heads - f.unit0;
    if (local < 0 || local >= f.units || !kv8_sequence(a, seq, u.first, u.rows, u.kv)) return;
    rb = (u.rows * p.group + p.per - 1) / p.per - 1 - l.at;
    if (rb < 0) return;
  }
  const int kvh = (f.unit0 + local) % a.kv_heads;
  const int r0 = rb * NW * 32, r1 = min(r0 + NW * 32, u.rows * p.group);
  if (r0 >= r1) return;
  int lo, hi;
  seen_range(p, u, r0 / p.group, (r1 - 1) / p.group, lo, hi);
  int used;
  const int chunk = range_keys(a, p, kTiledLeast, 64, used);
  const int from = __builtin_amdgcn_readfirstlane((lo & ~63) + split * chunk);
  const int to = __builtin_amdgcn_readfirstlane(min(hi, from + chunk));
  const int steps = to > from ? (to - from + 63) >> 6 : 0;

  const long long tile0 = static_cast<long long>(local) * (f.cap / 32) + from / 32;
  const _Float16* kf = f.k + tile0 * NF * 512;
  const _Float16* vf = f.v + tile0 * NF * 512;
  // Loads of steps past the last repeat it, into buffers that are not read again, so that
  // the number in flight is the same in every step.
  auto issue = [&](const _Float16* src, uint8_t* buffer, int step) {
    const _Float16* from_step = src + static_cast<long long>(min(step, steps - 1)) * 2 * NF * 512;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = wave * LOADS + i;             // uniform
      dma16(from_step + q * 512, 16 * lane, buffer + q * 1024);
    }
  };
  if (steps > 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) {
      issue(kf, s_k + i * kBytes, i);
      if (i < S - 1) issue(vf, s_v + i * kBytes, i);
    }
  }

  // the range's key scales, and its value scales against the largest
  constexpr float kLow = -3.0e38f;                // below every score
  constexpr float kShift = NQ == 2 ? 15.f : 11.f, kSlack = 15.f - kShift;
  const float* ks = f.ks + static_cast<long long>(local) * (f.cap / 16) + from / 16;
  const float* vs = f.vs + static_cast<long long>(local) * (f.cap / 16) + from / 16;
  float unit = 0.f;
  bool bad = false;
  for (int i = threadIdx.x; i < 4 * steps; i += 64 * NW) {
    unit = fmaxf(unit, vs[i]);
    bad = bad || (ks[i] < 0.f && from + 16 * i < to && from + 16 * i + 15 >= lo);   // a page missing
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) unit = fmaxf(unit, __shfl_xor(unit, o));
  bad = __any(bad);
  if (lane == 0) {
    s_unit[wave] = unit;
    s_bad[wave] = bad;
  }

  // q: row lane & 31, dimensions 16 s + 8 half + j
  f16x8 qf[NF][NQ];
  const int r = r0 + 32 * wave + (lane & 31);
  const bool has = r < r1;
  const int token = (has ? r : r0) / p.group, head = kvh * p.group + (has ? r : r0) - token * p.group;
  const int row_hi = has ? (p.causal ? min(u.kv, u.position(token) + 1) : u.kv) : 0;
  const int row_lo = p.window > 0 ? u.position(token) + 1 - p.window : 0;
  float factor, broken = 0.f;                     // broken: NaN for a row that is not finite
  {
    const long long at = (u.first + token) * p.q_stride + static_cast<long long>(head) * a.head_dim;
    float v[NF][8], top = 0.f;
    bool nan = false;
#pragma unroll
    for (int s = 0; s < NF; ++s) {
      const int d = 16 * s + 8 * half;
      load8<TYPE>(p.q, at + d, has && d < a.head_dim, p.vec, v[s]);
    }
#pragma unroll
    for (int s = 0; s < NF; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top = fmaxf(top, fabsf(v[s][j]));
        nan = nan || v[s][j] != v[s][j];
      }
    if (nan) top = INFINITY;
    top = fmaxf(top, __shfl_xor(top, 32));
    float inverse;
    float up = row_scale(top, inverse);
    if (inverse != inverse) {
      broken = inverse;
      inverse = 1.f;
      up = 0.f;
    }
    factor = fabsf(p.scale) * kLog2e * inverse;
    if (p.scale < 0.f) up = -up;
#pragma unroll
    for (int s = 0; s < NF; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = in_f32(broken != broken ? 0.f : v[s][j] * up);
        qf[s][0][j] = static_cast<_Float16>(x);
        if constexpr (NQ == 2) qf[s][1][j] = static_cast<_Float16>(x - static_cast<float>(qf[s][0][j]));
      }
  }
  // keys every row of the wave sees, and any of them
  int all_hi = row_hi, any_hi = row_hi, all_lo = row_lo;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all_hi = min(all_hi, __shfl_xor(all_hi, o));
    any_hi = max(any_hi, __shfl_xor(any_hi, o));
    all_lo = max(all_lo, __shfl_xor(all_lo, o));
  }
  all_hi = __builtin_amdgcn_readfirstlane(all_hi);
  any_hi = __builtin_amdgcn_readfirstlane(any_hi);
  all_lo = __builtin_amdgcn_readfirstlane(all_lo);
  __syncthreads();
  int any_bad = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    unit = fmaxf(unit, s_unit[w]);
    any_bad |= s_bad[w];
  }
  any_bad = __builtin_amdgcn_readfirstlane(any_bad);
  for (int i = threadIdx.x; i < 4 * steps; i += 64 * NW) {
    // a scale of 0 has codes of 0, so any b will do for it
    const float b = kShift + (vs[i] > 0.f ? fmaxf(__log2f(vs[i] / unit), -100.f) : 0.f);
    reinterpret_cast<float*>(s_c)[i] = ks[i];
    reinterpret_cast<float*>(s_b)[i] = b;
    reinterpret_cast<float*>(s_inv)[i] = __builtin_amdgcn_exp2f(-b);
  }

  float m = kLow, l = 0.f;
  f32x16 acc[DT], s[2], sn[2];
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[t][e] = 0.f;
  // quarter i of a step's score products: key tile i / 2, one half of the dimensions
  auto scores = [&](const f16x8 (&k)[NF / 2], int i, f32x16 (&o)[2]) {
    const int t = i >> 1;
    if ((i & 1) == 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < NF / 2; ++d)
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[d], qf[(i & 1) * (NF / 2) + d][q], o[t], 0, 0, 0);
  };
  // The compiler reads a fragment from LDS just before the MFMA that takes it; reads kept where
  // they are written have a quarter's arithmetic to arrive in (us, heads of 64 / 128 / 256: 99.6
  // -> 95.1 / 533 -> 528 / 193 -> 174).  With two terms the registers do not hold V's beside K's, and
  // the compiler keeps the order (f32, 128: 116 -> 113; pinned 191).
  auto pin = [] {
    if constexpr (NQ == 1) __builtin_amdgcn_sched_barrier(0);
  };
  if (steps > 0) wait_vmcnt<2 * (S - 1) * LOADS>();   // K of step 0
  __syncthreads();
  if (steps > 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f16x8 kq[NF / 2];
#pragma unroll
      for (int d = 0; d < NF / 2; ++d)
        kq[d] = *reinterpret_cast<const f16x8*>(s_k + 16 * lane + ((i >> 1) * NF + (i & 1) * (NF / 2) + d) * 1024);
      scores(kq, i, s);
    }
  }

  int kbuf = 0, vbuf = 0;                         // buffers of K and V of the step
  // s: the step's scores; sn: receives the next one's
  auto run = [&](int step, f32x16 (&s)[2], f32x16 (&sn)[2]) {
    const int tok = from + 64 * step;
    wait_vmcnt<2 * (S - 2) * LOADS>();            // this wave's loads of V of the step, K of the next
    ring_sync();                                  // everyone's; V of the step before, K of this are free
    const int vfree = vbuf > 0 ? vbuf - 1 : S - 1;
    issue(vf, s_v + vfree * kBytes, step + S - 1);
    issue(kf, s_k + kbuf * kBytes, step + S);
    kbuf = kbuf + 1 < S ? kbuf + 1 : 0;
    const uint8_t* vb = s_v + vbuf * kBytes + 16 * lane;
    const uint8_t* kb = s_k + kbuf * kBytes + 16 * lane;   // of the next step
    vbuf = vbuf + 1 < S ? vbuf + 1 : 0;
    if (tok >= any_hi) return;                    // none of the wave's rows sees more
    f16x8 kq[NF / 2], vq[DT];                     // a quarter's fragments of K and of V
    auto load_k = [&](int i) {
#pragma unroll
      for (int d = 0; d < NF / 2; ++d)
        kq[d] = *reinterpret_cast<const f16x8*>(kb + ((i >> 1) * NF + (i & 1) * (NF / 2) + d) * 1024);
    };
    auto load_v = [&](int i) {
#pragma unroll
      for (int t = 0; t < DT; ++t) vq[t] = *reinterpret_cast<const f16x8*>(vb + ((i >> 1) * NF + 2 * t + (i & 1)) * 1024);
    };
    load_k(0);
    pin();
    f32x4 c = s_c[step];
    const f32x4 b = s_b[step], inv = s_inv[step];
    if (any_bad || tok < all_lo || tok + 64 > all_hi) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int j = tok + 32 * t + 8 * (e >> 2) + 4 * half + (e & 3);
          if (j < row_lo || j >= row_hi || c[2 * t + (e >> 3)] < 0.f) s[t][e] = -INFINITY;
        }
    }
    float top = kLow;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = fmaxf(c[i] * factor, 1e-37f);        // above 0: masked scores stay -inf
      const f32x16& x = s[i >> 1];
      const int o = 8 * (i & 1);
      const float g = max3(max3(x[o], x[o + 1], x[o + 2]), max3(x[o + 3], x[o + 4], x[o + 5]),
                           max3(x[o + 6], x[o + 7], x[o + 7]));
      top = fmaxf(top, g * c[i]);
    }
    {
      auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
    }
    if (__any(top > m + kSlack)) {
      const float mn = fmaxf(m, top);
      const float alpha = __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[t][e] *= alpha;
      m = mn;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (NQ == 1) load_v(i);
      pin();
      scores(kq, i, sn);                          // past the last step: of no use, and not used
      if constexpr (NQ == 2) load_v(i);
      const float off = b[i] - m;
      float e8[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e8[j] = __builtin_amdgcn_exp2f(fmaf(s[i >> 1][8 * (i & 1) + j], c[i], off));
      f16x8 pf[NQ];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        pf[0][j] = static_cast<_Float16>(e8[j]);
        if constexpr (NQ == 2) pf[1][j] = static_cast<_Float16>(e8[j] - static_cast<float>(pf[0][j]));
      }
      // (an f16 dot for the sum would lose the probabilities that are subnormal there)
      const float sum = ((e8[0] + e8[1]) + (e8[2] + e8[3])) + ((e8[4] + e8[5]) + (e8[6] + e8[7]));
      l = fmaf(sum, inv[i], l);
      if (i < 3) load_k(i + 1);
      pin();
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int q = 0; q < NQ; ++q) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vq[t], pf[q], acc[t], 0, 0, 0);
    }
  };
  for (int step = 0; step < steps; step += 2) {
    run(step, s, sn);
    if (step + 1 < steps) run(step + 1, sn, s);
  }
  wait_vmcnt<0>();   // no load may land in LDS that is no longer this workgroup's
  l += __shfl_xor(l, 32);
  if (!has) return;
  const bool last = p.splits == 1;
  int unit_e;                                     // its power of two comes last: no factor underflows
  const float unit_m = split_unit(unit, unit_e);
  const float back = unit_m * (NQ == 2 ? 1.0f / 32768.0f : 1.0f / 2048.0f) + broken;   // 2^-kShift
  const float scale = last ? (l == 0.f ? 0.f : back / l) : back;
  const long long row = static_cast<long long>(u.first + token) * p.heads + head;
  const long long part = static_cast<long long>(split) * a.tokens * p.heads + row;
  if (!last) {
    if (half == 0) {
      p.stats[2 * part] = l == 0.f ? -INFINITY : m;
      p.stats[2 * part + 1] = l;
    }
    if (l == 0.f) return;
  }
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int d = 32 * t + 2 * e + 4 * half;
      if (d >= a.head_dim) continue;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = l == 0.f ? 0.f : ldexpf(acc[t][e + j] * scale, unit_e);
      if (last)
        store_n<TYPE, 4>(p.out, (u.first + token) * p.out_stride + static_cast<long long>(head) * a.head_dim + d,
                         p.vec, v);
      else
        store_n<QC_STORAGE_F32, 4>(p.part, part * a.head_dim + d, true, v);
    }
}

// Row `item` of a join's grid: `per` rows of each row block.
__device__ __forceinline__ bool join_row(const Kv8Args& a, const AttnArgs& p, int item, int per, Unit& u, int& token,
                                         int& head) {
  int seq, kvh, rb;
  if (!block_of(a, p, item / per, seq, kvh, rb) || seq >= a.seqs) return false;
  if (!kv8_sequence(a, seq, u.first, u.rows, u.kv)) return false;
  const int r = rb * p.per + item % per, all = u.rows * p.group;
  if (r >= all || all < p.rows_from || all >= p.rows_to) return false;
  token = r / p.group;
  head = kvh * p.group + r - token * p.group;
  return true;
}

// out = sum over the ranges of 2^(m_s - m) O_s over that of 2^(m_s - m) l_s: a
// workgroup a row.  256 / L groups of L threads (L >= head_dim / 4, a power of two) take the
// ranges in turn, four loads ahead, and meet in LDS in a fixed order.  (A wavefront a
// row, its ranges one after the other: 128 ranges of 32 rows 30 us, 5 so.)  `per`: rows of
// a block that are launched.
template <int TYPE>
__global__ __launch_bounds__(256) void attention_join(Kv8Args a, AttnArgs p, int per, int shift) {
  __shared__ float s_w[256], s_red[8];
  __shared__ f32x4 s_o[256];
  const int tid = threadIdx.x;
  Unit u;
  int token, head;
  if (!join_row(a, p, blockIdx.x, per, u, token, head)) return;
  const long long rows = static_cast<long long>(a.tokens) * p.heads;
  const long long row = static_cast<long long>(u.first + token) * p.heads + head;
  const float* stats = p.stats + 2 * row;
  float m = -INFINITY;
  for (int s = tid; s < p.splits; s += 256) m = fmaxf(m, stats[2 * s * rows]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if ((tid & 63) == 0) s_red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  const float ref = m == -INFINITY ? 0.f : m;
  const int group = tid >> shift, groups = 256 >> shift, d = 4 * (tid & ((1 << shift) - 1));
  float l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < p.splits; s0 += 256) {
    float w = 0.f;
    const int n = min(256, p.splits - s0);
    if (tid < n) {
      const float ls = stats[2 * (s0 + tid) * rows + 1];
      // a range with no key the row sees has no sums (one of a row that is not finite has a
      // sum of NaN): -1 marks it
      w = ls == 0.f ? -1.f : __builtin_amdgcn_exp2f(stats[2 * (s0 + tid) * rows] - ref);
      if (ls != 0.f) l = fmaf(w, ls, l);
    }
    s_w[tid] = w;
    __syncthreads();
    if (d < a.head_dim) {
      const float* o = p.part + (s0 * rows + row) * a.head_dim + d;
#pragma unroll 4
      for (int s = group; s < n; s += groups) {
        const float f = s_w[s];
        if (f == -1.f) continue;
        const f32x4 x = *reinterpret_cast<const f32x4*>(o + s * rows * a.head_dim);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, x[e], acc[e]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if ((tid & 63) == 0) s_red[4 + (tid >> 6)] = l;
  s_o[tid] = acc;
  __syncthreads();
  if (group > 0 || d >= a.head_dim) return;
  for (int g = 1; g < groups; ++g) acc += s_o[(g << shift) + tid];
  l = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = l == 0.f ? 0.f : acc[e] / l;
  store_n<TYPE, 4>(p.out, (u.first + token) * p.out_stride + static_cast<long long>(head) * a.head_dim + d, p.vec, v);
}

// The same for a few ranges: L threads a row, each through all of them.  Prompts split in
// two or four have thousands of rows, and a workgroup for each is mostly its own start.
constexpr int kFewSplits = 8;
template <int TYPE>
__global__ __launch_bounds__(256) void attention_join_few(Kv8Args a, AttnArgs p, int per, int shift) {
  const int d = 4 * (threadIdx.x & ((1 << shift) - 1));
  Unit u;
  int token, head;
  // (a wavefront's rows, 16 at most, are one block's where blocks are listed)
  if (!join_row(a, p, blockIdx.x * (256 >> shift) + (threadIdx.x >> shift), per, u, token, head) || d >= a.head_dim) return;
  const long long rows = static_cast<long long>(a.tokens) * p.heads;
  const long long row = static_cast<long long>(u.first + token) * p.heads + head;
  float ms[kFewSplits], ls[kFewSplits], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    ms[s] = -INFINITY;
    ls[s] = 0.f;
    if (s < p.splits) {
      ms[s] = p.stats[2 * (s * rows + row)];
      ls[s] = p.stats[2 * (s * rows + row) + 1];
    }
    m = fmaxf(m, ms[s]);
  }
  const float ref = m == -INFINITY ? 0.f : m;
  f32x4 x[kFewSplits], acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (ls[s] != 0.f) x[s] = *reinterpret_cast<const f32x4*>(p.part + (s * rows + row) * a.head_dim + d);
  }
#pragma unroll
  for (int s = 0; s < kFewSplits; ++s) {
    const float w = __builtin_amdgcn_exp2f(ms[s] - ref);
    l = fmaf(w, ls[s], l);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(w, x[s][e], acc[e]);
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = l == 0.f ? 0.f : acc[e] / l;
  store_n<TYPE, 4>(p.out, (u.first + token) * p.out_stride + static_cast<long long>(head) * a.head_dim + d, p.vec, v);
}

// A call's partial sums where its keys are split.
hipError_t part_buffers(const Kv8Args& a, AttnArgs& p, StreamWorkspace* ws, hipStream_t s) {
  const size_t outs = static_cast<size_t>(p.splits) * a.tokens * p.heads;
  void* buf = nullptr;
  const hipError_t e = stream_buffer(ws, s, outs * (a.head_dim + 2) * sizeof(float), 0, &buf);
  p.part = static_cast<float*>(buf);
  p.stats = p.part + outs * a.head_dim;
  return e;
}

// blocks: row blocks of all key heads (what block_of takes).
template <int TYPE>
hipError_t run_join(const Kv8Args& a, const AttnArgs& p, long long blocks, hipStream_t s) {
  int shift = 2;
  while ((4 << shift) < a.head_dim) ++shift;
  const bool one = p.listed != kBlocks && p.row_blocks == 1;
  const int per = one ? std::min<long long>(p.per, static_cast<long long>(a.max_new) * p.group) : p.per;
  const long long items = blocks * per;
  if (items > INT_MAX - 256) return hipErrorInvalidValue;
  const int rows = p.splits <= kFewSplits ? 256 >> shift : 1;   // of a workgroup
  if (!kv8_grid_fits((items + rows - 1) / rows, 256)) return hipErrorInvalidValue;
  if (p.splits <= kFewSplits) {
    attention_join_few<TYPE><<<static_cast<unsigned>((items + rows - 1) / rows), 256, 0, s>>>(a, p, per, shift);
    return hipGetLastError();
  }
  attention_join<TYPE><<<static_cast<unsigned>(items), 256, 0, s>>>(a, p, per, shift);
  return hipGetLastError();
}

// Keys that a block of `rows` rows can see, from a multiple of `align` on.
long long key_span(const Kv8Args& a, const AttnArgs& p, int rows, int align) {
  if (p.window <= 0) return a.max_kv;
  return std::min<long long>(a.max_kv, static_cast<long long>(p.window) + (rows + p.group - 1) / p.group + align);
}

template <int DP, int RT, int TYPE>
hipError_t run_direct(const Kv8Args& a, AttnArgs p, hipStream_t s) {
  const long long rows = std::min<long long>(static_cast<long long>(a.max_new) * p.group, p.rows_to - 1);
  p.per = RT * 16;
  p.row_blocks = static_cast<int>((rows + p.per - 1) / p.per);
  const long long span = key_span(a, p, RT * 16, 32);
  const long long padded = static_cast<long long>(a.seqs) * p.row_blocks;
  const long long there = static_cast<long long>(a.tokens) * p.group / p.per + a.seqs;   // at most
  p.listed = kv8_listed(padded, there) ? kBlocks : kPadded;
  const long long units = std::min(padded, p.listed == kBlocks ? there : padded) * a.kv_heads;
  const long long want = std::max<long long>(1, 2LL * device_cu_count() / units);
  long long chunk = (span + want - 1) / want;
  chunk = std::max<long long>(32 * kWaves, (chunk + 31) / 32 * 32);
  // ranges of 4096 keys at most, or of 16384 where their sums would take more than 1 GB
  const long long range_bytes = static_cast<long long>(a.tokens) * p.heads * (a.head_dim + 2) * 4;
  chunk = std::min<long long>(chunk, (span + 4095) / 4096 * range_bytes > (1LL << 30) ? 16 * kMaxGroups : 4096);
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>((span + chunk - 1) / chunk);
  p.want = static_cast<int>(std::min<long long>(want, p.splits));
  p.span = static_cast<int>(span);
  const long long grid = units * p.splits;
  if (!kv8_grid_fits(grid, 64 * kWaves)) return hipErrorInvalidValue;
  std::unique_lock<std::mutex> hold;
  if (p.splits > 1) {
    StreamWorkspace* ws = nullptr;
    hipError_t e = stream_workspace(s, &ws);
    if (e != hipSuccess) return e;
    hold = std::unique_lock<std::mutex>(ws->call);
    if ((e = part_buffers(a, p, ws, s)) != hipSuccess) return e;
  }
  attention_direct<DP, RT, TYPE><<<static_cast<unsigned>(grid), 64 * kWaves, 0, s>>>(a, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return e;
  return run_join<TYPE>(a, p, units, s);
}

// Bytes of fragments laid out at a time; a call with more goes in passes of whole units.
constexpr long long kFragPass = 1LL << 30;

// The tiled form's grid for sequences of p.rows_from rows or more: units laid out at most, row
// blocks of a key head, ranges of keys.
struct TiledPlan {
  long long units, blocks;
};
TiledPlan plan_tiled(const Kv8Args& a, AttnArgs& p, int per, int max_groups) {
  const long long rows = static_cast<long long>(a.max_new) * p.group;
  p.per = per;
  p.row_blocks = static_cast<int>((rows + per - 1) / per);
  const long long span = key_span(a, p, per, 64);
  const long long all = static_cast<long long>(a.tokens) * p.group;
  const long long seqs = p.rows_from > 0 ? std::min<long long>(a.seqs, all / p.rows_from) : a.seqs;
  const long long padded = seqs * p.row_blocks, there = all / per + seqs;   // at most
  p.listed = p.rows_from > 0 || padded > there ? kBlocks : kPadded;
  const long long blocks = std::min(padded, p.listed == kBlocks ? there : padded);
  const long long want = std::max<long long>(1, device_cu_count() / (blocks * a.kv_heads));
  long long chunk = ((span + want - 1) / want + 63) / 64 * 64;
  chunk = std::max<long long>(chunk, kTiledLeast);
  chunk = std::min<long long>(chunk, 16 * max_groups);
  p.chunk = static_cast<int>(chunk);
  p.splits = static_cast<int>((span + chunk - 1) / chunk);
  p.want = static_cast<int>(std::min<long long>(want, p.splits));
  p.span = static_cast<int>(span);
  return {seqs * a.kv_heads, blocks};
}

template <int DP, int NW, int TYPE>
hipError_t run_tiled(const Kv8Args& a, AttnArgs p, hipStream_t s) {
  const TiledPlan plan = plan_tiled(a, p, 32 * NW, kTiledGroups<DP>);
  const long long units = plan.units, blocks = plan.blocks;
  Frags f = {};
  f.cap = (a.max_kv + 63) / 64 * 64;
  const long long unit_bytes = static_cast<long long>(f.cap) * DP * 4 + f.cap / 2;   // two of f16, scales
  const long long pass = std::min(units, std::max<long long>(1, kFragPass / unit_bytes));
  if (!kv8_grid_fits((p.listed == kPadded ? pass * p.row_blocks : blocks * a.kv_heads) * p.splits, 64 * NW) ||
      !kv8_grid_fits(pass * (f.cap / 32), 256))
    return hipErrorInvalidValue;
  StreamWorkspace* ws = nullptr;
  hipError_t e = stream_workspace(s, &ws);
  if (e != hipSuccess) return e;
  std::unique_lock<std::mutex> hold(ws->call);
  if (p.splits > 1 && (e = part_buffers(a, p, ws, s)) != hipSuccess) return e;
  void* buf = nullptr;
  if ((e = stream_buffer(ws, s, static_cast<size_t>(pass) * unit_bytes, 1, &buf)) != hipSuccess) return e;
  f.k = static_cast<_Float16*>(buf);
  f.v = f.k + pass * f.cap * DP;
  f.ks = reinterpret_cast<float*>(f.v + pass * f.cap * DP);
  f.vs = f.ks + pass * (f.cap / 16);
  for (long long u0 = 0; u0 < units; u0 += pass) {
    const int n = static_cast<int>(std::min(pass, units - u0));
    f.unit0 = static_cast<int>(u0);
    f.units = n;
    const int tiles = f.cap / 32;
    AttnArgs lay = p;
    if (p.listed != kPadded) lay.listed = kSequences;
    attention_layout<DP><<<static_cast<unsigned>(n) * tiles, 256, 0, s>>>(a, lay, f, tiles);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const long long grid = (p.listed == kPadded ? n * p.row_blocks : blocks * a.kv_heads) * p.splits;
    attention_tiled<DP, NW, TYPE><<<static_cast<unsigned>(grid), 64 * NW, 0, s>>>(a, p, f);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return p.splits > 1 ? run_join<TYPE>(a, p, blocks * a.kv_heads, s) : hipSuccess;
}

// The tiled form lays the cache out first and reads 64 keys for 256 rows (128 of heads above 128) at
// a time, so it takes prompts: sequences of 512 rows a key head or more, and three workgroups
// to four CUs; up to 1024 keys, where the direct form is mostly its workgroups' starts, 256
// rows and one to two CUs.  Below that, one tile of 16 rows a workgroup or two: two read the keys
// half as often, one makes twice the workgroups (heads above 128: of less than half the
// registers).  us, one / two / tiled, causal, key heads x rows x keys:
//                        8 x 512 x 8000     16 x 1024 x 500    16 x 2048 x 2000     64 x 512 x 2000
//   bf16, heads of 64     45 / 36 / 44        14 / 14 / 21       62 / 50 / 45         65 / 50 / 49
//   bf16, 128             64 / 51 / 55        22 / 20 / 29      102 / 81 / 62        104 / 82 / 73
//   bf16, 256             99 / 103 / 82       42 / 47 / 42      183 / 191 / 103      198 / 192 / 126
//   f32, 128              76 / 62 / 78        27 / 25 / 41      125 / 100 / 86       127 / 102 / 100
// and, bf16, 128, 192 x 256 x 500 57 / 57 / 44, 16 x 2048 x 500 (128 workgroups) 33 / 36 / 30.  Over
// 2000 cases of 2 to 192 key heads, 48 to 2048 rows and 500 to 8000 keys the rule is 0.6%
// off the best of the three.
//
// A ragged batch may hold both kinds: the rows counted are those that its tokens allow, and where
// not every sequence can have as many, those that have are laid out and the others
// read directly: 4096 new tokens beside 63 sequences of one, 4000 to 8000 keys, 2317 us
// with all laid out, 700 so (the prompt alone 460, the others 170).
template <int DP, int TYPE>
hipError_t run_rows(const Kv8Args& a, AttnArgs p, hipStream_t s) {
  constexpr int NW = DP == 256 ? 4 : 8;
  const bool brief = a.max_kv <= 1024;
  const int many = brief ? 256 : 512;
  const long long rows = static_cast<long long>(a.max_new) * p.group;
  const long long all = std::min(a.seqs * rows, static_cast<long long>(a.tokens) * p.group);   // of a key head
  p.rows_to = INT_MAX;
  bool tiled = p.route == 3;
  if (p.route == 0 && rows >= many) {
    AttnArgs q = p;
    if (all < static_cast<long long>(a.seqs) * many) q.rows_from = many;
    const long long groups = plan_tiled(a, q, 32 * NW, kTiledGroups<DP>).blocks * a.kv_heads * q.splits;
    tiled = 4 * groups >= (brief ? 2 : 3) * device_cu_count();
    if (tiled) p.rows_from = q.rows_from;
  }
  if (tiled && p.rows_from == 0) return run_tiled<DP, NW, TYPE>(a, p, s);
  double keys = a.max_kv;
  if (p.causal) keys -= 0.5 * std::min(a.max_new, a.max_kv);
  if (p.window > 0) keys = std::min<double>(keys, p.window);
  const double pairs = static_cast<double>(all) * a.kv_heads / 16 * keys;
  const bool two = p.route == 0 ? rows > 16 && (DP <= 128 ? pairs >= 0x1p19 : keys >= 600 && pairs >= 0x1p20)
                                : p.route == 2;
  AttnArgs few = p;
  few.rows_from = 0;
  if (tiled) few.rows_to = many;
  hipError_t e = hipSuccess;
  if constexpr (DP < 256 || TYPE != QC_STORAGE_F32) {   // (two of f32 256 do not fit the registers)
    e = two ? run_direct<DP, 2, TYPE>(a, few, s) : run_direct<DP, 1, TYPE>(a, few, s);
  } else {
    e = run_direct<DP, 1, TYPE>(a, few, s);
  }
  return tiled && e == hipSuccess ? run_tiled<DP, NW, TYPE>(a, p, s) : e;
}

template <int TYPE>
hipError_t run_typed(const Kv8Args& a, const AttnArgs& p, hipStream_t s) {
  if (a.head_dim <= 64) return run_rows<64, TYPE>(a, p, s);
  if (a.head_dim <= 128) return run_rows<128, TYPE>(a, p, s);
  return run_rows<256, TYPE>(a, p, s);
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8Attention& r, int* status, hipStream_t s) {
  const Kv8Args a = kv8_args(*r.cache, *r.batch, status);
  AttnArgs p = {};
  p.q = r.q;
  p.out = r.out;
  p.q_stride = r.q_stride;
  p.out_stride = r.out_stride;
  p.heads = static_cast<int>(r.heads);
  p.group = p.heads / a.kv_heads;
  p.scale = r.scale;
  p.causal = r.causal;
  p.window = static_cast<int>(r.window);
  p.route = r.route;
  const int size = r.type == QC_STORAGE_F32 ? 4 : 2;
  p.vec = ((reinterpret_cast<uintptr_t>(r.q) | reinterpret_cast<uintptr_t>(r.out) |
            static_cast<uintptr_t>(r.q_stride * size) | static_cast<uintptr_t>(r.out_stride * size)) & 15) == 0;
  switch (r.type) {
    case QC_STORAGE_F32: return run_typed<QC_STORAGE_F32>(a, p, s);
    case QC_STORAGE_F16: return run_typed<QC_STORAGE_F16>(a, p, s);
    default: return run_typed<QC_STORAGE_BF16>(a, p, s);
  }
}

}  // namespace qc
