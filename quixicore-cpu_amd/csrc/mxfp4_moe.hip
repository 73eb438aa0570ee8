// A mixture-of-experts feed-forward with MXFP4 weights for a few tokens on gfx950:
// l = x R^T + b, the k experts of the largest l (ties to the lowest index), their shares p
// (softmax of l over the chosen, or over all), and
//   y = residual + sum_s p_s D_e (act(G_e x) * (U_e x)),  e = e_s.
//
// Logits are sums in 64 bits, so that which experts are chosen does not hang on the order of a sum.
//
// Weights are operands of v_mfma_scale_f32_16x16x128_f8f6f4 as they are stored: 32 codes (16 bytes, one block of a
// row) and the block's scale byte a lane.  Activations meet them as sums of e4m3 terms under a power of two for each
// 32: with v in [2^7, 2^8) at the largest, a term holds 4 bits of what the terms before it left, and its
// scale is 2^4 below theirs.  x of bf16 is 2 terms (its 8 bits), of f16 3 (11), of f32 6 (24); the hidden values are 3
// (to 2^-12 of a value, beside the 2^-9 that a bf16 output is rounded by), 4 (2^-16) and 6.
//
// The instruction adds 16 products on a grid 2^-13 below the largest one's exponent and cuts what is below it (measured;
// the sums of 16 and the accumulator meet in f32).  So every term but the last is a multiple of 2^-2, which with
// codes of 2^-1 to 4 and terms of up to 2^8 is that grid: its sums are exact, and what it leaves is in the next.  With six
// terms that gives a f32 product's error (1e-6 of the result; e4m3 terms down to their own 2^-9 gave 3e-5).  A value
// far below its block's largest m so keeps an error of 2^-14 m (bf16; f16 2^-18 m, f32 2^-30 m).
#include <algorithm>

#include "qc_device.h"
#include "qc_internal.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPass = 512;              // tokens of a pass
constexpr int kMaxExperts = 1024;       // (and 64 of a token)
constexpr int kSmall = 16;              // pairs of a token and an expert that are worked on one by one (see pair_by_pair)

struct MoeArgs {
  const void* router;
  const float* bias;
  const uint8_t *gu, *gus, *dn, *dns;
  int router_type, experts, dim, inter, top;
  const void* x;
  long long x_stride;
  const void* residual;
  long long residual_stride;
  void* y;
  long long y_stride;
  int tokens, normalize, gelu;
  float scale;
  double* logits;        // [tokens][experts]
  int* ids;              // [tokens][top]
  float* shares;
  uint8_t* xq;           // x in terms: [terms][tokens][dim] e4m3
  uint8_t* xs;           // [tokens][scale_row(dim)] the first term's biased exponents
  uint8_t* hq;           // the hidden values likewise, by pairs (token * top + slot)
  uint8_t* hs;
  float* o;              // [parts][tokens * top][dim]
  int* plan;             // of more pairs than kSmall: see below
  int parts;             // of K in the second product
  int vec;               // x rows and the router allow 16-byte loads
};

template <int TYPE>
__device__ __forceinline__ void load_n(const void* p, long long at, bool vec, float* v) {
  constexpr int V = Storage<TYPE>::per16;
  const auto* q = static_cast<const typename Storage<TYPE>::raw*>(p) + at;
  if (vec) {
    decode16<TYPE>(*reinterpret_cast<const u32x4*>(q), v);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = decode<TYPE>(q[j]);
  }
}

// Sum over the wavefront.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, 0xF, 0xF, true);
  const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(lo)) | static_cast<uint64_t>(hi) << 32);
}
__device__ __forceinline__ double wave_sum(double v) {
  v += dpp_f64<0xB1>(v);     // lanes 1, 2, then 4 and 8 (mirrors) away
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  v += dpp_f64<0x140>(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// Bytes of a row of scales: those of four steps, whole.
__host__ __device__ __forceinline__ int scale_row(int k) { return (k / 32 + 15) & ~15; }

// Biased exponent of the first of N terms for a block whose largest magnitude is `top`; 255, NaN, where that is not
// finite.
template <int N>
__device__ __forceinline__ uint32_t block_scale(float top) {
  if (!(top <= 3.402823466e38f)) return 255;
  int e = -127;
  if (top > 0.f) (void)frexpf(top, &e);
  return max(e - 8 + 127, 4 * (N - 1));
}

// 2^(biased - 127) and its inverse, exactly.
__device__ __forceinline__ float power(int biased) { return biased <= 0 ? __uint_as_float(0x00400000u) : __uint_as_float(biased << 23); }

// Four values as N dwords of e4m3, v being what is left; nothing is where the scale is 255.
template <int N>
__device__ __forceinline__ void e4m3_terms(float (&v)[4], uint32_t scale, uint32_t (&out)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int b = static_cast<int>(scale) - 4 * n;
    const float down = scale == 255 ? 0.f : power(254 - b), up = power(b);
    float t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      t[j] = v[j] * down;
      if (n < N - 1) t[j] = __builtin_rintf(t[j] * 4.f) * 0.25f;
    }
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], w, true);
    out[n] = scale == 255 ? 0 : static_cast<uint32_t>(w);
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[0] -= lo[0] * up;
    v[1] -= lo[1] * up;
    v[2] -= hi[0] * up;
    v[3] -= hi[1] * up;
  }
}

// A wavefront: one expert's logits of LT tokens.  The first eight experts' share the writing of x's terms (one wavefront
// alone took 11.5 us for 17 f32 tokens of 2752).
template <int TYPE, int RTYPE, int NX, int LT>
__global__ __launch_bounds__(64) void moe_logits(MoeArgs a) {
  constexpr int XV = Storage<TYPE>::per16, RV = Storage<RTYPE>::per16, V = XV > RV ? XV : RV;
  const int lane = threadIdx.x, e = blockIdx.x % a.experts, t0 = blockIdx.x / a.experts * LT;
  auto load_x = [&](int t, int d, float* x) {
#pragma unroll
    for (int j = 0; j < V; j += XV) load_n<TYPE>(a.x, min(t0 + t, a.tokens - 1) * a.x_stride + d + j, a.vec, x + j);
  };
  double acc[LT][2] = {};
#pragma unroll 4
  for (int d = lane * V; d < a.dim; d += 64 * V) {
    float r[V], x[LT][V];
#pragma unroll
    for (int j = 0; j < V; j += RV) load_n<RTYPE>(a.router, static_cast<long long>(e) * a.dim + d + j, a.vec, r + j);
    for (int t = 0; t < LT; ++t) load_x(t, d, x[t]);
#pragma unroll
    for (int t = 0; t < LT; ++t)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[t][j & 1] = fma(static_cast<double>(x[t][j]), static_cast<double>(r[j]), acc[t][j & 1]);
  }
  const int share = min(a.experts, 8);
  for (int d = (64 * e + lane) * V; e < share && d < a.dim; d += 64 * share * V) {
    for (int t = 0; t < LT && t0 + t < a.tokens; ++t) {
      float x[V], top = 0.f;
      load_x(t, d, x);
#pragma unroll
      for (int j = 0; j < V; ++j) top = x[j] == x[j] ? fmaxf(top, fabsf(x[j])) : INFINITY;
      top = fmaxf(top, dpp_f32<0xB1>(top));                // a block: 4 lanes, or 8
      top = fmaxf(top, dpp_f32<0x4E>(top));
      if (V == 4) top = fmaxf(top, dpp_f32<0x141>(top));
      const uint32_t scale = block_scale<NX>(top);
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        float v[4] = {x[j], x[j + 1], x[j + 2], x[j + 3]};
        uint32_t w[NX];
        e4m3_terms<NX>(v, scale, w);
#pragma unroll
        for (int n = 0; n < NX; ++n)
          *reinterpret_cast<uint32_t*>(a.xq + (static_cast<long long>(n) * a.tokens + t0 + t) * a.dim + d + j) = w[n];
      }
      if (d % 32 == 0) a.xs[static_cast<long long>(t0 + t) * scale_row(a.dim) + d / 32] = static_cast<uint8_t>(scale);
    }
  }
#pragma unroll
  for (int t = 0; t < LT; ++t) {
    const double sum = wave_sum(acc[t][0] + acc[t][1]);
    if (lane == 0 && t0 + t < a.tokens)
      a.logits[static_cast<long long>(t0 + t) * a.experts + e] = sum + (a.bias != nullptr ? a.bias[e] : 0.f);
  }
}

// A token's logits into LDS, NaN as the lowest; an even number of them.
template <int NT>
__device__ __forceinline__ void load_logits(const MoeArgs& a, int t, double* l) {
  for (int e = threadIdx.x; e < ((a.experts + 1) & ~1); e += NT) {
    const double v = e < a.experts ? a.logits[static_cast<long long>(t) * a.experts + e] : -INFINITY;
    l[e] = v == v ? v : -INFINITY;
  }
  __syncthreads();
}

// How many experts come before e: those of larger logits, and of equal ones of lower indexes.
__device__ __forceinline__ int rank_of(const double* l, int experts, int e) {
  typedef double f64x2 __attribute__((ext_vector_type(2)));
  const double mine = l[e];
  int n = 0;
#pragma unroll 4
  for (int i = 0; i < experts; i += 2) {
    const f64x2 v = *reinterpret_cast<const f64x2*>(l + i);
    n += v[0] > mine || (v[0] == mine && i < e) ? 1 : 0;
    n += v[1] > mine || (v[1] == mine && i + 1 < e) ? 1 : 0;   // (the one that evens them comes last)
  }
  return n;
}

// A token's experts and shares: l its logits, in LDS; s_sum: NT / 64 + 1 doubles there.  Slots for which wanted(s)
// holds are handed to put(s, expert, share).
template <int NT, class Wanted, class Put>
__device__ __forceinline__ void shares_of(const MoeArgs& a, const double* l, double* s_sum, Wanted&& wanted, Put&& put) {
  constexpr int PER = kMaxExperts / NT;
  const int tid = threadIdx.x;
  int rank[PER];
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = tid + i * NT;
    rank[i] = e < a.experts ? rank_of(l, a.experts, e) : kMaxExperts;
    if (rank[i] == 0) s_sum[NT / 64] = l[e];
  }
  __syncthreads();
  const double first = s_sum[NT / 64];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (rank[i] < (a.normalize ? a.top : kMaxExperts)) sum += exp(l[tid + i * NT] - first);
  sum = wave_sum(sum);
  if ((tid & 63) == 0) s_sum[tid >> 6] = sum;
  __syncthreads();
  sum = 0.0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) sum += s_sum[w];
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (rank[i] < a.top && wanted(rank[i]))
      put(rank[i], tid + i * NT, static_cast<float>(exp(l[tid + i * NT] - first) / sum * a.scale));
}

// The pairs (token * top + slot) by their experts: plan[0] experts that any token chose, plan[1 + u] the u-th of them,
// plan[1 + E + u] where its pairs begin in order = plan + 2 + 2 E (and one past the last's).  The order within an
// expert's does not matter: a pair's sums do not depend on its place.  A workgroup of NT threads; n: E counts in LDS.
template <int NT>
__device__ __forceinline__ void make_plan(const MoeArgs& a, int* n, int* s_wave) {
  const int tid = threadIdx.x, pairs = a.tokens * a.top, E = a.experts;
  for (int e = tid; e < E; e += NT) n[e] = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += NT) atomicAdd(n + a.ids[i], 1);
  __syncthreads();
  // starts and ranks of the experts that are hit, a chunk of NT at a time
  int start = 0, rank = 0;
  for (int e0 = 0; e0 < E; e0 += NT) {
    const int e = e0 + tid, mine = e < E ? n[e] : 0;
    const uint64_t some = __ballot(mine > 0);
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int below = __shfl_up(sum, o);
      if ((tid & 63) >= o) sum += below;
    }
    if ((tid & 63) == 63) {
      s_wave[tid >> 6] = sum;
      s_wave[NT / 64 + (tid >> 6)] = __popcll(some);
    }
    __syncthreads();
    int at = start + sum - mine, r = rank + __popcll(some & ((1ull << (tid & 63)) - 1));
    for (int w = 0; w < NT / 64; ++w) {
      if (w < tid >> 6) {
        at += s_wave[w];
        r += s_wave[NT / 64 + w];
      }
      start += s_wave[w];
      rank += s_wave[NT / 64 + w];
    }
    if (mine > 0) {
      a.plan[1 + r] = e;
      a.plan[1 + E + r] = at;
    }
    if (e < E) n[e] = at;
    __syncthreads();
  }
  if (tid == 0) {
    a.plan[0] = rank;
    a.plan[1 + E + rank] = pairs;
  }
  for (int i = tid; i < pairs; i += NT) a.plan[2 + 2 * E + atomicAdd(n + a.ids[i], 1)] = i;
}

// A workgroup a token, and one for the plan.
__global__ __launch_bounds__(256) void moe_select(MoeArgs a) {
  __shared__ __attribute__((aligned(16))) double l[kMaxExperts];
  __shared__ double s_sum[5];
  const int t = blockIdx.x;
  load_logits<256>(a, t, l);
  shares_of<256>(a, l, s_sum, [](int) { return true; },
                 [&](int s, int e, float p) {
                   a.ids[t * a.top + s] = e;
                   a.shares[t * a.top + s] = p;
                 });
}
__global__ __launch_bounds__(1024) void moe_plan(MoeArgs a) {
  __shared__ int n[kMaxExperts], s_wave[32];
  make_plan<1024>(a, n, s_wave);
}

// Both in one workgroup: a thread takes logits of any token.  For few comparisons, tokens * experts^2: one launch of 7.6 us
// (8 tokens, 64 experts) in place of two of 4.3 and 3.1 and the gap between; 64 tokens, 64 experts: 28 us.  Of a pass of 512
// tokens and kCompare comparisons there are (512 kCompare)^1/2 logits at most.
constexpr int kCompare = 1 << 16, kSelect = 6 * 1024;
static_assert(1LL * kSelect * kSelect >= 1LL * kPass * kCompare, "room for the logits");
__global__ __launch_bounds__(1024) void moe_select_few(MoeArgs a) {
  __shared__ __attribute__((aligned(16))) double l[kSelect + 2];
  __shared__ double first[kPass];
  __shared__ int n[kMaxExperts], s_wave[32];
  const int tid = threadIdx.x, E = a.experts, all = a.tokens * E;
  for (int i = tid; i < all; i += 1024) {
    const double v = a.logits[i];
    l[i] = v == v ? v : -INFINITY;
  }
  __syncthreads();
  int rank[kSelect / 1024];
#pragma unroll
  for (int k = 0; k < kSelect / 1024; ++k) {
    const int i = tid + 1024 * k;
    rank[k] = kMaxExperts;
    if (i >= all) continue;
    const int t = i / E, e = i - t * E;
    const double mine = l[i], *row = l + t * E;
    int r = 0;
    for (int j = 0; j < E; ++j) r += row[j] > mine || (row[j] == mine && j < e) ? 1 : 0;
    rank[k] = r;
    if (r == 0) first[t] = mine;
  }
  __syncthreads();
  double v[kSelect / 1024];
#pragma unroll
  for (int k = 0; k < kSelect / 1024; ++k) {
    const int i = tid + 1024 * k;
    v[k] = i < all ? exp(l[i] - first[i / E]) : 0.0;
  }
  __syncthreads();
  // the row's terms in the order of their sum: the chosen by rank, or all
#pragma unroll
  for (int k = 0; k < kSelect / 1024; ++k) {
    const int i = tid + 1024 * k;
    if (i < all && (!a.normalize || rank[k] < a.top)) l[a.normalize ? i / E * E + rank[k] : i] = v[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSelect / 1024; ++k) {
    const int i = tid + 1024 * k;
    if (rank[k] >= a.top) continue;
    const int t = i / E, slot = t * a.top + rank[k];
    double sum = 0.0;
    for (int j = 0; j < (a.normalize ? a.top : E); ++j) sum += l[t * E + j];
    a.ids[slot] = i - t * E;
    a.shares[slot] = static_cast<float>(v[k] / sum * a.scale);
  }
  __threadfence_block();
  __syncthreads();
  make_plan<1024>(a, n, s_wave);
}

// act(gate) * up
__device__ __forceinline__ float gated(bool gelu, float v, float u) {
  if (gelu) return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v))) * u;
  return v / (1.0f + expf(-v)) * u;
}

// Largest over the four lanes of a column.
__device__ __forceinline__ float lanes16_max(float v) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// The hidden values of rows r0 .. r0 + 31 of a pair, from tiles of 16 gate and up rows: lane l has column l & 15,
// rows 4 (l >> 4) + e of each.  All lanes take part; `in`: the lane's column is one.
template <int NH>
__device__ __forceinline__ void store_hidden(const MoeArgs& a, const f32x4* gate, const f32x4* up, long long pair, int r0, bool in) {
  const long long pairs = static_cast<long long>(a.tokens) * a.top;
  const int g = (threadIdx.x & 63) >> 4;
  float v[2][4], top = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[i][e] = gated(a.gelu, gate[i][e], up[i][e]);
      top = v[i][e] == v[i][e] ? fmaxf(top, fabsf(v[i][e])) : INFINITY;
    }
  const uint32_t scale = block_scale<NH>(lanes16_max(top));
  if (!in) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t w[NH];
    e4m3_terms<NH>(v[i], scale, w);
#pragma unroll
    for (int n = 0; n < NH; ++n)
      *reinterpret_cast<uint32_t*>(a.hq + (n * pairs + pair) * a.inter + r0 + 16 * i + 4 * g) = w[n];
  }
  if (g == 0) a.hs[pair * scale_row(a.inter) + r0 / 32] = static_cast<uint8_t>(scale);
}

// Barrier after which LDS that the waves have written can be read, and what they have read be overwritten; loads from
// memory go on.
__device__ __forceinline__ void lds_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- Products -------------------------------------------------------------------
//
// A step is 128 elements of K, four blocks of 32.  Lane l of a wavefront holds, of a tile of 16 rows of w, block
// 4 step + (l >> 4) of row l & 15 and its scale byte, of a term of x the same block of column l & 15.

// The MFMA is not known to need all lanes: without this the compiler moves the last one, and what it takes, under
// a branch that some lanes skip.
__device__ __forceinline__ void settle(f32x4& v) { asm volatile("" : "+v"(v)); }

// Where a wavefront finds R tiles of 16 rows of w; lane l reads row l & 15 of each.
template <int R>
struct Rows {
  const uint8_t* codes[R];    // of the tile's first row
  const uint8_t* scales[R];
  uint32_t last[R];           // the last place from scales on that 8 bytes can be read at
  uint32_t code_row, scale_row;
  int blocks;                 // of a row
  __device__ __forceinline__ void begin(int k) {
    blocks = k / 32;
    code_row = (threadIdx.x & 15) * static_cast<uint32_t>(blocks) * 16;
    scale_row = (threadIdx.x & 15) * static_cast<uint32_t>(blocks);
  }
  // tile i from `row` on, of `rows` in the matrices at c and s
  __device__ __forceinline__ void set(int i, const uint8_t* c, const uint8_t* s, long long row, long long rows) {
    codes[i] = c + row * blocks * 16;
    scales[i] = s + row * blocks;
    last[i] = static_cast<uint32_t>(min((rows - row) * blocks - 8, 0x7FFFFFFFll));
  }
};

// Codes of a step.
template <int R>
struct Codes {
  u32x4 w[R];
  __device__ __forceinline__ void load(const Rows<R>& r, int step) {
    const int b = min(4 * step + static_cast<int>((threadIdx.x & 63) >> 4), r.blocks - 1);   // past K: x is zero there
    const uint32_t at = r.code_row + 16u * b;
#pragma unroll
    for (int i = 0; i < R; ++i) w[i] = *reinterpret_cast<const u32x4*>(r.codes[i] + at);
  }
};

// Scales of two steps: 8 bytes of a row, the same for its four lanes (a byte a step and lane asks for as many lines as the
// codes do: 64 tokens through 8 experts of 4096 x 14336, 207 + 131 us so, 143 + 93 with 16 bytes for four steps).  A
// row's last ones come with the next row's first, the array's with the ones before, to be shifted down.
template <int R>
struct Scales {
  u32x2 w[R];
  __device__ __forceinline__ void load(const Rows<R>& r, int step) {
    const uint32_t at = r.scale_row + 4u * min(step, (r.blocks - 1) >> 2);
#pragma unroll
    for (int i = 0; i < R; ++i) __builtin_memcpy(&w[i], r.scales[i] + min(at, r.last[i]), 8);
  }
  // once they are there; `step` as loaded
  __device__ __forceinline__ void arrange(const Rows<R>& r, int step) {
    const uint32_t at = r.scale_row + 4u * min(step, (r.blocks - 1) >> 2);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const uint64_t v = __builtin_bit_cast(uint64_t, w[i]);
      w[i] = __builtin_bit_cast(u32x2, v >> (8 * (at - min(at, r.last[i]))));
    }
  }
};

// acc + a tile's codes w under the scale byte `scale` times a term of x under the biased exponent sx: of the step's eight 16-byte chunks of e4m3 a lane holds two, l >> 4 and 4 + (l >> 4).
__device__ __forceinline__ f32x4 times(const u32x4& w, int scale, const u32x4& lo, const u32x4& hi, int sx, const f32x4& acc) {
  i32x8 A, B;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    A[e] = w[e];
    B[e] = lo[e];
    B[e + 4] = hi[e];
  }
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, acc, 4, 0, 0, scale, 0, sx);
}

// The lane's byte of a step's dword; any finite one past K, where x is zero.
__device__ __forceinline__ int scale_of(uint32_t w, int step, int blocks) {
  const int g = (threadIdx.x & 63) >> 4;
  return 4 * step + g < blocks ? w >> (8 * g) & 255 : 127;
}

// Few pairs: each on its own, one column of x.  It goes to LDS in parts of K.  Three launches, each a chain of dependent
// reads: one bf16 token, 8 of 64 experts of 2048 x 1024 (27 MB, 5.6 us of bytes) 4.6 + 10.2 + 7.0 us.
//
// Hidden rows: workgroup (pair, 32 rows); its four waves take a quarter of the steps each.  The expert is found from the
// logits by each workgroup for itself, and written by the first of the pair.
constexpr int kUpPart = 8192;
template <int NX, int NH>
__global__ __launch_bounds__(256) void moe_small_up(MoeArgs a, int tiles) {
  constexpr int D = 4;
  __shared__ __attribute__((aligned(16))) double l[kMaxExperts];
  __shared__ double s_sum[5];
  __shared__ int s_expert;
  __shared__ __attribute__((aligned(16))) uint8_t s_x[NX][kUpPart];
  __shared__ uint8_t s_xs[kUpPart / 32];
  __shared__ f32x4 s_acc[3][4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int pair = blockIdx.x / tiles, tile = blockIdx.x - pair * tiles, t = pair / a.top, slot = pair - t * a.top;
  auto stage = [&](int k0) {
    const int n = min(kUpPart, a.dim - k0);
    for (int k = 16 * tid; k < ((n + 127) & ~127); k += 16 * 256)
#pragma unroll
      for (int i = 0; i < NX; ++i)
        *reinterpret_cast<u32x4*>(s_x[i] + k) =
            k < n ? *reinterpret_cast<const u32x4*>(a.xq + (static_cast<long long>(i) * a.tokens + t) * a.dim + k0 + k)
                  : u32x4{0, 0, 0, 0};
    for (int k = tid; k < (n + 127) / 128 * 4; k += 256)
      s_xs[k] = k < n / 32 ? a.xs[static_cast<long long>(t) * scale_row(a.dim) + k0 / 32 + k] : 127;
  };
  stage(0);
  load_logits<256>(a, t, l);
  if (tile == 0) {
    shares_of<256>(a, l, s_sum, [&](int s) { return s == slot; },
                   [&](int, int e, float p) {
                     a.ids[pair] = e;
                     a.shares[pair] = p;
                     s_expert = e;
                   });
  } else {
    for (int e = tid; e < a.experts; e += 256)
      if (rank_of(l, a.experts, e) == slot) s_expert = e;
  }
  __syncthreads();
  const int expert = __builtin_amdgcn_readfirstlane(s_expert);
  Rows<4> r;                                                // tiles: gate, gate, up, up
  r.begin(a.dim);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.set(i, a.gu, a.gus, (2ll * expert + (i >> 1)) * a.inter + 32 * tile + 16 * (i & 1), 2ll * a.experts * a.inter);
  f32x4 acc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.dim; k0 += kUpPart) {
    // the wave's steps of this part of K, D at a time
    const int base = k0 / 128, all = (min(a.dim - k0, kUpPart) + 127) / 128;
    const int first = base + all * wave / 4, end = base + all * (wave + 1) / 4, last = max(end - 1, first);
    Codes<4> w[D];
    Scales<4> sc[D / 2];
#pragma unroll
    for (int d = 0; d < D; d += 2) sc[d / 2].load(r, first + d);
#pragma unroll
    for (int d = 0; d < D; ++d) w[d].load(r, min(first + d, last));
    if (k0 > 0) {
      __syncthreads();
      stage(k0);
      __syncthreads();
    }
    auto multiply = [&](const Codes<4>& v, const Scales<4>& sv, int d, int s) {
      const int at = 128 * (s - base), sx = s_xs[at / 32 + g];
      int sw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sw[i] = scale_of(sv.w[i][d & 1], s, r.blocks);
#pragma unroll
      for (int n = 0; n < NX; ++n) {
        const u32x4* x = reinterpret_cast<const u32x4*>(s_x[n] + at);
        const u32x4 lo = x[g], hi = x[4 + g];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = times(v.w[i], sw[i], lo, hi, sx - 4 * n, acc[i]);
      }
    };
    int s0 = first;
    for (; s0 + D < end; s0 += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (d % 2 == 0) sc[d / 2].arrange(r, s0 + d);
        multiply(w[d], sc[d / 2], d, s0 + d);
        __builtin_amdgcn_sched_barrier(0);
        w[d].load(r, min(s0 + d + D, last));
        if (d % 2 == 1) sc[d / 2].load(r, s0 + d - 1 + D);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (d % 2 == 0) sc[d / 2].arrange(r, s0 + d);
      if (s0 + d < end) multiply(w[d], sc[d / 2], d, s0 + d);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) settle(acc[i]);
  if (wave > 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_acc[wave - 1][i][lane] = acc[i];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int p = 0; p < 3; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += s_acc[p][i][lane];
  store_hidden<NH>(a, acc, acc + 2, pair, 32 * tile, (lane & 15) == 0);
}

// Outputs: workgroup 16 rows of all pairs' experts, its sixteen waves shared among the pairs; the sums over K and
// over the pairs of a token in order.
constexpr int kDownLds = 49152;      // bytes of the hidden values in LDS
// Whether a pass is worked on pair by pair: not where rows are so long that this launch's work-items, 64 of dim, pass 32 bits.
bool pair_by_pair(long long pairs, long long dim) { return pairs <= kSmall && dim / 16 <= static_cast<long long>(UINT32_MAX) / 1024; }
template <int TYPE, int NH>
__global__ __launch_bounds__(1024) void moe_small_down(MoeArgs a, int shift) {   // 2^shift waves a pair
  typedef typename Storage<TYPE>::raw raw;
  constexpr int D = 4;
  __shared__ __attribute__((aligned(16))) uint8_t s_h[kDownLds];
  __shared__ uint8_t s_hs[kDownLds / 32];
  __shared__ f32x4 s_acc[16][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int pairs = a.tokens * a.top, r0 = 16 * blockIdx.x;
  const int pair = wave >> shift, part = wave & ((1 << shift) - 1);
  const bool busy = pair < pairs;
  const int expert = __builtin_amdgcn_readfirstlane(a.ids[busy ? pair : 0]);
  Rows<1> rows;
  rows.begin(a.inter);
  rows.set(0, a.dn, a.dns, static_cast<long long>(expert) * a.dim + r0, static_cast<long long>(a.experts) * a.dim);
  const int most = kDownLds / (pairs * NH) & ~127;         // elements of K at a time
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < a.inter; k0 += most) {
    const int n = min(most, a.inter - k0), wide = (n + 127) & ~127, chunks = wide / 16;
    // the wave's steps of this part of K, D at a time
    const int base = k0 / 128, all = wide / 128;
    const int first = base + (all * part >> shift), end = base + (all * (part + 1) >> shift), last = max(end - 1, first);
    Codes<1> w[D];
    Scales<1> sc[D / 2];
#pragma unroll
    for (int d = 0; d < D; d += 2) sc[d / 2].load(rows, first + d);
#pragma unroll
    for (int d = 0; d < D; ++d) w[d].load(rows, min(first + d, last));
    if (k0 > 0) __syncthreads();
    for (int i = tid; i < pairs * NH * chunks; i += 1024) {
      const int r = i / chunks, k = 16 * (i - r * chunks);  // row r: term r / pairs of pair r % pairs
      *reinterpret_cast<u32x4*>(s_h + r * wide + k) =
          k < n ? *reinterpret_cast<const u32x4*>(a.hq + static_cast<long long>(r) * a.inter + k0 + k) : u32x4{0, 0, 0, 0};
    }
    for (int i = tid; i < pairs * (wide / 32); i += 1024) {
      const int r = i / (wide / 32), k = i - r * (wide / 32);
      s_hs[i] = k < n / 32 ? a.hs[static_cast<long long>(r) * scale_row(a.inter) + k0 / 32 + k] : 127;
    }
    lds_sync();
    if (!busy) continue;
    auto multiply = [&](const Codes<1>& v, const Scales<1>& sv, int d, int s) {
      const int at = 128 * (s - base), sx = s_hs[(pair * wide + at) / 32 + g], sw = scale_of(sv.w[0][d & 1], s, rows.blocks);
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        const u32x4* x = reinterpret_cast<const u32x4*>(s_h + (i * pairs + pair) * wide + at);
        acc = times(v.w[0], sw, x[g], x[4 + g], sx - 4 * i, acc);
      }
    };
    int s0 = first;
    for (; s0 + D < end; s0 += D)
#pragma unroll
      for (int d = 0; d < D; ++d) {
        if (d % 2 == 0) sc[d / 2].arrange(rows, s0 + d);
        multiply(w[d], sc[d / 2], d, s0 + d);
        __builtin_amdgcn_sched_barrier(0);
        w[d].load(rows, min(s0 + d + D, last));
        if (d % 2 == 1) sc[d / 2].load(rows, s0 + d - 1 + D);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
    for (int d = 0; d < D; ++d) {
      if (d % 2 == 0) sc[d / 2].arrange(rows, s0 + d);
      if (s0 + d < end) multiply(w[d], sc[d / 2], d, s0 + d);
    }
  }
  settle(acc);
  if ((lane & 15) == 0) s_acc[wave][g] = acc;
  __syncthreads();
  const int t = tid >> 4, d = tid & 15;
  if (t >= a.tokens) return;
  float v = a.residual != nullptr ? decode<TYPE>(static_cast<const raw*>(a.residual)[t * a.residual_stride + r0 + d]) : 0.f;
  for (int s = 0; s < a.top; ++s) {
    float sum = 0.f;
    for (int p = 0; p < 1 << shift; ++p) sum += s_acc[((t * a.top + s) << shift) + p][d >> 2][d & 3];
    v += a.shares[t * a.top + s] * sum;
  }
  static_cast<raw*>(a.y)[t * a.y_stride + r0 + d] = encode<TYPE>(v);
}

// More pairs, by their experts.
//
// Workgroup: 256 rows of w, 64 by wave (UP: 32 gate and 32 up rows of the same hidden ones), and CT tiles of 16 columns.
// K goes in chunks of Q steps.  Codes come straight to registers, a chunk ahead; x, which all waves share, and the scales,
// 4 Q bytes of a row at a time, by way of LDS, a chunk ahead too, with one barrier a chunk: 16-byte piece c of column n's
// chunk lies at place c ^ (n & 15), so that an MFMA's reads meet in no bank.
//
// What bounds it is what a wave has to do beside the MFMAs, as few of them fit a SIMD: a barrier and new addresses each step
// (140 VALU instructions beside 16 MFMAs, all operands through an LDS ring) took 172 + 91 us for 64 tokens through 8 experts
// of 4096 x 14336, a byte of scales a lane and step 207 + 131; so 140 + 73 by
// the same clock, the first passes of a process, and 125 + 65 later: 500 and 250 MB, 4.0 and 3.8 TB/s.  Codes or
// scales two chunks ahead change nothing (17 f32 tokens through 25 of 2752 x 1376: 37.4 us, 38.0 and 38.2).
template <int CT, int NX>
struct Chunk {
  static constexpr int Q = 2;
  static constexpr int kRow = 128 * Q;                                   // bytes of a column and term
  static constexpr int PER = CT * 16 * NX * kRow / 16 / 256;             // 16-byte pieces a thread
  static constexpr int WAVES = CT * NX >= 12 ? 1 : CT == 1 && NX < 6 ? 3 : 2;   // a SIMD: what LDS, then registers hold
};

template <bool UP, int CT, int NX, int NH>
__global__ __launch_bounds__(256, (Chunk<CT, NX>::WAVES)) void moe_rows(MoeArgs a, int tiles) {
  typedef Chunk<CT, NX> C;
  constexpr int Q = C::Q, PER = C::PER, kRow = C::kRow;
  __shared__ __attribute__((aligned(1024))) uint8_t s_x[2][CT * 16 * NX * kRow];
  __shared__ __attribute__((aligned(16))) uint32_t s_scale[2][256][Q], s_xs[2][CT * 16][Q];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4;
  const int parts = UP ? 1 : a.parts, E = a.experts;
  const int part = blockIdx.x % parts, tile = blockIdx.x / parts % tiles, u = blockIdx.x / parts / tiles;
  const int* plan = a.plan;
  if (u >= plan[0]) return;
  const int expert = __builtin_amdgcn_readfirstlane(plan[1 + u]);
  const int first = __builtin_amdgcn_readfirstlane(plan[1 + E + u]), count = __builtin_amdgcn_readfirstlane(plan[2 + E + u]) - first;
  const int* list = plan + 2 + 2 * E + first;
  const int K = UP ? a.dim : a.inter, blocks = K / 32, all = (blocks + 3) / 4, rows = UP ? a.inter : a.dim;
  const int s0 = all * part / parts, s1 = all * (part + 1) / parts;     // steps
  // the wave's 64 rows: two halves of 32, where they are there
  const int r0 = (tile * 4 + wave) * (UP ? 32 : 64);
  const bool real = r0 < rows;
  long long row[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = UP ? r0 : r0 + 32 * i, in = at < rows ? at : 0;
    row[i] = UP ? (2ll * expert + i) * a.inter + in : static_cast<long long>(expert) * a.dim + in;
  }
  const long long all_rows = (UP ? 2ll * a.inter : static_cast<long long>(a.dim)) * E;
  Rows<4> rw;
  rw.begin(K);
#pragma unroll
  for (int t = 0; t < 4; ++t) rw.set(t, UP ? a.gu : a.dn, UP ? a.gus : a.dns, row[t >> 1] + 16 * (t & 1), all_rows);
  // scales: a row a lane, 4 Q bytes from the one that the array's last ones are before
  const uint8_t* scales = UP ? a.gus : a.dns;
  const long long srow = ((lane < 32 ? row[0] : row[1]) + (lane & 31)) * blocks;
  const uint8_t* sfrom = scales + srow;
  const int sleft = static_cast<int>(min(all_rows * blocks - 4 * Q - srow, 0x7FFFFFFFll));
  const long long pairs = static_cast<long long>(a.tokens) * a.top;
  const uint8_t* src = UP ? a.xq : a.hq;
  const uint8_t* src_scales = UP ? a.xs : a.hs;
  const long long src_term = (UP ? a.tokens : pairs) * K;
  const int xs_row = scale_row(K);
  int xat[2][2];                                            // a column's piece of even and odd steps, low and high half
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) xat[i][h] = (lane & 15) * kRow + (((8 * i + 4 * h + g) ^ (lane & 15)) * 16);

  for (int c0 = 0; c0 < count; c0 += 16 * CT) {
    // the thread's pieces of x: of columns past the last that one again, past K zeros
    static_assert(256 % (8 * Q) == 0, "a thread's pieces are at one place of their rows");
    const int piece = 16 * (tid % (8 * Q));
    uint32_t from[PER];                                     // (the host keeps a pass's terms below 4 GB)
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int r = (tid + i * 256) / (8 * Q), n = r / (16 * CT), col = r % (16 * CT);
      const int pair = list[min(c0 + col, count - 1)];
      from[i] = static_cast<uint32_t>(n * src_term + static_cast<long long>(UP ? pair / a.top : pair) * K);
    }
    const int xs_id = min(tid, CT * 16 * Q - 1), xs_pair = list[min(c0 + xs_id / Q, count - 1)];
    const uint32_t xs_from = static_cast<uint32_t>(UP ? xs_pair / a.top : xs_pair) * static_cast<uint32_t>(xs_row);

    u32x4 xr[PER];
    uint32_t xsr, sr[Q];
    auto load_x = [&](int s) {                              // of steps s .. s + Q - 1
#pragma unroll
      for (int i = 0; i < PER; ++i)
        xr[i] = *reinterpret_cast<const u32x4*>(src + (from[i] + static_cast<uint32_t>(min(128 * s + piece, K - 16))));
      xsr = *reinterpret_cast<const uint32_t*>(src_scales + (xs_from + static_cast<uint32_t>(min(4 * (s + xs_id % Q), xs_row - 4))));
      __builtin_memcpy(sr, sfrom + min(4 * min(s, all - 1), sleft), 4 * Q);
    };
    auto put_x = [&](int s, int buffer) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int id = tid + i * 256, r = id / (8 * Q), c = id % (8 * Q);
        *reinterpret_cast<u32x4*>(s_x[buffer] + r * kRow + ((c ^ (r & 15)) * 16)) =
            128 * s + piece < K ? xr[i] : u32x4{0, 0, 0, 0};
      }
      auto finite = [&](uint32_t v, int step) {             // past K: zeros under any finite scale
        const int left = blocks - 4 * step;
        const uint32_t keep = left >= 4 ? ~0u : (1u << (8 * max(left, 0))) - 1;
        return (v & keep) | (0x7F7F7F7Fu & ~keep);
      };
      if (tid < CT * 16 * Q) s_xs[buffer][xs_id / Q][xs_id % Q] = finite(xsr, s + xs_id % Q);
      // what is past the array's end is not needed
      const uint32_t by = max(4 * min(s, all - 1) - sleft, 0), bits = 8 * (by & 3);
#pragma unroll
      for (int d = 0; d < Q; ++d) {
        uint32_t lo = sr[d], hi = d + 1 < Q ? sr[d + 1] : 0;
#pragma unroll
        for (int e = 1; e < Q; ++e)
          if (by >> 2 == static_cast<uint32_t>(e)) {
            lo = d + e < Q ? sr[d + e < Q ? d + e : 0] : 0;
            hi = d + e + 1 < Q ? sr[d + e + 1 < Q ? d + e + 1 : 0] : 0;
          }
        s_scale[buffer][tid][d] = finite(__builtin_amdgcn_alignbit(hi, lo, bits), s + d);
      }
    };
    f32x4 acc[4][CT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < CT; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    Codes<4> w[Q];
    auto multiply = [&](const Codes<4>& v, int d, int buffer) {
      int sw[4], sx[CT];
#pragma unroll
      for (int t = 0; t < 4; ++t) sw[t] = s_scale[buffer][64 * wave + 16 * t + (lane & 15)][d] >> (8 * g);   // (the low byte counts)
#pragma unroll
      for (int i = 0; i < CT; ++i) sx[i] = s_xs[buffer][16 * i + (lane & 15)][d] >> (8 * g);
#pragma unroll
      for (int n = 0; n < NX; ++n)
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const uint8_t* x = s_x[buffer] + (n * CT + i) * 16 * kRow + 256 * (d >> 1);
          const u32x4 lo = *reinterpret_cast<const u32x4*>(x + xat[d & 1][0]), hi = *reinterpret_cast<const u32x4*>(x + xat[d & 1][1]);
#pragma unroll
          for (int t = 0; t < 4; ++t) acc[t][i] = times(v.w[t], sw[t], lo, hi, sx[i] - 4 * n, acc[t][i]);
        }
    };
    // (no load under a condition: the compiler would wait for all of them where the ways meet)
    // Loads and MFMAs stay as they are written: a load of codes that the compiler moves up takes registers of its own, to be
    // waited for and copied at the loop's end.
    auto in_order = [](f32x4 (&v)[4][CT]) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < CT; ++i) settle(v[t][i]);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    load_x(s0);
    in_order(acc);
#pragma unroll
    for (int d = 0; d < Q; ++d) w[d].load(rw, min(s0 + d, s1 - 1));
    in_order(acc);
    if (c0 > 0) lds_sync();                                 // everyone has read the last chunk
    put_x(s0, 0);
    int buffer = 0, s = s0;
    for (; s + Q < s1; s += Q) {
      lds_sync();
      load_x(s + Q);
      in_order(acc);
#pragma unroll
      for (int d = 0; d < Q; ++d) {
        multiply(w[d], d, buffer);
        in_order(acc);
        w[d].load(rw, min(s + d + Q, s1 - 1));
        in_order(acc);
      }
      buffer ^= 1;
      put_x(s + Q, buffer);
    }
    lds_sync();
#pragma unroll
    for (int d = 0; d < Q; ++d)
      if (s + d < s1) multiply(w[d], d, buffer);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < CT; ++i) settle(acc[t][i]);
    if (!real) continue;
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int at = c0 + 16 * i + (lane & 15);
      const bool in = at < count;
      const int pair = list[min(at, count - 1)];
      if constexpr (UP) {
        const f32x4 gate[2] = {acc[0][i], acc[1][i]}, up[2] = {acc[2][i], acc[3][i]};
        store_hidden<NH>(a, gate, up, pair, r0, in);
      } else if (in) {
        float* o = a.o + (part * pairs + pair) * a.dim + r0 + 4 * g;
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (r0 + 16 * t < a.dim) *reinterpret_cast<f32x4*>(o + 16 * t) = acc[t][i];
      }
    }
  }
}

// y = residual + the shares times the pairs' sums, in the order of their slots.
template <int TYPE>
__global__ __launch_bounds__(256) void moe_join(MoeArgs a) {
  typedef typename Storage<TYPE>::raw raw;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int quads = a.dim / 4, t = static_cast<int>(i / quads), d = static_cast<int>(i - static_cast<long long>(t) * quads) * 4;
  if (t >= a.tokens) return;
  const long long pairs = static_cast<long long>(a.tokens) * a.top;
  const raw* r = static_cast<const raw*>(a.residual) + t * a.residual_stride + d;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (a.residual != nullptr)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = decode<TYPE>(r[e]);
  for (int s = 0; s < a.top; ++s) {
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < a.parts; ++p)
      sum += *reinterpret_cast<const f32x4*>(a.o + (p * pairs + static_cast<long long>(t) * a.top + s) * a.dim + d);
    v += a.shares[t * a.top + s] * sum;
  }
  raw* y = static_cast<raw*>(a.y) + t * a.y_stride + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = encode<TYPE>(v[e]);
}

template <bool UP, int N, int NH>
hipError_t run_rows(const MoeArgs& a, int hits, hipStream_t s) {
  const int pairs = a.tokens * a.top, tiles = UP ? (a.inter + 127) / 128 : (a.dim + 255) / 256;
  const unsigned grid = static_cast<unsigned>(hits) * tiles * (UP ? 1 : a.parts);
  if (a.tokens <= 16 || pairs <= 10 * hits) moe_rows<UP, 1, N, NH><<<grid, 256, 0, s>>>(a, tiles);
  else if (a.tokens <= 32 || pairs <= 24 * hits || N > 3) moe_rows<UP, 2, N, NH><<<grid, 256, 0, s>>>(a, tiles);
  else moe_rows<UP, (N > 3 ? 2 : 4), N, NH><<<grid, 256, 0, s>>>(a, tiles);   // (more terms than LDS holds)
  return hipGetLastError();
}

template <int TYPE, int NX, int LT>
hipError_t run_logits(const MoeArgs& a, hipStream_t s) {
  const unsigned grid = static_cast<unsigned>(a.experts) * ((a.tokens + LT - 1) / LT);
  switch (a.router_type) {
    case QC_STORAGE_F32: moe_logits<TYPE, QC_STORAGE_F32, NX, LT><<<grid, 64, 0, s>>>(a); break;
    case QC_STORAGE_F16: moe_logits<TYPE, QC_STORAGE_F16, NX, LT><<<grid, 64, 0, s>>>(a); break;
    default: moe_logits<TYPE, QC_STORAGE_BF16, NX, LT><<<grid, 64, 0, s>>>(a);
  }
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_pass(const MoeArgs& a, hipStream_t s) {
  constexpr int NX = TYPE == QC_STORAGE_F32 ? 6 : TYPE == QC_STORAGE_F16 ? 3 : 2;
  constexpr int NH = TYPE == QC_STORAGE_F32 ? 6 : TYPE == QC_STORAGE_F16 ? 4 : 3;
  const bool many = static_cast<long long>(a.tokens) * a.experts >= 16LL * device_cu_count();
  hipError_t e = many ? run_logits<TYPE, NX, 4>(a, s) : run_logits<TYPE, NX, 1>(a, s);
  if (e != hipSuccess) return e;
  const int pairs = a.tokens * a.top, hits = std::min(a.experts, pairs);
  if (pair_by_pair(pairs, a.dim)) {
    const int tiles = a.inter / 32;
    moe_small_up<NX, NH><<<static_cast<unsigned>(pairs) * tiles, 256, 0, s>>>(a, tiles);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    int shift = 0;
    while ((2 << shift) * pairs <= 16) ++shift;
    moe_small_down<TYPE, NH><<<a.dim / 16, 1024, 0, s>>>(a, shift);
    return hipGetLastError();
  }
  if (static_cast<long long>(a.tokens) * a.experts * a.experts <= kCompare) {
    moe_select_few<<<1, 1024, 0, s>>>(a);
  } else {
    moe_select<<<a.tokens, 256, 0, s>>>(a);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    moe_plan<<<1, 1024, 0, s>>>(a);
  }
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if ((e = run_rows<true, NX, NH>(a, hits, s)) != hipSuccess) return e;
  if ((e = run_rows<false, NH, NH>(a, hits, s)) != hipSuccess) return e;
  const long long quads = static_cast<long long>(a.tokens) * (a.dim / 4);
  moe_join<TYPE><<<static_cast<unsigned>((quads + 255) / 256), 256, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mxfp4_moe(const Moe& m, hipStream_t s) {
  const qc_mxfp4_moe& l = *m.layer;
  MoeArgs a = {};
  a.router = l.router;
  a.bias = l.router_bias;
  a.router_type = l.router_type;
  a.gu = l.gate_up_codes;
  a.gus = l.gate_up_scales;
  a.dn = l.down_codes;
  a.dns = l.down_scales;
  a.experts = static_cast<int>(l.experts);
  a.dim = static_cast<int>(l.dim);
  a.inter = static_cast<int>(l.inter);
  a.top = static_cast<int>(m.top);
  a.x_stride = m.x_stride;
  a.residual_stride = m.residual_stride;
  a.y_stride = m.y_stride;
  a.normalize = m.normalize;
  a.gelu = m.gelu_tanh;
  a.scale = m.scale;
  const int size = m.type == QC_STORAGE_F32 ? 4 : 2;
  a.vec = ((reinterpret_cast<uintptr_t>(m.x) | reinterpret_cast<uintptr_t>(l.router) |
            static_cast<uintptr_t>(m.x_stride * size)) & 15) == 0;
  const int nx = m.type == QC_STORAGE_F32 ? 6 : m.type == QC_STORAGE_F16 ? 3 : 2;
  const int nh = m.type == QC_STORAGE_F32 ? 6 : m.type == QC_STORAGE_F16 ? 4 : 3;
  // tokens of a pass: so that offsets into its terms fit 32 bits, and a grid over pairs and 32 rows of inter 2^32 threads
  const long long term_bytes = std::max<long long>(nx * l.dim, nh * static_cast<long long>(a.top) * l.inter);
  // (and so that the pairs' outputs, whose parts are one where rows are long, take 1 GB)
  const long long pass = std::max<long long>(1, std::min<long long>({kPass, (1LL << 32) / term_bytes - 1, (1LL << 28) / (a.top * l.inter),
                                                                    (1LL << 28) / (a.top * l.dim)}));
  const long long t = std::min(m.tokens, pass), pairs = t * a.top;
  // parts of K in the second product: workgroups for the chip twice, steps enough for each
  const long long down = std::min<long long>(a.experts, pairs) * ((a.dim + 255) / 256);
  a.parts = static_cast<int>(std::max<long long>(1, std::min<long long>({2LL * device_cu_count() / down, a.inter / 1024, 8})));
  const auto whole = [](long long n) { return (n + 255) / 256 * 256; };
  const long long parts[7] = {whole(t * a.experts * 8), whole(nx * t * a.dim), whole(t * scale_row(a.dim)),
                              whole(nh * pairs * a.inter), whole(pairs * scale_row(a.inter)),
                              pair_by_pair(pairs, a.dim) ? 0 : whole(a.parts * pairs * a.dim * 4), whole((2 + 2 * a.experts + pairs) * 4)};
  long long bytes = 0;
  for (long long n : parts) bytes += n;
  StreamWorkspace* ws = nullptr;
  hipError_t e = stream_workspace(s, &ws);
  if (e != hipSuccess) return e;
  std::unique_lock<std::mutex> hold(ws->call);
  void* buf = nullptr;
  e = stream_buffer(ws, s, static_cast<size_t>(bytes), 0, &buf);
  if (e != hipSuccess) return e;
  uint8_t* at = static_cast<uint8_t*>(buf);
  a.logits = reinterpret_cast<double*>(at);
  a.xq = at += parts[0];
  a.xs = at += parts[1];
  a.hq = at += parts[2];
  a.hs = at += parts[3];
  a.o = reinterpret_cast<float*>(at += parts[4]);
  a.plan = reinterpret_cast<int*>(at + parts[5]);
  for (long long t0 = 0; t0 < m.tokens; t0 += pass) {
    a.tokens = static_cast<int>(std::min(pass, m.tokens - t0));
    a.x = static_cast<const uint8_t*>(m.x) + t0 * m.x_stride * size;
    a.residual = m.residual != nullptr ? static_cast<const uint8_t*>(m.residual) + t0 * m.residual_stride * size : nullptr;
    a.y = static_cast<uint8_t*>(m.y) + t0 * m.y_stride * size;
    a.ids = m.ids + t0 * a.top;
    a.shares = m.weights + t0 * a.top;
    switch (m.type) {
      case QC_STORAGE_F32: e = run_pass<QC_STORAGE_F32>(a, s); break;
      case QC_STORAGE_F16: e = run_pass<QC_STORAGE_F16>(a, s); break;
      default: e = run_pass<QC_STORAGE_BF16>(a, s);
    }
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace qc
