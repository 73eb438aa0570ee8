// A mixture-of-experts feed-forward with MXFP4 weights for a few tokens on gfx950:
// l = x R^T + b, the k experts of the largest l (ties to the lowest index), their shares p
// (softmax of l over the chosen, or over all), and
//   y = residual + sum_s p_s D_e (act(G_e x) * (U_e x)),  e = e_s.
//
// Logits are sums in 64 bits, so that which experts are chosen does not hang on the order of a sum.
// Weights are decoded in registers to bf16 (a code times its block's power of two is exact there) for
// v_mfma_f32_16x16x32_bf16; activations enter as sums of bf16 terms: x as 1 (bf16), 2 (f16, exact) or 3 (f32, 24
// bits), the hidden values as 2 (16 bits; 16-bit x and y) or 3 (f32). Sums are f32.
#include <algorithm>

#include "qc_internal.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kPass = 512;          // tokens of a pass
constexpr int kMaxExperts = 1024;   // (and 64 of a token)

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
  double* logits;      // [tokens][experts]
  int* ids;            // [tokens][top]
  float* shares;
  uint16_t* xt;        // [terms][tokens][dim] bf16
  uint16_t* h;         // [terms][tokens * top][inter] bf16
  float* o;            // [tokens * top][dim]
  int vec;             // x rows and the router allow 16-byte loads
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

// A wavefront: one expert's logits of kLogitTokens tokens.
constexpr int kLogitTokens = 4;
template <int TYPE, int RTYPE>
__global__ __launch_bounds__(kThreads) void moe_logits(MoeArgs a) {
  constexpr int V = Storage<TYPE>::per16 < Storage<RTYPE>::per16 ? Storage<RTYPE>::per16 : Storage<TYPE>::per16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int groups = (a.experts + 3) / 4;
  const int e = (blockIdx.x % groups) * 4 + wave, t0 = blockIdx.x / groups * kLogitTokens;
  if (e >= a.experts) return;
  double acc[kLogitTokens] = {};
  for (int d = lane * V; d < a.dim; d += 64 * V) {
    float r[V], x[V];
#pragma unroll
    for (int j = 0; j < V; j += Storage<RTYPE>::per16)
      load_n<RTYPE>(a.router, static_cast<long long>(e) * a.dim + d + j, a.vec, r + j);
#pragma unroll
    for (int t = 0; t < kLogitTokens; ++t) {
#pragma unroll
      for (int j = 0; j < V; j += Storage<TYPE>::per16)
        load_n<TYPE>(a.x, min(t0 + t, a.tokens - 1) * a.x_stride + d + j, a.vec, x + j);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[t] = fma(static_cast<double>(x[j]), static_cast<double>(r[j]), acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < kLogitTokens; ++t) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) acc[t] += __shfl_xor(acc[t], o);
    if (lane == 0 && t0 + t < a.tokens)
      a.logits[static_cast<long long>(t0 + t) * a.experts + e] = acc[t] + (a.bias != nullptr ? a.bias[e] : 0.f);
  }
}

// x as a sum of N bf16 terms.
template <int N>
__device__ __forceinline__ void bf16_terms(float v, uint16_t* t) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const __bf16 b = static_cast<__bf16>(v);
    t[i] = __builtin_bit_cast(uint16_t, b);
    v -= static_cast<float>(b);
  }
}

// A wavefront a token: its experts and their shares, and its row in bf16 terms.  A logit that is NaN counts as
// the lowest.
template <int TYPE, int NX>
__global__ __launch_bounds__(kThreads) void moe_select(MoeArgs a) {
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.tokens) return;
  const double* l = a.logits + static_cast<long long>(t) * a.experts;
  auto at = [&](int e) {
    const double v = l[e];
    return v == v ? v : -INFINITY;
  };
  uint32_t taken = 0;              // of the lane's experts lane, lane + 64, ...
  double mine = 0.0, first = 0.0;  // lane s: the logit of slot s; the largest
  int id = 0;
  for (int s = 0; s < a.top; ++s) {
    double best = -INFINITY;
    int where = INT32_MAX;
    for (int e = lane, i = 0; e < a.experts; e += 64, ++i)
      if (!(taken >> i & 1) && (where == INT32_MAX || at(e) > best)) {
        best = at(e);
        where = e;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const double v = __shfl_xor(best, o);
      const int w = __shfl_xor(where, o);
      if (w != INT32_MAX && (where == INT32_MAX || v > best || (v == best && w < where))) {
        best = v;
        where = w;
      }
    }
    if ((where & 63) == lane) taken |= 1u << (where >> 6);
    if (s == 0) first = best;
    if (lane == s) {
      mine = best;
      id = where;
    }
  }
  double sum = 0.0;
  const double weight = lane < a.top ? exp(mine - first) : 0.0;
  if (a.normalize) {
    sum = weight;
  } else {
    for (int e = lane; e < a.experts; e += 64) sum += exp(at(e) - first);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  if (lane < a.top) {
    a.ids[t * a.top + lane] = id;
    a.shares[t * a.top + lane] = static_cast<float>(weight / sum * a.scale);
  }
  constexpr int V = Storage<TYPE>::per16;
  for (int d = lane * V; d < a.dim; d += 64 * V) {
    float v[V];
    load_n<TYPE>(a.x, t * a.x_stride + d, a.vec, v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      uint16_t w[NX];
      bf16_terms<NX>(v[j], w);
#pragma unroll
      for (int i = 0; i < NX; ++i) a.xt[(static_cast<long long>(i) * a.tokens + t) * a.dim + d + j] = w[i];
    }
  }
}

// What a workgroup of a grid over the experts that are hit works on.
struct Chosen {
  int expert, count;
};
// The u-th expert that any token chose, and its pairs (token * top + slot, by token) in list; all threads take
// part.  False where there are not as many.
__device__ __forceinline__ bool find_expert(const MoeArgs& a, int u, Chosen& c, uint32_t* hit, int* list, int* sums) {
  const int tid = threadIdx.x, words = (a.experts + 31) / 32, pairs = a.tokens * a.top;
  for (int i = tid; i < words; i += kThreads) hit[i] = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += kThreads) atomicOr(hit + (a.ids[i] >> 5), 1u << (a.ids[i] & 31));
  __syncthreads();
  c.expert = -1;
  for (int w = 0; w < words; ++w) {
    uint32_t v = hit[w];
    const int n = __popc(v);
    if (u < n) {
      for (; u > 0; --u) v &= v - 1;
      c.expert = 32 * w + __ffs(v) - 1;
      break;
    }
    u -= n;
  }
  if (c.expert < 0) return false;
  c.count = 0;
  for (int t0 = 0; t0 < a.tokens; t0 += kThreads) {
    const int t = t0 + tid;
    int slot = -1;
    if (t < a.tokens)
      for (int s = 0; s < a.top; ++s)
        if (a.ids[t * a.top + s] == c.expert) slot = s;
    const uint64_t in = __ballot(slot >= 0);
    if ((tid & 63) == 0) sums[tid >> 6] = __popcll(in);
    __syncthreads();
    int before = c.count;
    for (int w = 0; w < tid >> 6; ++w) before += sums[w];
    if (slot >= 0) list[before + __popcll(in & ((1ull << (tid & 63)) - 1))] = t * a.top + slot;
    for (int w = 0; w < kThreads / 64; ++w) c.count += sums[w];
    __syncthreads();
  }
  return true;
}

// Eight codes times their block's power of two.
__device__ __forceinline__ bf16x8 decode8(uint32_t c, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
  const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
  return bf16x8{a[0], a[1], b[0], b[1], d[0], d[1], e[0], e[1]};
}

// acc[i][c] += rows of w (tile i of 16) times columns of x (tile c of 16), over K steps [from, to) of four blocks of
// 32.  Lane l holds, of a step, block 4 step + (l >> 4) of row l & 15: its 16 bytes are the operands of
// four MFMAs, eight codes each; of x the same eight elements of column l & 15.
template <int RT, int CT, int NX>
__device__ __forceinline__ void product(const uint8_t* const (&codes)[RT], const uint8_t* const (&scales)[RT],
                                        const uint16_t* const (&x)[CT], long long term, int blocks, int from, int to,
                                        f32x4 (&acc)[RT][CT]) {
  const int g = (threadIdx.x & 63) >> 4;
  for (int s = from; s < to; ++s) {
    const int b = 4 * s + g;
    const bool in = b < blocks;
    const int bb = in ? b : blocks - 1;
    u32x4 w[RT];
    float f[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      w[i] = *reinterpret_cast<const u32x4*>(codes[i] + 16 * bb);
      f[i] = __uint_as_float(static_cast<uint32_t>(scales[i][bb]) << 23);
      if (!in) {
        w[i] = u32x4{0, 0, 0, 0};
        f[i] = 1.0f;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bf16x8 xf[CT][NX];
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int n = 0; n < NX; ++n) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(x[c] + n * term + 32 * bb + 8 * j);
          xf[c][n] = __builtin_bit_cast(bf16x8, in ? v : u32x4{0, 0, 0, 0});
        }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const bf16x8 wf = decode8(w[i][j], f[i]);
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
          for (int n = 0; n < NX; ++n)
            acc[i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, xf[c][n], acc[i][c], 0, 0, 0);
      }
    }
  }
}

// Sums of the KS waves that share rows, in their order, in the first one's acc.
template <int KS, int N>
__device__ __forceinline__ void join(f32x4* acc, f32x4* lds) {
  if constexpr (KS == 1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % KS, row = wave / KS;
  __syncthreads();
  if (part > 0)
    for (int i = 0; i < N; ++i) lds[((row * (KS - 1) + part - 1) * N + i) * 64 + lane] = acc[i];
  __syncthreads();
  if (part == 0)
    for (int p = 1; p < KS; ++p)
      for (int i = 0; i < N; ++i) acc[i] += lds[((row * (KS - 1) + p - 1) * N + i) * 64 + lane];
}

// Workgroup: 4 / KS tiles of 16 hidden rows of an expert, KS waves each over parts of K.
template <int CT, int NX, int NH, int KS>
__global__ __launch_bounds__(kThreads) void moe_up(MoeArgs a, int tiles) {
  __shared__ uint32_t hit[kMaxExperts / 32];
  __shared__ int list[kPass], sums[4];
  __shared__ f32x4 s_acc[KS > 1 ? 4 * 2 * CT * 64 : 1];
  Chosen c;
  if (!find_expert(a, blockIdx.x / tiles, c, hit, list, sums)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = ((blockIdx.x % tiles) * (4 / KS) + wave / KS) * 16, part = wave % KS;
  const int blocks = a.dim / 32, steps = (blocks + 3) / 4;
  const bool real = r0 < a.inter;
  const long long row = static_cast<long long>(c.expert) * 2 * a.inter + min(r0, a.inter - 16) + (lane & 15);
  const uint8_t* codes[2] = {a.gu + row * (a.dim / 2), a.gu + (row + a.inter) * (a.dim / 2)};
  const uint8_t* scales[2] = {a.gus + row * blocks, a.gus + (row + a.inter) * blocks};
  const long long pairs = static_cast<long long>(a.tokens) * a.top;
  for (int c0 = 0; c0 < c.count; c0 += 16 * CT) {
    const uint16_t* x[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
      x[i] = a.xt + static_cast<long long>(list[min(c0 + 16 * i + (lane & 15), c.count - 1)] / a.top) * a.dim;
    f32x4 acc[2][CT];
#pragma unroll
    for (int i = 0; i < CT; ++i) acc[0][i] = acc[1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    product<2, CT, NX>(codes, scales, x, static_cast<long long>(a.tokens) * a.dim, blocks, steps * part / KS,
                       steps * (part + 1) / KS, acc);
    join<KS, 2 * CT>(&acc[0][0], s_acc);
    if (part > 0 || !real) continue;
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int at = c0 + 16 * i + (lane & 15);
      if (at >= c.count) continue;
      uint16_t w[4][NH];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v = acc[0][i][e], u = acc[1][i][e];
        float f;
        if (a.gelu) f = 0.5f * v * (1.0f + tanhf(0.7978845608028654f * (v + 0.044715f * v * v * v)));
        else f = v / (1.0f + expf(-v));
        bf16_terms<NH>(f * u, w[e]);
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
        *reinterpret_cast<u32x2*>(a.h + (n * pairs + list[at]) * a.inter + r0 + 4 * (lane >> 4)) =
            u32x2{static_cast<uint32_t>(w[0][n]) | static_cast<uint32_t>(w[1][n]) << 16,
                  static_cast<uint32_t>(w[2][n]) | static_cast<uint32_t>(w[3][n]) << 16};
    }
  }
}

// The same of the second product: o = share times the sums, a row a pair.
template <int CT, int NH, int KS>
__global__ __launch_bounds__(kThreads) void moe_down(MoeArgs a, int tiles) {
  __shared__ uint32_t hit[kMaxExperts / 32];
  __shared__ int list[kPass], sums[4];
  __shared__ f32x4 s_acc[KS > 1 ? 4 * 2 * CT * 64 : 1];
  Chosen c;
  if (!find_expert(a, blockIdx.x / tiles, c, hit, list, sums)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r0 = ((blockIdx.x % tiles) * (4 / KS) + wave / KS) * 32, part = wave % KS;
  const int blocks = a.inter / 32, steps = (blocks + 3) / 4;
  const bool real = r0 < a.dim;
  const long long row = static_cast<long long>(c.expert) * a.dim + min(r0, a.dim - 32) + (lane & 15);
  const uint8_t* codes[2] = {a.dn + row * (a.inter / 2), a.dn + (row + 16) * (a.inter / 2)};
  const uint8_t* scales[2] = {a.dns + row * blocks, a.dns + (row + 16) * blocks};
  const long long pairs = static_cast<long long>(a.tokens) * a.top;
  for (int c0 = 0; c0 < c.count; c0 += 16 * CT) {
    const uint16_t* x[CT];
#pragma unroll
    for (int i = 0; i < CT; ++i)
      x[i] = a.h + static_cast<long long>(list[min(c0 + 16 * i + (lane & 15), c.count - 1)]) * a.inter;
    f32x4 acc[2][CT];
#pragma unroll
    for (int i = 0; i < CT; ++i) acc[0][i] = acc[1][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    product<2, CT, NH>(codes, scales, x, pairs * a.inter, blocks, steps * part / KS, steps * (part + 1) / KS, acc);
    join<KS, 2 * CT>(&acc[0][0], s_acc);
    if (part > 0 || !real) continue;
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int at = c0 + 16 * i + (lane & 15);
      if (at >= c.count) continue;
      const float p = a.shares[list[at]];
#pragma unroll
      for (int n = 0; n < 2; ++n)
        *reinterpret_cast<f32x4*>(a.o + static_cast<long long>(list[at]) * a.dim + r0 + 16 * n + 4 * (lane >> 4)) =
            acc[n][i] * p;
    }
  }
}

// y = residual + the pairs' sums in the order of their slots.
template <int TYPE>
__global__ __launch_bounds__(kThreads) void moe_join(MoeArgs a) {
  typedef typename Storage<TYPE>::raw raw;
  const long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x;
  const int quads = a.dim / 4, t = static_cast<int>(i / quads), d = static_cast<int>(i - static_cast<long long>(t) * quads) * 4;
  if (t >= a.tokens) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.top; ++s)
    v += *reinterpret_cast<const f32x4*>(a.o + (static_cast<long long>(t) * a.top + s) * a.dim + d);
  const raw* r = static_cast<const raw*>(a.residual) + t * a.residual_stride + d;
  raw* y = static_cast<raw*>(a.y) + t * a.y_stride + d;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = encode<TYPE>(a.residual != nullptr ? decode<TYPE>(r[e]) + v[e] : v[e]);
}

template <int TYPE, int CT, int NX, int NH>
hipError_t run_products(const MoeArgs& a, int hits, hipStream_t s) {
  constexpr int KS = 4;
  const int up = (a.inter + 64 / KS - 1) / (64 / KS), down = (a.dim + 128 / KS - 1) / (128 / KS);
  moe_up<CT, NX, NH, KS><<<static_cast<unsigned>(hits) * up, kThreads, 0, s>>>(a, up);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  moe_down<CT, NH, KS><<<static_cast<unsigned>(hits) * down, kThreads, 0, s>>>(a, down);
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_pass(const MoeArgs& a, hipStream_t s) {
  constexpr int NX = TYPE == QC_STORAGE_F32 ? 3 : TYPE == QC_STORAGE_F16 ? 2 : 1;
  constexpr int NH = TYPE == QC_STORAGE_F32 ? 3 : 2;
  const unsigned grid = static_cast<unsigned>((a.experts + 3) / 4) * ((a.tokens + kLogitTokens - 1) / kLogitTokens);
  switch (a.router_type) {
    case QC_STORAGE_F32: moe_logits<TYPE, QC_STORAGE_F32><<<grid, kThreads, 0, s>>>(a); break;
    case QC_STORAGE_F16: moe_logits<TYPE, QC_STORAGE_F16><<<grid, kThreads, 0, s>>>(a); break;
    default: moe_logits<TYPE, QC_STORAGE_BF16><<<grid, kThreads, 0, s>>>(a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  moe_select<TYPE, NX><<<(a.tokens + 3) / 4, kThreads, 0, s>>>(a);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  const int pairs = a.tokens * a.top, hits = std::min(a.experts, pairs);
  if (a.tokens <= 16 || pairs <= 12 * a.experts) e = run_products<TYPE, 1, NX, NH>(a, hits, s);
  else if (pairs <= 24 * a.experts) e = run_products<TYPE, 2, NX, NH>(a, hits, s);
  else e = run_products<TYPE, 4, NX, NH>(a, hits, s);
  if (e != hipSuccess) return e;
  const long long quads = static_cast<long long>(a.tokens) * (a.dim / 4);
  moe_join<TYPE><<<static_cast<unsigned>((quads + kThreads - 1) / kThreads), kThreads, 0, s>>>(a);
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
  const int nx = m.type == QC_STORAGE_F32 ? 3 : m.type == QC_STORAGE_F16 ? 2 : 1, nh = m.type == QC_STORAGE_F32 ? 3 : 2;
  const long long t = std::min<long long>(m.tokens, kPass), pairs = t * a.top;
  const auto whole = [](long long n) { return (n + 255) / 256 * 256; };
  const long long parts[4] = {whole(t * a.experts * 8), whole(nx * t * a.dim * 2), whole(nh * pairs * a.inter * 2),
                              whole(pairs * a.dim * 4)};
  StreamWorkspace* ws = nullptr;
  hipError_t e = stream_workspace(s, &ws);
  if (e != hipSuccess) return e;
  std::unique_lock<std::mutex> hold(ws->call);
  void* buf = nullptr;
  e = stream_buffer(ws, s, static_cast<size_t>(parts[0] + parts[1] + parts[2] + parts[3]), 0, &buf);
  if (e != hipSuccess) return e;
  uint8_t* at = static_cast<uint8_t*>(buf);
  a.logits = reinterpret_cast<double*>(at);
  a.xt = reinterpret_cast<uint16_t*>(at += parts[0]);
  a.h = reinterpret_cast<uint16_t*>(at += parts[1]);
  a.o = reinterpret_cast<float*>(at + parts[2]);
  for (long long t0 = 0; t0 < m.tokens; t0 += kPass) {
    a.tokens = static_cast<int>(std::min<long long>(kPass, m.tokens - t0));
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
