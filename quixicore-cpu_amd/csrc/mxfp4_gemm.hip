// Products of two MXFP4 matrices on gfx950's block-scaled 4-bit MFMA:
// y[m][n] = sum_b 2^(ew[n][b] + ex[m][b]) sum_{i in b} w[n][b][i] x[m][b][i].
//
// v_mfma_scale_f32_{16x16x128,32x32x64}_f8f6f4 takes, per lane, 32 codes (16 bytes,
// one block of one row) and that block's scale byte, so the stored bytes are the
// operands: nothing is decoded.  Products are exact, sums f32.  Which blocks of a row
// meet in one instruction is free as long as both operands agree.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "qc_internal.h"
#include "qc_lds_dma.h"
#include "qc_storage.h"

namespace qc {
namespace {

using namespace storage;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i32x8 fp4_operand(const i32x4& v) {
  i32x8 o;
  o[0] = v[0];
  o[1] = v[1];
  o[2] = v[2];
  o[3] = v[3];
  return o;
}

// A workgroup owns TN rows of w and TM rows of x, cut into WGN x WGM wave tiles of 32 x
// 32 instructions; KG waves share a wave tile, each with 4 / KG of every step's quarters,
// and add their sums at the end.  A K step is one 128-byte line of codes (8 blocks) of every
// row and its 8 scale bytes, copied to a stage of an S-deep LDS ring by global_load_lds: codes
// 8 rows an instruction, 16-byte chunk c of row r at position c ^ ((r >> 1) & 7); scales
// 32 rows an instruction, lane l the bytes 4 (l >> 5) .. + 3 of row l & 31.  Quarter q of a
// step multiplies, with v_mfma_scale_f32_32x32x64, chunks q and 4 + q of the rows: lane l
// holds chunk 4 (l >> 5) + q of row l & 31, whose scale is byte q of the dword that it
// holds for the whole step.
//
// What bounds it: with few rows of x the stream of w (M = 1, 14336 x 4096: 31 MB, 7.1 us, of
// which a launch and the first bytes are about 3; a form without LDS, 16 rows a workgroup and
// the codes straight to registers, took 9.2, M = 32 17 against 8); with many, a step's chain
// of barrier, LDS reads and MFMAs, the LDS traffic (a 256 x 256 tile reads its 64 KB stage
// three times and writes it once, as many cycles as its MFMAs) and MFMA power: M = 4096,
// 14336 x 4096, quantised normal values, 155 us = 3.1 PFLOP/s, the matrix cores busy half of
// it (this instruction on operands that stay in registers reaches 6.5 PFLOP/s: 74 us). Eight
// waves of 64 x 128 there: four of 128 x 128 are 6% slower, sixteen of 64 x 64 3%; 128 x 128
// tiles (M = 512) take 14 us with eight waves, 24 with four.
__device__ __forceinline__ void ring_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroup b's tile: each XCD (b % 8) takes a contiguous range of an order of bands
// of kBand tiles of x, so that it reads few panels of either operand.
constexpr int kXcds = 8, kBand = 4;
__device__ __forceinline__ void tile_at(int b, int total, int tiles_n, int tiles_m, int& tn, int& tm) {
  const int q = total / kXcds, r = total % kXcds;
  const int xcd = b % kXcds, idx = b / kXcds;
  const int t = xcd * q + min(xcd, r) + idx;
  const int band = t / (tiles_n * kBand);
  const int rem = t - band * tiles_n * kBand;
  const int gm = min(tiles_m - band * kBand, kBand);
  tn = rem / gm;
  tm = band * kBand + rem % gm;
}

// PACKED: scale rows of any number of bytes, so that a row begins at any byte of a dword. A step
// then loads the three dwords that its 8 bytes lie in, the third by 64 rows an instruction, and the
// two that hold a lane's four bytes are shifted together.  (The array itself begins at a
// dword; the one that holds its last bytes is read whole.)  Against rows laid out by a launch before:
// M = 1, 14336 x 4064 11.4 -> 8.5 us, M = 77, 5461 x 2752 9.9 -> 8.4.
template <int TN, int TM, int S, int WGN, int WGM, int KG, int TYPE, bool PACKED>
__global__ __launch_bounds__(64 * WGN * WGM * KG, 1) void mxfp4_ring(
    const uint8_t* __restrict__ w, const uint8_t* __restrict__ ws, const uint8_t* __restrict__ x,
    const uint8_t* __restrict__ xs, void* __restrict__ y, int m, int n, int blocks,
    int scale_stride, int tiles_n, int tiles_m) {
  constexpr int NW = WGN * WGM * KG;
  constexpr int QN = 4 / KG;                        // quarters of a step that a wave multiplies
  constexpr int FN = TN / WGN / 32, FM = TM / WGM / 32;
  constexpr int R = TN + TM;                        // rows of a stage, w's first
  // loads a wave and step (beyond the stage's share the last one again: the same bytes)
  constexpr int GC = (R / 8 + NW - 1) / NW, GS = (R / 32 + NW - 1) / NW;
  constexpr int X = PACKED ? (R + 63) / 64 : 0;     // loads of third dwords
  constexpr int GX = (X + NW - 1) / NW;
  constexpr int G = GC + GS + GX;
  constexpr int kStage = R * 136 + X * 256;         // codes, scales, third dwords
  static_assert(FN >= 1 && FM >= 1 && S >= 2 && G * (S - 1) < 64, "tile");
  static_assert(S * kStage <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S * kStage];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tn, tm;
  tile_at(blockIdx.x, tiles_n * tiles_m, tiles_n, tiles_m, tn, tm);
  const int n0 = tn * TN, m0 = tm * TM;
  const int bytes = blocks * 16;                    // of a row's codes
  const int nk = (blocks + 7) / 8;                  // steps

  // Load j < GC of a wave: rows 8 (wave GC + j) + lane / 8 of the stage, lane writing
  // position lane % 8.  Rows past the matrix repeat its last one.
  const uint8_t* cbase[GC];
  uint32_t cvo[GC];
  int ccol[GC];
#pragma unroll
  for (int j = 0; j < GC; ++j) {
    const int r8 = 8 * min(wave * GC + j, R / 8 - 1);   // uniform
    const bool is_w = r8 < TN;
    const int first = is_w ? n0 : m0, limit = is_w ? n : m, base = is_w ? r8 : r8 - TN;
    cbase[j] = (is_w ? w : x) + static_cast<long long>(first) * bytes;
    const int r = min(first + base + (lane >> 3), limit - 1) - first;
    ccol[j] = ((lane & 7) ^ (((r8 >> 1) + (lane >> 4)) & 7)) * 16;
    cvo[j] = static_cast<uint32_t>(r) * bytes;
  }
  const uint8_t* sbase[GS];
  uint32_t svo[GS], slast[GS];                      // slast: the array's last dword
#pragma unroll
  for (int j = 0; j < GS; ++j) {
    const int r32 = 32 * min(wave * GS + j, R / 32 - 1);
    const bool is_w = r32 < TN;
    const int first = is_w ? n0 : m0, limit = is_w ? n : m, base = is_w ? r32 : r32 - TN;
    const long long at = static_cast<long long>(first) * scale_stride;
    const int r = min(first + base + (lane & 31), limit - 1) - first;
    sbase[j] = (is_w ? ws : xs) + (PACKED ? at & ~3ll : at);
    svo[j] = static_cast<uint32_t>(r) * scale_stride;
    slast[j] = 0;
    if constexpr (PACKED) {
      svo[j] = (static_cast<uint32_t>(at & 3) + svo[j]) & ~3u;
      const long long last = ((static_cast<long long>(limit) * scale_stride - 1) & ~3ll) - (at & ~3ll);
      slast[j] = static_cast<uint32_t>(last < 0x7FFFFFFF ? last : 0x7FFFFFFF);
    }
  }
  const uint8_t* xat[GX ? GX : 1];                  // third dword of the lane's row at step 0
  const uint8_t* xlast[GX ? GX : 1];
#pragma unroll
  for (int j = 0; j < GX; ++j) {
    const int rr = min(64 * min(wave * GX + j, X - 1) + lane, R - 1);
    const bool is_w = rr < TN;
    const int limit = is_w ? n : m;
    const long long row = min((is_w ? n0 + rr : m0 + rr - TN), limit - 1);
    const uint8_t* array = is_w ? ws : xs;
    xat[j] = array + ((row * scale_stride) & ~3ll) + 8;
    xlast[j] = array + ((static_cast<long long>(limit) * scale_stride - 1) & ~3ll);
  }
  auto issue = [&](int step, int stage, int from, int to) {
    uint8_t* base = lds + stage * kStage;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      if (j < from || j >= to) continue;
      if (j < GC) {
        const int col = min(128 * step + ccol[j < GC ? j : 0], bytes - 16);
        dma16(cbase[j < GC ? j : 0], cvo[j < GC ? j : 0] + col, base + min(wave * GC + j, R / 8 - 1) * 1024);
      } else if (j < GC + GS) {
        const int i = j - GC < GS ? j - GC : 0;
        const int col = 8 * step + 4 * (lane >> 5);
        dma4(sbase[i], PACKED ? min(svo[i] + col, slast[i]) : svo[i] + min(col, scale_stride - 4),
             base + R * 128 + min(wave * GS + i, R / 32 - 1) * 256);
      } else {
        const int i = j - GC - GS;
        const uint8_t* at = xat[i] + 8 * step;
        dma4_addr(at < xlast[i] ? at : xlast[i], base + R * 136 + min(wave * GX + i, X - 1) * 256);
      }
    }
  };

  const int kg = wave / (WGN * WGM), tile = wave % (WGN * WGM);
  const int wn = (tile / WGM) * FN * 32, wm = (tile % WGM) * FM * 32;
  const int q0 = kg * QN;
  const int key = (lane >> 1) & 7;
  i32x4 fa[2][FN], fb[2][FM];
  int sa[2][FN], sb[2][FM];                         // scales of this step and the next
  auto read_frags = [&](int stage, int j, int slot) {     // quarter q0 + j
    const uint8_t* base = lds + stage * kStage + (lane & 31) * 128 + (((4 * (lane >> 5) + q0 + j) ^ key) * 16);
#pragma unroll
    for (int i = 0; i < FN; ++i) fa[slot][i] = *reinterpret_cast<const i32x4*>(base + (wn + 32 * i) * 128);
#pragma unroll
    for (int j = 0; j < FM; ++j) fb[slot][j] = *reinterpret_cast<const i32x4*>(base + (TN + wm + 32 * j) * 128);
  };
  uint32_t ba[FN], bb[FM];                          // PACKED: the byte of a dword that a row begins at
  if constexpr (PACKED) {
#pragma unroll
    for (int i = 0; i < FN; ++i) ba[i] = (static_cast<uint32_t>(min(n0 + wn + 32 * i + (lane & 31), n - 1)) * scale_stride) & 3;
#pragma unroll
    for (int j = 0; j < FM; ++j) bb[j] = (static_cast<uint32_t>(min(m0 + wm + 32 * j + (lane & 31), m - 1)) * scale_stride) & 3;
  }
  // the dword after a lane's: its row's second or third
  const int after = (lane < 32 ? R * 128 + 128 : R * 136) + 4 * (lane & 31), after_by = lane < 32 ? 256 : 128;
  auto read_scales = [&](int stage, int slot) {
    const uint8_t* base = lds + stage * kStage;
    auto read = [&](int rows32, uint32_t byte) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(base + R * 128 + 4 * lane + rows32 * 256);
      if constexpr (!PACKED) return static_cast<int>(v) >> (8 * q0);
      const uint32_t next = *reinterpret_cast<const uint32_t*>(base + after + rows32 * after_by);
      return static_cast<int>(__builtin_amdgcn_alignbyte(next, v, byte)) >> (8 * q0);
    };
#pragma unroll
    for (int i = 0; i < FN; ++i) sa[slot][i] = read(wn / 32 + i, PACKED ? ba[i] : 0);
#pragma unroll
    for (int j = 0; j < FM; ++j) sb[slot][j] = read((TN + wm) / 32 + j, PACKED ? bb[j] : 0);
  };
  f32x16 acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  auto mfmas = [&](auto quarter, int slot, int ss) {
    constexpr int Q = decltype(quarter)::value;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
            fp4_operand(fa[slot][i]), fp4_operand(fb[slot][j]), acc[i][j], 4, 4, Q, sa[ss][i], Q,
            sb[ss][j]);
  };

#pragma unroll
  for (int st = 0; st < S; ++st) issue(min(st, nk - 1), st, 0, G);
  wait_vmcnt<(S - 1) * G>();
  ring_barrier();
  read_scales(0, 0);
  read_frags(0, 0, 0);
  int stage = 0;
  // slots: quarter j of a step in j & 1, the next step's first in the one not in use
  auto step = [&](int k, auto par) {
    constexpr int P = decltype(par)::value;
    constexpr int FIRST = QN == 1 ? P : 0, LAST = QN == 1 ? P : 1;
    if constexpr (QN == 4) {
      read_frags(stage, 1, 1);
      mfmas(std::integral_constant<int, 0>(), 0, P);
      read_frags(stage, 2, 0);
      mfmas(std::integral_constant<int, 1>(), 1, P);
      read_frags(stage, 3, 1);
      mfmas(std::integral_constant<int, 2>(), 0, P);
    } else if constexpr (QN == 2) {
      read_frags(stage, 1, 1);
      mfmas(std::integral_constant<int, 0>(), 0, P);
    }
    // step k + 1 is in; every wave has read all of stage
    wait_vmcnt<(S - 2) * G>();
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt(0)
    ring_barrier();
    issue(min(k + S, nk - 1), stage, 0, G);
    stage = stage + 1 < S ? stage + 1 : 0;
    read_scales(stage, P ^ 1);
    read_frags(stage, 0, FIRST ^ (QN == 1 ? 1 : 0));
    mfmas(std::integral_constant<int, QN - 1>(), LAST, P);
  };
  int k = 0;
  for (; k + 2 < nk; k += 2) {
    step(k, std::integral_constant<int, 0>());
    step(k + 1, std::integral_constant<int, 1>());
  }
  int ss = 0;
  if (k + 1 < nk) {
    step(k, std::integral_constant<int, 0>());
    ss = 1;
  }
  {
    // the last step: blocks past the row's end count as zeros
    const int left = blocks - 8 * (nk - 1);
    int za[FN], zb[FM];
#pragma unroll
    for (int i = 0; i < FN; ++i) za[i] = ss ? sa[1][i] : sa[0][i];
#pragma unroll
    for (int j = 0; j < FM; ++j) zb[j] = ss ? sb[1][j] : sb[0][j];
    auto last = [&](auto quarter) {
      constexpr int Q = decltype(quarter)::value;
      read_frags(stage, Q, 0);
      const bool in = 4 * (lane >> 5) + q0 + Q < left;
      const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < FN; ++i) {
        fa[0][i] = in ? fa[0][i] : zero;
        sa[0][i] = in ? za[i] : 0;
      }
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        fb[0][j] = in ? fb[0][j] : zero;
        sb[0][j] = in ? zb[j] : 0;
      }
      mfmas(quarter, 0, 0);
    };
    if (left > q0) last(std::integral_constant<int, 0>());
    if constexpr (QN > 1)
      if (left > q0 + 1) last(std::integral_constant<int, 1>());
    if constexpr (QN > 2) {
      if (left > 2) last(std::integral_constant<int, 2>());
      if (left > 3) last(std::integral_constant<int, 3>());
    }
  }
  wait_vmcnt<0>();   // no load may land in LDS that is no longer this workgroup's
  if constexpr (KG > 1) {
    // the quarters' sums meet in the ring's LDS, added in their order
    static_assert((KG - 1) * WGN * WGM * FN * FM * 4096 <= S * kStage, "sums fit the ring");
    f32x16* sums = reinterpret_cast<f32x16*>(lds);
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));
    __syncthreads();
    if (kg > 0) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
          sums[((((kg - 1) * WGN * WGM + tile) * FN + i) * FM + j) * 64 + lane] = acc[i][j];
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int g = 0; g < KG - 1; ++g)
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] += sums[(((g * WGN * WGM + tile) * FN + i) * FM + j) * 64 + lane];
  }

  // Lane l has row wm + 32 j + (l & 31) of x and, in register e, row 8 (e >> 2) + 4 (l >> 5) + (e & 3) of
  // w: 8 bytes of y here and there.  32 rows at a time go through the ring's LDS and out
  // in whole lines, 16 bytes a lane where rows of y allow it, else an element a lane: M = 4096, 14336 x
  // 4096, bf16 184 -> 161 us, M = 3099, 16231 x 832 186 -> 81.
  typedef typename Storage<TYPE>::raw raw;
  constexpr int kCols = FN * 32, kPer16 = Storage<TYPE>::per16, kRow = kCols * sizeof(raw) + 16;
  static_assert(KG == 1 || WGN * WGM == 1, "the sums of other waves are in the way");
  static_assert(WGN * WGM * 32 * kRow <= S * kStage, "rows fit the ring");
  if constexpr (KG == 1) __syncthreads();          // every wave has read the last stage
  uint8_t* rows = lds + tile * 32 * kRow;
  const bool vec = n % kPer16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0;
  raw* out = static_cast<raw*>(y);
  auto in_order = [] {                              // of the wave's own LDS accesses
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
#pragma unroll
  for (int j = 0; j < FM; ++j) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        uint8_t* at = rows + (lane & 31) * kRow + (32 * i + 2 * e + 4 * (lane >> 5)) * sizeof(raw);
        if constexpr (TYPE == QC_STORAGE_F32)
          *reinterpret_cast<f32x4*>(at) = f32x4{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]};
        else
          *reinterpret_cast<u32x2*>(at) = u32x2{encode2<TYPE>(acc[i][j][e], acc[i][j][e + 1]),
                                                encode2<TYPE>(acc[i][j][e + 2], acc[i][j][e + 3])};
      }
    in_order();
    const int mj = m0 + wm + 32 * j, nj = n0 + wn;
    if (vec) {
      constexpr int kChunks = kCols / kPer16;
#pragma unroll
      for (int c = 0; c < kChunks / 2; ++c) {
        const int id = 64 * c + lane, r = id / kChunks, col = id % kChunks * kPer16;
        if (mj + r < m && nj + col < n)
          *reinterpret_cast<u32x4*>(out + static_cast<long long>(mj + r) * n + nj + col) =
              *reinterpret_cast<const u32x4*>(rows + r * kRow + col * sizeof(raw));
      }
    } else {
#pragma unroll 8
      for (int c = 0; c < kCols / 2; ++c) {
        const int id = 64 * c + lane, r = id / kCols, col = id % kCols;
        if (mj + r < m && nj + col < n)
          out[static_cast<long long>(mj + r) * n + nj + col] = *reinterpret_cast<const raw*>(rows + r * kRow + col * sizeof(raw));
      }
    }
    in_order();
  }
}

// Scale rows laid out for the ring, whose loads are dwords (arrays that begin at any byte, and rows of any
// length for the largest tile).  Bytes past a row's blocks are zero.
__global__ __launch_bounds__(256) void pad_scales(const uint8_t* __restrict__ ws, long long n,
                                                  const uint8_t* __restrict__ xs, long long m,
                                                  int blocks, int stride, uint32_t* __restrict__ out) {
  const int words = stride / 4;
  const long long total = (n + m) * words;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<long long>(gridDim.x) * 256) {
    const long long r = i / words;
    const int b = 4 * static_cast<int>(i - r * words);
    const uint8_t* src = r < n ? ws + r * blocks : xs + (r - n) * blocks;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (b + e < blocks) v |= static_cast<uint32_t>(src[b + e]) << (8 * e);
    out[i] = v;
  }
}

struct Operands {
  const uint8_t *w, *ws, *x, *xs;
  void* y;
  int m, n, blocks;
};

// The tiles, and what a product of K costs with each: fixed + K / 4096 (first + more (rounds - 1)) us,
// rounds being the tiles over the CUs, of which `whole` counts started rounds whole. Fitted
// to 730 sizes of M 1 to 4096, N 256 to 16384, K 256 to 14336, over which the tile chosen is 0.2%
// slower than the best (a fit to half of them, on the other half: 0.3%).  us at K = 4096:
//            32x32  64x32  64x64  128x64  128x128  256x128  256x256
// 1 x 14336    7.7    7.5    8.4     9.8     12.3     20.4     30.4
// 64 x 4096    5.4    6.7    7.8    10.4     11.7     19.7     27.8
// 128 x 14336 23.1   20.4   14.5    12.4     14.9     22.2     32.3
// 512 x 4096  23.3   22.6   14.0    12.0     14.4     21.5     32.2
// 512 x 14336 72.0   62.4   40.9    37.3     28.7     25.3     36.0
// 2048 x 14336 261    230    154     133      103       97       80
struct Tile {
  int tn, tm;
  double fixed, first, more, whole;
};
constexpr int kTiles = 7;
constexpr Tile kTile[kTiles] = {{32, 32, 3.3, 3.0, 3.9, 0.7},     {64, 32, 3.3, 4.8, 6.3, 1.0},
                                {64, 64, 3.6, 5.2, 8.7, 1.0},     {128, 64, 3.2, 11.1, 11.3, 1.0},
                                {128, 128, 4.8, 12.4, 22.1, 1.0}, {256, 128, 5.7, 25.5, 40.3, 0.7},
                                {256, 256, 20.5, 27.9, 48.1, 1.0}};

int choose_tile(long long m, long long n, long long k, int cus) {
  int best = 0;
  double least = 0.0;
  for (int i = 0; i < kTiles; ++i) {
    const Tile& t = kTile[i];
    const double tiles = static_cast<double>((n + t.tn - 1) / t.tn) * static_cast<double>((m + t.tm - 1) / t.tm);
    const double rounds = t.whole * std::ceil(tiles / cus) + (1.0 - t.whole) * tiles / cus;
    const double cost = t.fixed + static_cast<double>(k) / 4096.0 * (t.first + t.more * std::max(0.0, rounds - 1.0));
    if (i == 0 || cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}

template <int TN, int TM, int S, int WGN, int WGM, int KG, int TYPE>
hipError_t run_ring(const Operands& o, int scale_stride, hipStream_t s) {
  const int tiles_n = (o.n + TN - 1) / TN, tiles_m = (o.m + TM - 1) / TM;
  if (static_cast<long long>(tiles_n) * tiles_m > INT_MAX) return hipErrorInvalidValue;
  auto kernel = mxfp4_ring<TN, TM, S, WGN, WGM, KG, TYPE, false>;
  if constexpr (TN * TM < 256 * 256)
    if (scale_stride % 4 != 0) kernel = mxfp4_ring<TN, TM, S, WGN, WGM, KG, TYPE, true>;
  kernel<<<static_cast<unsigned>(tiles_n) * tiles_m, 64 * WGN * WGM * KG, 0, s>>>(
      o.w, o.ws, o.x, o.xs, o.y, o.m, o.n, o.blocks, scale_stride, tiles_n, tiles_m);
  return hipGetLastError();
}

template <int TYPE>
hipError_t run_gemm(Operands o, int route, hipStream_t s) {
  StreamWorkspace* ws = nullptr;
  std::unique_lock<std::mutex> hold;
  // a tile's codes are addressed with 32 bits: 32 rows of long ones
  const int tile = o.blocks > (1 << 19) ? 0 : route > 0 ? route - 1 : choose_tile(o.m, o.n, 32LL * o.blocks, device_cu_count());
  int stride = o.blocks;
  // Rows of scales that do not begin at dwords: laid out first for the largest tile, whose LDS
  // has no time for the third dwords (us, laid out / in the ring, K = 4064, N = 14336: M = 1 11.4 /
  // 8.5, 512 35.2 / 34.6, 2048 97.4 / 100.9, 4096 209.7 / 214.6).
  if ((o.blocks % 4 != 0 && tile == kTiles - 1) || ((reinterpret_cast<uintptr_t>(o.ws) | reinterpret_cast<uintptr_t>(o.xs)) & 3) != 0) {
    hipError_t e = stream_workspace(s, &ws);
    if (e != hipSuccess) return e;
    hold = std::unique_lock<std::mutex>(ws->call);
    stride = (o.blocks + 3) / 4 * 4;
    void* buf = nullptr;
    const long long rows = static_cast<long long>(o.n) + o.m;
    e = stream_buffer(ws, s, static_cast<size_t>(rows) * stride, 0, &buf);
    if (e != hipSuccess) return e;
    const long long words = rows * (stride / 4);
    const int grid = static_cast<int>(std::min<long long>((words + 255) / 256, 4096));
    pad_scales<<<grid, 256, 0, s>>>(o.ws, o.n, o.xs, o.m, o.blocks, stride, static_cast<uint32_t*>(buf));
    if ((e = hipGetLastError()) != hipSuccess) return e;
    o.ws = static_cast<const uint8_t*>(buf);
    o.xs = o.ws + static_cast<long long>(o.n) * stride;
  }
  switch (tile) {
    case 0: return run_ring<32, 32, 4, 1, 1, 2, TYPE>(o, stride, s);
    case 1: return run_ring<64, 32, 4, 2, 1, 1, TYPE>(o, stride, s);
    case 2: return run_ring<64, 64, 4, 2, 2, 1, TYPE>(o, stride, s);
    case 3: return run_ring<128, 64, 3, 4, 2, 1, TYPE>(o, stride, s);
    case 4: return run_ring<128, 128, 4, 4, 2, 1, TYPE>(o, stride, s);
    case 5: return run_ring<256, 128, 3, 4, 2, 1, TYPE>(o, stride, s);
    default: return run_ring<256, 256, 2, 4, 2, 1, TYPE>(o, stride, s);
  }
}

}  // namespace

hipError_t launch_mxfp4_gemm(const uint8_t* w, const uint8_t* ws, const uint8_t* x,
                             const uint8_t* xs, void* y, int type, long long m, long long n,
                             long long k, int route, hipStream_t s) {
  const Operands o = {w, ws, x, xs, y, static_cast<int>(m), static_cast<int>(n), static_cast<int>(k / 32)};
  switch (type) {
    case QC_STORAGE_F32: return run_gemm<QC_STORAGE_F32>(o, route, s);
    case QC_STORAGE_F16: return run_gemm<QC_STORAGE_F16>(o, route, s);
    default: return run_gemm<QC_STORAGE_BF16>(o, route, s);
  }
}

}  // namespace qc
