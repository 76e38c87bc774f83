// Matrix products of bfloat16 operands on the matrix cores of MI355X (gfx950), as tiles for kernels with epilogues of
// their own (ews_loss.hip).
//
//   D[j, i] = sum_k Q[j, k] P[i, k]      both operands with k contiguous, float32 sums
//
// A workgroup of WI x WJ wavefronts owns I = 32 TI WI by J = 32 TJ WJ results, each wavefront TI x TJ blocks of 32 x 32
// (v_mfma_f32_32x32x16_bf16: lane l holds row l % 32 of either operand at k = 8 (l / 32) + 0..7, and results
// j = l % 32, i = 8 (r / 4) + 4 (l / 32) + r % 4 of register r). P is the instruction's first operand so that a lane
// holds four consecutive i of one j: the contiguous direction of every result written here.
//
// k runs in blocks of 64. A block's rows lie in LDS as eight 16-byte pieces, piece c of row r at c ^ (r % 8): rows are
// 128 bytes apart, so eight rows that read the same k read eight different groups of banks.
//
// Float32 operands come as three bfloat16 planes (x = x0 + x1 + x2 exactly, |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x|) and are
// multiplied as six products, the smallest first: the three left out are at most 2^-23 of x w, 2^-26 or so at random.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ews_vec.h"

namespace ews {
namespace tiles {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
using vec::u32x4;

struct Operand {
  const uint16_t* p;
  int64_t ld;      // elements between rows, a multiple of 8
  int64_t plane;   // elements between planes
  int rows;        // rows that may be read (a tile's further rows read the last one)
};

template <int WI_, int WJ_, int TI_, int TJ_>
struct Tile {
  static constexpr int WI = WI_, WJ = WJ_, TI = TI_, TJ = TJ_;
  static constexpr int I = 32 * TI * WI, J = 32 * TJ * WJ;
  static constexpr int kThreads = 64 * WI * WJ;
  static constexpr int kSlab = 32 * TI;                    // consecutive i of one wavefront
  static constexpr int kRowWords = kSlab + 4;              // a staged result row, padded off the banks
  static constexpr int kStageBytes = WI * WJ * 32 * kRowWords * 4;
  static constexpr int kLoadBytes = (I + J) * 128;
  static constexpr int kLdsBytes = kStageBytes > kLoadBytes ? kStageBytes : kLoadBytes;
};

constexpr int kPairs = 6;
__device__ __forceinline__ int piece_p(int pair) { return (0x001102 >> (4 * pair)) & 15; }  // 2 0 1 1 0 0
__device__ __forceinline__ int piece_q(int pair) { return (0x010120 >> (4 * pair)) & 15; }  // 0 2 1 0 1 0

// One operand's rows of a k block, global memory to registers and on to LDS.
template <int ROWS, int THREADS>
struct Loader {
  static constexpr int kEach = ROWS * 8 / THREADS;
  u32x4 r[kEach];
  __device__ __forceinline__ void fetch(const Operand& o, int piece, int row0, int64_t k) {
#pragma unroll
    for (int c = 0; c < kEach; ++c) {
      const int idx = threadIdx.x + c * THREADS;
      const int row = idx >> 3, pos = idx & 7;
      const int src = row0 + row < o.rows ? row0 + row : o.rows - 1;
      r[c] = *reinterpret_cast<const u32x4*>(o.p + piece * o.plane + src * o.ld + k + 8 * (pos ^ (row & 7)));
    }
  }
  __device__ __forceinline__ void put(char* lds) const {
#pragma unroll
    for (int c = 0; c < kEach; ++c) *reinterpret_cast<u32x4*>(lds + (threadIdx.x + c * THREADS) * 16) = r[c];
  }
};

// The results of the workgroup's tile at (i0, j0) over k blocks [kb0, kb1); pairs: 1, or kPairs for three planes.
template <class T>
__device__ __forceinline__ void product(const Operand& P, const Operand& Q, int i0, int j0, int kb0, int kb1,
                                        int pairs, char* lds, f32x16 (&acc)[T::TI][T::TJ]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave % T::WI, wj = wave / T::WI;
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;
  if (kb0 >= kb1) return;
  char* ldsP = lds;
  char* ldsQ = lds + T::I * 128;
  Loader<T::I, T::kThreads> lp;
  Loader<T::J, T::kThreads> lq;
  const int steps = (kb1 - kb0) * pairs;
  auto fetch = [&](int s) {
    const int pair = pairs == 1 ? kPairs - 1 : s % pairs;
    const int64_t k = (int64_t)(kb0 + s / pairs) * 64;
    lp.fetch(P, piece_p(pair), i0, k);
    lq.fetch(Q, piece_q(pair), j0, k);
  };
  fetch(0);
  lp.put(ldsP);
  lq.put(ldsQ);
  __syncthreads();
  const int r32 = lane & 31, half = lane >> 5;
  const char* rowP = ldsP + (wi * T::TI * 32 + r32) * 128;
  const char* rowQ = ldsQ + (wj * T::TJ * 32 + r32) * 128;
  for (int s = 0; s < steps; ++s) {
    if (s + 1 < steps) fetch(s + 1);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      const int off = ((ks * 2 + half) ^ (r32 & 7)) * 16;
      bf16x8 fp[T::TI], fq[T::TJ];
#pragma unroll
      for (int a = 0; a < T::TI; ++a) fp[a] = *reinterpret_cast<const bf16x8*>(rowP + a * 32 * 128 + off);
#pragma unroll
      for (int b = 0; b < T::TJ; ++b) fq[b] = *reinterpret_cast<const bf16x8*>(rowQ + b * 32 * 128 + off);
#pragma unroll
      for (int a = 0; a < T::TI; ++a)
#pragma unroll
        for (int b = 0; b < T::TJ; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fp[a], fq[b], acc[a][b], 0, 0, 0);
    }
    __syncthreads();
    if (s + 1 < steps) {
      lp.put(ldsP);
      lq.put(ldsQ);
      __syncthreads();
    }
  }
}

// Tile coordinates of a workgroup. Consecutive workgroups go to the eight XCDs in turn; each XCD gets a contiguous
// stretch of tiles, walked in groups of eight j so that the tiles in flight on one XCD share rows in its L2.
__device__ __forceinline__ void tile_of(int id, int ti, int tj, int& i, int& j) {
  const int n = ti * tj, xcd = id & 7, at = id >> 3;
  const int each = n >> 3, more = n & 7;
  id = xcd * each + (xcd < more ? xcd : more) + at;
  const int group = id / (8 * ti);
  const int rest = id - group * 8 * ti;
  const int width = tj - group * 8 < 8 ? tj - group * 8 : 8;
  i = rest / width;
  j = group * 8 + rest % width;
}

// A wavefront's block column b of its results, staged through its own part of LDS and handed on as rows: f(jrow, i, x)
// gets eight consecutive results x of tile row jrow from tile column i on. Every lane of a row's lanes calls it.
template <class T, class F>
__device__ __forceinline__ void rows_of(char* lds, const f32x16 (&acc)[T::TI][T::TJ], int b, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave % T::WI, wj = wave / T::WI;
  float* stage = reinterpret_cast<float*>(lds) + wave * 32 * T::kRowWords;
  const int r32 = lane & 31, half = lane >> 5;
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<vec::f32x4*>(stage + r32 * T::kRowWords + a * 32 + g * 8 + half * 4) =
          vec::f32x4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  constexpr int kLanes = T::kSlab / 8;   // lanes of one row
#pragma unroll
  for (int it = 0; it < 32 * kLanes / 64; ++it) {
    const int row = it * (64 / kLanes) + lane / kLanes;
    const int col = (lane % kLanes) * 8;
    const float* s = stage + row * T::kRowWords + col;
    const vec::f32x4 lo = *reinterpret_cast<const vec::f32x4*>(s);
    const vec::f32x4 hi = *reinterpret_cast<const vec::f32x4*>(s + 4);
    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    f((wj * T::TJ + b) * 32 + row, wi * T::kSlab + col, x);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace tiles
}  // namespace ews
