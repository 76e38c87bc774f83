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
// k runs in stages of 64. A stage's rows (128 bytes each: whole cache lines) are copied straight from global memory to
// LDS (buffer loads to LDS: no registers, no instructions to store them) into one half of the tile's LDS while the other
// half is multiplied. Operands are read sixteen k ahead of their products, so when a stage's last sixteen are in
// registers its half is free: there is the stage's one barrier. Before it a wavefront waits until its own copies of the
// next stage have arrived; after it the products go on at once, and the copies of the stage after the next begin.
// Reads and copies go out one by one between products that do not wait for them.
// The 16-byte piece c of row r lies at c ^ (r / 2) % 8. A 16-byte read serves lanes {0-3, 12-15, 20-27}, then {4-11,
// 16-19, 28-31}, and so the other half: the rows of each such sixteen lie in sixteen different groups of four banks.
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
  static constexpr int kCopiesP = I * 8 / kThreads;        // 16-byte pieces a thread copies in a stage
  static constexpr int kCopiesQ = J * 8 / kThreads;
  static constexpr int kBytesP = kCopiesP * kThreads * 16;
  static constexpr int kStage = (kCopiesP + kCopiesQ) * kThreads * 16;
  static constexpr int kLdsBytes = kStageBytes > 2 * kStage ? kStageBytes : 2 * kStage;
};

constexpr int kPairs = 6;
__device__ __forceinline__ int piece_p(int pair) { return (0x001102 >> (4 * pair)) & 15; }  // 2 0 1 1 0 0
__device__ __forceinline__ int piece_q(int pair) { return (0x010120 >> (4 * pair)) & 15; }  // 0 2 1 0 1 0

__device__ __forceinline__ int place(int row, int piece) { return piece ^ ((row >> 1) & 7); }

typedef __attribute__((address_space(3))) void lds_void;

// One operand's rows of a tile: what each thread copies, and the copies of a stage.
template <int COPIES, int THREADS>
struct Copier {
  const uint16_t* base;
  int64_t plane;
  int offset[COPIES];   // bytes from the tile's first row; at most 256 rows of 2^22 numbers apart
  __device__ __forceinline__ Copier(const Operand& o, int row0) {
    row0 = row0 < o.rows ? row0 : o.rows - 1;
    base = o.p + row0 * o.ld;
    plane = o.plane;
#pragma unroll
    for (int c = 0; c < COPIES; ++c) {
      const int idx = threadIdx.x + c * THREADS;
      const int row = idx >> 3;
      const int src = row0 + row < o.rows ? row : o.rows - 1 - row0;
      offset[c] = (int)((uint32_t)src * (uint32_t)(o.ld * 2) + 16 * place(row, idx & 7));
    }
  }
  // The address of the rows of k block kb.
  __device__ __forceinline__ const uint16_t* at(int piece, int kb) const {
    return base + piece * plane + (int64_t)kb * 64;
  }
  // One of the copies; `to`: this wavefront's kilobyte of the stage.
  __device__ __forceinline__ void copy(int c, const uint16_t* from, char* to) const {
#if defined(__HIP_DEVICE_COMPILE__)  // the host's pass does not know the buffer builtins
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)from, 0, -1, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + c * THREADS * 16), 16, offset[c], 0, 0, 0);
#endif
  }
};

// Waits until no more than N of this wavefront's loads are on their way and its LDS reads are done, then for everyone.
template <int N>
__device__ __forceinline__ void arrive() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The results of the workgroup's tile at (i0, j0) over k blocks [kb0, kb1); PAIRS: 1, or kPairs for three planes. On
// return LDS is free.
template <class T, int PAIRS>
__device__ __forceinline__ void product(const Operand& P, const Operand& Q, int i0, int j0, int kb0, int kb1,
                                        char* lds, f32x16 (&acc)[T::TI][T::TJ]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wi = wave % T::WI, wj = wave / T::WI;
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.0f;
  if (kb0 >= kb1) return;
  const Copier<T::kCopiesP, T::kThreads> cp(P, i0);
  const Copier<T::kCopiesQ, T::kThreads> cq(Q, j0);
  const int stages = (kb1 - kb0) * PAIRS;
  constexpr int kCopies = T::kCopiesP + T::kCopiesQ, kReads = T::TI + T::TJ, kProducts = T::TI * T::TJ;
  constexpr int kMost = kReads > kProducts ? kReads : kProducts, kSlots = kMost > kCopies ? kMost : kCopies;
  // past the last stage the copies repeat it, into a half that nobody reads again
  const uint16_t *fromP, *fromQ;
  char* to;
  auto aim = [&](int s) {
    const int t = s < stages ? s : stages - 1;
    const int pair = PAIRS == 1 ? kPairs - 1 : t % PAIRS;
    fromP = cp.at(piece_p(pair), kb0 + t / PAIRS);
    fromQ = cq.at(piece_q(pair), kb0 + t / PAIRS);
    to = lds + (s & 1) * T::kStage + wave * 1024;
  };
  auto copy = [&](int c) {
    if (c < T::kCopiesP)
      cp.copy(c, fromP, to);
    else
      cq.copy(c - T::kCopiesP, fromQ, to + T::kBytesP);
  };
  const int r32 = lane & 31, half = lane >> 5;
  const int atP = (wi * T::TI * 32 + r32) * 128, atQ = T::kBytesP + (wj * T::TJ * 32 + r32) * 128;
  int at[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) at[k] = place(r32, 2 * k + half) * 16;
  struct Sixteen {
    bf16x8 p[T::TI], q[T::TJ];
  } even, odd;
  // the n-th of a sixteen's reads: the first product's two first
  auto read = [&](Sixteen& f, int s, int k, int n) {
    const char* stage = lds + (s & 1) * T::kStage + at[k];
    if (n >= 1 && n <= T::TJ)
      f.q[n - 1] = *reinterpret_cast<const bf16x8*>(stage + atQ + (n - 1) * 4096);
    else
      f.p[n ? n - T::TJ : 0] = *reinterpret_cast<const bf16x8*>(stage + atP + (n ? n - T::TJ : 0) * 4096);
  };
  // the products of one sixteen, and between them the reads of sixteen k of stage s and where asked its successor's copies
  auto multiply = [&](const Sixteen& f, Sixteen& next, int s, int k, bool copies) {
#pragma unroll
    for (int i = 0; i < kSlots; ++i) {
      if (i < kReads) read(next, s, k, i);
      if (copies && i < kCopies) copy(i);
      if (i < kProducts) {
        const int a = i / T::TJ, b = i % T::TJ;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.p[a], f.q[b], acc[a][b], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0x6);  // scalar and vector arithmetic may move past
    }
  };
  aim(0);
#pragma unroll
  for (int c = 0; c < kCopies; ++c) copy(c);
  const bf16x8 zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int a = 0; a < T::TI; ++a) odd.p[a] = zero;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) odd.q[b] = zero;
  for (int s = 0; s < stages; ++s) {
    arrive<0>();
    aim(s + 1);
    multiply(odd, even, s, 0, true);  // the stage before's last sixteen (at first nothing)
    multiply(even, odd, s, 1, false);
    multiply(odd, even, s, 2, false);
    multiply(even, odd, s, 3, false);
  }
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
      acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(odd.p[a], odd.q[b], acc[a][b], 0, 0, 0);
  arrive<0>();
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

struct Eight {
  float x[8];
};

// A wavefront's block column b of its results, staged through its own part of LDS and handed on as rows of numbers of
// type W: f(jrow, i, x) gets the results of tile row jrow from tile column i on; float and uint16_t (whole numbers, cut
// from floats in range) 16 bytes of them, Eight eight floats.
template <class T, typename W, class F>
__device__ __forceinline__ void rows_of(char* lds, const f32x16 (&acc)[T::TI][T::TJ], int b, F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave % T::WI, wj = wave / T::WI;
  char* stage = lds + wave * 32 * T::kRowWords * 4;
  const int r32 = lane & 31, half = lane >> 5;
  constexpr bool kHalf = sizeof(W) == 2;
  constexpr int kRow = kHalf ? T::kSlab * 2 + 16 : T::kRowWords * 4;  // bytes between rows
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const vec::f32x4 x = {acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
      const int at = r32 * kRow + (a * 32 + g * 8 + half * 4) * (kHalf ? 2 : 4);
      if (kHalf)
        *reinterpret_cast<vec::u32x2*>(stage + at) =
            vec::u32x2{(uint32_t)x[0] | ((uint32_t)x[1] << 16), (uint32_t)x[2] | ((uint32_t)x[3] << 16)};
      else
        *reinterpret_cast<vec::f32x4*>(stage + at) = x;
    }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  constexpr int kEach = sizeof(W) == sizeof(Eight) ? 8 : 16 / (int)sizeof(W);  // numbers handed on at a time
  constexpr int kLanes = T::kSlab / kEach;                                     // lanes of one row
  constexpr int kBytes = kHalf ? 16 : 4 * kEach;
#pragma unroll
  for (int it = 0; it < 32 * kLanes / 64; ++it) {
    const int row = it * (64 / kLanes) + lane / kLanes;
    const char* s = stage + row * kRow + (lane % kLanes) * kBytes;
    const int j = (wj * T::TJ + b) * 32 + row, i = wi * T::kSlab + (lane % kLanes) * kEach;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(s);
    if constexpr (kEach == 8 && !kHalf) {
      const vec::f32x4 x = __builtin_bit_cast(vec::f32x4, lo), y = *reinterpret_cast<const vec::f32x4*>(s + 16);
      f(j, i, Eight{{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}});
    } else {
      f(j, i, lo);
    }
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

}  // namespace tiles
}  // namespace ews
