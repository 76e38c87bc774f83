// Matrix products of bfloat16 operands on the matrix cores of MI355X (gfx950), as tiles for kernels with epilogues of
// their own (ews_loss.hip, ews_gated.hip).
//
//   D[j, i] = sum_k Q[j, k] P[i, k]      float32 sums; each operand with k contiguous, or stored turned, k its rows
//
// A workgroup of WI x WJ wavefronts owns I = 32 TI WI by J = 32 TJ WJ results, each wavefront TI x TJ blocks of 32 x 32
// (v_mfma_f32_32x32x16_bf16: lane l holds row l % 32 of either operand at k = 8 (l / 32) + 0..7, and results
// j = l % 32, i = 8 (r / 4) + 4 (l / 32) + r % 4 of register r). P is the instruction's first operand so that a lane
// holds four consecutive i of one j: the contiguous direction of every result written here.
//
// k runs in stages of 64. A stage's rows (128 bytes each: whole cache lines) are copied straight from global memory to
// LDS (buffer loads to LDS: no registers, no instructions to store them) into one half of the tile's LDS while the
// other half is multiplied. Operands are read sixteen k ahead of their products, so when a stage's last sixteen are in
// registers its half is free: there is the stage's one barrier. Before it a wavefront waits until its own copies of the
// next stage have arrived; after it the products go on at once, and the copies of the stage after the next begin.
// Reads and copies go out one by one between products that do not wait for them.
//
// The 16-byte piece c of row r lies at c ^ (r / 2) % 8. A 16-byte read serves lanes {0-3, 12-15, 20-27}, then {4-11,
// 16-19, 28-31}, and so the other half: the rows of each such sixteen lie in sixteen different groups of four banks.
//
// A turned operand's stage is 64 rows of k, each as wide as the tile. It is read by the LDS's transposing reads
// (sixteen lanes name four rows of k by sixteen columns, each gets four k of its column), two to a fragment, so nothing
// is turned in memory. Piece c of row k lies at c ^ 4 (k % 4): the four rows that 32 lanes read at a time are in
// different banks.
//
// 256 x 256 tiles of eight wavefronts (two a SIMD, 128 KB of LDS) run at 1.16 PFLOP/s in products of 7400 x 2048 x
// 32000 and at 1.10 to 1.22 in ten times larger ones; the library's products of the same sizes, calls in a row, at 0.89
// (32000 summed) and 1.17 (2048 summed), and at 1.16.
//
// Float32 operands come as three bfloat16 planes (x = x0 + x1 + x2 exactly, |x1| <= 2^-8 |x|, |x2| <= 2^-16 |x|) and
// are multiplied as six products, the smallest first: the three left out are at most 2^-23 of x w, 2^-26 or so at
// random.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ews_vec.h"

namespace ews {
namespace tiles {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
using vec::u32x4;

struct Operand {
  const uint16_t* p;
  int64_t ld;      // elements between rows, a multiple of 8, 2^22 at most
  int64_t plane;   // elements between planes
  int rows;        // rows that may be read; what a tile has beyond them reads the last one
  int cols;        // turned: columns that may be read, a multiple of 8, likewise
};

template <int WI_, int WJ_, int TI_, int TJ_>
struct Tile {
  static constexpr int WI = WI_, WJ = WJ_, TI = TI_, TJ = TJ_;
  static constexpr int I = 32 * TI * WI, J = 32 * TJ * WJ;
  static constexpr int kThreads = 64 * WI * WJ;
  static constexpr int kWaves = TI * TJ > 4 ? 2 : 4;       // on a SIMD, as far as registers go
  static constexpr int kSlab = 32 * TI;                    // consecutive i of one wavefront
  static constexpr int kRowWords = kSlab + 4;              // a staged result row, padded off the banks
  static constexpr int kStageBytes = WI * WJ * 32 * kRowWords * 4;
  static constexpr int kCopiesP = I * 8 / kThreads;        // 16-byte pieces a thread copies in a stage
  static constexpr int kCopiesQ = J * 8 / kThreads;
  static constexpr int kBytesP = kCopiesP * kThreads * 16;
  static constexpr int kStage = (kCopiesP + kCopiesQ) * kThreads * 16;
  static constexpr int kLdsBytes = kStageBytes > 2 * kStage ? kStageBytes : 2 * kStage;
  static constexpr int kLdsBytesOne = kStageBytes > kStage ? kStageBytes : kStage;  // for products of one stage
};

constexpr int kPairs = 6;
__device__ __forceinline__ constexpr int piece_p(int pair) { return (0x001102 >> (4 * pair)) & 15; }  // 2 0 1 1 0 0
__device__ __forceinline__ constexpr int piece_q(int pair) { return (0x010120 >> (4 * pair)) & 15; }  // 0 2 1 0 1 0

__device__ __forceinline__ int place(int row, int piece) { return piece ^ ((row >> 1) & 7); }
template <int WIDTH>
__device__ __forceinline__ int place_turned(int k, int piece) {
  return WIDTH >= 128 ? piece ^ ((k & 3) << 2) : piece;
}

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// BYTES (16 or 4) a lane from `from` + offset to `to` on. Written out, not a builtin: before every transposing read the
// compiler would wait for all the copies that it knows of. It has no result in a register; who reads what it wrote
// waits in arrive().
template <int BYTES = 16>
__device__ __forceinline__ void copy_piece(const void* from, uint32_t offset, char* to) {
  const uint64_t at = (uint64_t)from;
  const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu, 0xffffffffu, 0x00020000u};
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)to;
  if (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset),
                 "s"(rsrc)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset),
                 "s"(rsrc)
                 : "memory", "m0");
}

// One operand of a tile, WIDTH results wide: what each thread copies of a stage.
template <bool TURNED, int WIDTH, int THREADS>
struct Copier {
  static constexpr int kCopies = WIDTH * 8 / THREADS;
  static constexpr int kPieces = TURNED ? WIDTH / 8 : 8;  // pieces of a stage's row
  const uint16_t* base;
  int64_t plane;
  uint32_t stride;           // bytes between rows
  int rows, first, cols;
  uint32_t offset[kCopies];  // bytes from the stage's first row
  __device__ __forceinline__ Copier(const Operand& o, int tile)
      : plane(o.plane), stride((uint32_t)o.ld * 2), rows(o.rows), first(tile), cols(o.cols) {
    if (TURNED) {
      base = o.p;
      aim_turned(63);
    } else {
      first = first < rows ? first : rows - 1;
      base = o.p + first * o.ld;
#pragma unroll
      for (int c = 0; c < kCopies; ++c) {
        const int idx = threadIdx.x + c * THREADS;
        const int row = idx / kPieces;
        offset[c] = (uint32_t)(first + row < rows ? row : rows - 1 - first) * stride + 16 * place(row, idx % kPieces);
      }
    }
  }
  // Turned: a stage's rows of k, those past `last` read it again.
  __device__ __forceinline__ void aim_turned(int last) {
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const int idx = threadIdx.x + c * THREADS;
      const int k = idx / kPieces;
      const int col = first + 8 * place_turned<WIDTH>(k, idx % kPieces);
      offset[c] = (uint32_t)(k < last ? k : last) * stride + 2 * (col < cols ? col : cols - 8);
    }
  }
  // The address of k block kb; blocks are asked for in order, so one that is not whole is the last.
  __device__ __forceinline__ const uint16_t* at(int piece, int kb) {
    if (!TURNED) return base + piece * plane + (int64_t)kb * 64;
    if (rows - kb * 64 < 64) aim_turned(rows - 1 - kb * 64);
    return base + piece * plane + (int64_t)kb * 64 * (stride / 2);
  }
  // One of the copies; `to`: this wavefront's kilobyte of the stage.
  __device__ __forceinline__ void copy(int c, const uint16_t* from, char* to) const {
    copy_piece(from, offset[c], to + c * THREADS * 16);
  }
};

// The first operand's copier: a kernel may bring an operand of a type of its own.
template <class O, class T, bool TURNED>
struct CopierOf {
  typedef Copier<TURNED, T::I, T::kThreads> type;
};

// A wavefront's fragments of one operand: BLOCKS blocks of 32 from block `first` of the tile on.
template <bool TURNED, int WIDTH, int BLOCKS>
struct Reader {
  int at[TURNED ? BLOCKS : 4];
  __device__ __forceinline__ Reader(int first, int lane) {
    const int r32 = lane & 31, half = lane >> 5;
    if (TURNED) {
      const int k = (lane >> 2) & 3;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
        at[b] = (8 * half + k) * WIDTH * 2 +
                place_turned<WIDTH>(k, (first + b) * 4 + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) * 16 +
                (lane & 1) * 8;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) at[k] = (first * 32 + r32) * 128 + place(r32, 2 * k + half) * 16;
    }
  }
  // Block b at the stage's k-th sixteen.
  __device__ __forceinline__ bf16x8 get(char* stage, int k, int b) const {
    if (!TURNED) return *reinterpret_cast<const bf16x8*>(stage + at[k] + b * 4096);
#if defined(__HIP_DEVICE_COMPILE__)  // the host's pass does not know the builtin
    char* from = stage + at[b] + k * 16 * WIDTH * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)from);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(from + 4 * WIDTH * 2));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#else
    return bf16x8{};
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

// The results of the workgroup's tile at (i0, j0) over k blocks [kb0, kb1); PAIRS: 1, 2 for two planes of Q alone, or
// kPairs for three of either. On return LDS is free.
template <class T, int PAIRS, bool TURNED_P, bool TURNED_Q, class O>
__device__ __forceinline__ void product(const O& P, const Operand& Q, int i0, int j0, int kb0, int kb1,
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
  typename CopierOf<O, T, TURNED_P>::type cp(P, i0);
  Copier<TURNED_Q, T::J, T::kThreads> cq(Q, j0);
  const int stages = (kb1 - kb0) * PAIRS;
  constexpr int kCopies = T::kCopiesP + T::kCopiesQ, kReads = T::TI + T::TJ, kProducts = T::TI * T::TJ;
  constexpr int kMost = kReads > kProducts ? kReads : kProducts, kSlots = kMost > kCopies ? kMost : kCopies;
  const uint16_t *fromP, *fromQ;
  char* to;
  auto aim = [&](int s) {
    const int pair = PAIRS == 1 ? kPairs - 1 : s % PAIRS;
    fromP = cp.at(PAIRS == 2 ? 0 : piece_p(pair), kb0 + s / PAIRS);
    fromQ = cq.at(PAIRS == 2 ? 1 - pair : piece_q(pair), kb0 + s / PAIRS);
    to = lds + (s & 1) * T::kStage + wave * 1024;
  };
  auto copy = [&](int c) {
    if (c < T::kCopiesP)
      cp.copy(c, fromP, to);
    else
      cq.copy(c - T::kCopiesP, fromQ, to + T::kBytesP);
  };
  const Reader<TURNED_P, T::I, T::TI> rp(wi * T::TI, lane);
  const Reader<TURNED_Q, T::J, T::TJ> rq(wj * T::TJ, lane);
  struct Sixteen {
    bf16x8 p[T::TI], q[T::TJ];
  } even, odd;
  // the n-th of a sixteen's reads: the first product's two first
  auto read = [&](Sixteen& f, int s, int k, int n) {
    char* stage = lds + (s & 1) * T::kStage;
    if (n >= 1 && n <= T::TJ)
      f.q[n - 1] = rq.get(stage + T::kBytesP, k, n - 1);
    else
      f.p[n ? n - T::TJ : 0] = rp.get(stage, k, n ? n - T::TJ : 0);
  };
  // the products of one sixteen, and between them the reads of sixteen k of stage s and where asked its successor's
  // copies
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
  auto stage = [&](int s, bool copies) {
    arrive<0>();
    if (copies) aim(s + 1);
    multiply(odd, even, s, 0, copies);  // the stage before's last sixteen (at first nothing)
    multiply(even, odd, s, 1, false);
    multiply(odd, even, s, 2, false);
    multiply(even, odd, s, 3, false);
  };
  for (int s = 0; s + 1 < stages; ++s) stage(s, true);
  stage(stages - 1, false);
#pragma unroll
  for (int a = 0; a < T::TI; ++a)
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
      acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(odd.p[a], odd.q[b], acc[a][b], 0, 0, 0);
  arrive<0>();
}

// Tile coordinates of a workgroup. Consecutive workgroups go to the eight XCDs in turn; each XCD gets a contiguous
// stretch of tiles, walked in groups of up to eight j, as equal as can be, so that the tiles in flight on one XCD share
// rows in its L2 (41 j in five groups of eight and one of one: 0.83 PFLOP/s where 32 in four reach 1.06).
__device__ __forceinline__ void tile_of(int id, int ti, int tj, int& i, int& j) {
  const int n = ti * tj, xcd = id & 7, at = id >> 3;
  const int each = n >> 3, more = n & 7;
  id = xcd * each + (xcd < more ? xcd : more) + at;
  const int groups = (tj + 7) >> 3;
  const int wide = tj / groups, wider = tj % groups;  // the first `wider` groups have one j more
  const int split = wider * (wide + 1) * ti;
  int group, rest, width;
  if (id < split) {
    width = wide + 1;
    group = id / (width * ti);
    rest = id - group * width * ti;
    j = group * width;
  } else {
    width = wide;
    group = (id - split) / (width * ti);
    rest = id - split - group * width * ti;
    j = wider * (wide + 1) + group * width;
  }
  i = rest / width;
  j += rest % width;
}

struct Eight {
  float x[8];
};
struct One {
  float x;
};

// A wavefront's block column b of its results, staged through its own part of LDS and handed on as rows of numbers of
// type W: f(jrow, i, x) gets the results of tile row jrow from tile column i on; float and uint16_t (65535ths of
// results held to [0, 1]) 16 bytes of them, Eight eight floats, One one, neighbouring lanes neighbouring results.
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
            vec::u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(x[0], x[1])),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(x[2], x[3]))};
      else
        *reinterpret_cast<vec::f32x4*>(stage + at) = x;
    }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  constexpr bool kOne = std::is_same<W, One>::value;
  constexpr int kEach = kOne ? 1 : sizeof(W) == sizeof(Eight) ? 8 : 16 / (int)sizeof(W);  // numbers handed on at a time
  constexpr int kLanes = T::kSlab / kEach < 64 ? T::kSlab / kEach : 64;                   // lanes of one row
  if constexpr (kOne) {
    for (int row = 0; row < 32; ++row)
#pragma unroll
      for (int c = 0; c < T::kSlab; c += 64)
        if (T::kSlab >= 64 || lane < T::kSlab)
          f((wj * T::TJ + b) * 32 + row, wi * T::kSlab + c + lane,
            One{*reinterpret_cast<const float*>(stage + row * kRow + (c + lane) * 4)});
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    return;
  }
  constexpr int kBytes = kHalf ? 16 : 4 * kEach;
#pragma unroll
  for (int it = 0; it < (kOne ? 0 : 32 * kLanes / 64); ++it) {
    const int row = it * (64 / kLanes) + lane / kLanes;
    const char* s = stage + row * kRow + (lane % kLanes) * kBytes;
    const int j = (wj * T::TJ + b) * 32 + row, i = wi * T::kSlab + (lane % kLanes) * kEach;
    const u32x4 lo = *reinterpret_cast<const u32x4*>(s);
    if constexpr (kOne) {
    } else if constexpr (kEach == 8 && !kHalf) {
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
