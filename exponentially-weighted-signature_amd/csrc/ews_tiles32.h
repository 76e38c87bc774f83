// The products of ews_tiles.h with a float32 first operand read as it is: for products that its bytes bound, where
// packing it into planes first (read 4 bytes, write 6, read 12 in six products' stages) costs more than the
// products do. 128 rows by 30000 x 2048, logits and dh: 0.25 ms, 2.0 TB/s of W; 0.51 ms packed.
//
// k runs in stages of 32. The first operand's stage is copied to LDS in float32 (rows of 128 bytes, or turned: 32 rows
// of k, as wide as the tile) and cut into three bfloat16 planes in registers, on the way from LDS to the matrix cores;
// the second comes as three planes. A stage does all six products at once, so either is read once. Several workgroups
// share a CU and hide each other's waits: nothing is read ahead across the barrier. Rows that do not start at multiples
// of 16 bytes are copied four bytes a lane.
#pragma once

#include "ews_tiles.h"

namespace ews {
namespace tiles {

template <int TJ_, int BYTES>
struct Tile32 {
  static constexpr int WI = 4, WJ = 1, TI = 1, TJ = TJ_;
  static constexpr int I = 128, J = 32 * TJ;
  static constexpr int kThreads = 256;
  static constexpr int kWaves = 4;
  static constexpr int kSlab = 32;
  static constexpr int kRowWords = kSlab + 4;
  static constexpr int kStageBytes = WI * 32 * kRowWords * 4;
  static constexpr int kCopy = BYTES;                      // bytes a lane copies of the first operand at a time
  static constexpr int kCopiesP = I * 128 / BYTES / kThreads;
  static constexpr int kCopiesQ = (12 * J + kThreads - 1) / kThreads;
  static constexpr int kBytesP = I * 128;
  static constexpr int kStage = kBytesP + kCopiesQ * kThreads * 16;
  static constexpr int kLdsBytes = kStageBytes > 2 * kStage ? kStageBytes : 2 * kStage;
};

// The float32 operand: ld, rows and cols in numbers (ld and cols multiples of 4 where 16 bytes are copied at a time).
struct Operand32 {
  const float* p;
  int64_t ld;
  int rows, cols;
};

template <class T, bool TURNED>
struct Copier32 {
  static constexpr int kEach = T::kCopy / 4;                  // numbers a lane copies at a time
  static constexpr int kRow = (TURNED ? T::I : 32) / kEach;   // lanes to a stage's row
  const float* base;
  int64_t ld;
  int rows, cols, first;
  uint32_t offset[T::kCopiesP];
  __device__ __forceinline__ Copier32(const Operand32& o, int tile)
      : base(o.p), ld(o.ld), rows(o.rows), cols(o.cols), first(tile) {
    if (!TURNED) {
      first = first < rows ? first : rows - 1;
      base += first * ld;
    }
    aim(32);
  }
  // What each thread copies of a stage of `left` k; further ones read the last again (product32 takes them out).
  __device__ __forceinline__ void aim(int left) {
    const uint32_t stride = (uint32_t)ld * 4;
#pragma unroll
    for (int c = 0; c < T::kCopiesP; ++c) {
      const int idx = threadIdx.x + c * T::kThreads;
      const int row = idx / kRow, at = idx % kRow * kEach, pos = at >> 2, in = at & 3;
      if (TURNED) {
        // the halves of a wavefront read rows eight apart: in different banks
        const int col = first + 4 * (pos ^ (((row >> 3) & 1) << 3)) + in;
        offset[c] = (uint32_t)(row < left ? row : left - 1) * stride + 4 * (col < cols ? col : cols - kEach);
      } else {
        const int col = 4 * place(row, pos) + in;
        offset[c] = (uint32_t)(first + row < rows ? row : rows - 1 - first) * stride +
                    4 * (col < left ? col : left - kEach);
      }
    }
  }
  __device__ __forceinline__ const float* at(int kb) {
    const int left = (TURNED ? rows : cols) - kb * 32;
    if (left < 32) aim(left);
    return base + (int64_t)kb * 32 * (TURNED ? ld : 1);
  }
};

// Three planes of eight numbers. CAREFUL: finite numbers stay finite (the first plane is held to bfloat16's range), and
// an infinity is (1, 0, infinity) with its sign, as in planes() of ews_loss.hip. Otherwise infinities and numbers that
// round to one in bfloat16 have a plane of NaN, so that every result they are in is NaN.
template <bool CAREFUL>
__device__ __forceinline__ void cut(const float (&x)[8], bf16x8 (&p)[3]) {
  constexpr float kMost = 3.3895313892515355e+38f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const bool infinite = CAREFUL && __builtin_isinf(x[e]);
    p[0][e] = (__bf16)(infinite ? copysignf(1.0f, x[e]) : CAREFUL ? fminf(fmaxf(x[e], -kMost), kMost) : x[e]);
    const float b = x[e] - (float)p[0][e];
    p[1][e] = (__bf16)(infinite ? 0.0f : b);
    p[2][e] = (__bf16)(b - (float)p[1][e]);
  }
}

template <class T, bool TURNED, bool CAREFUL>
__device__ __forceinline__ void product32_once(const Operand32& P, const Operand& Q, int i0, int j0, int kb0, int kb1,
                                               char* lds, f32x16 (&acc)[T::TI][T::TJ]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int b = 0; b < T::TJ; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][b][r] = 0.0f;
  if (kb0 >= kb1) return;
  Copier32<T, TURNED> cp(P, i0);
  uint32_t offset[T::kCopiesQ];
#pragma unroll
  for (int c = 0; c < T::kCopiesQ; ++c) {
    int idx = threadIdx.x + c * T::kThreads;
    idx = idx < 12 * T::J ? idx : 12 * T::J - 1;  // what is over repeats the last piece, into a place nobody reads
    const int row = (idx >> 2) % T::J, src = j0 + row < Q.rows ? j0 + row : Q.rows - 1;
    offset[c] = (uint32_t)(2 * ((idx / (4 * T::J)) * Q.plane + src * Q.ld + 8 * ((idx & 3) ^ ((row >> 2) & 3))));
  }
  auto copy = [&](int kb, int half) {
    const float* fromP = cp.at(kb);
    const uint16_t* fromQ = Q.p + (int64_t)kb * 32;
    char* to = lds + half * T::kStage;
#pragma unroll
    for (int c = 0; c < T::kCopiesP; ++c)
      copy_piece<T::kCopy>(fromP, cp.offset[c], to + (wave * 64 + c * T::kThreads) * T::kCopy);
#pragma unroll
    for (int c = 0; c < T::kCopiesQ; ++c)
      copy_piece(fromQ, offset[c], to + T::kBytesP + (wave * 64 + c * T::kThreads) * 16);
  };
  const int r32 = lane & 31, half = lane >> 5;
  copy(kb0, 0);
  for (int kb = kb0, s = 0; kb < kb1; ++kb, s ^= 1) {
    arrive<0>();
    if (kb + 1 < kb1) copy(kb + 1, s ^ 1);
    const char* stage = lds + s * T::kStage;
#pragma unroll(CAREFUL ? 1 : 2)
    for (int ks = 0; ks < 2; ++ks) {
      float x[8];
      if (TURNED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = 16 * ks + 8 * half + e, col = wave * 32 + r32;
          x[e] =
              *reinterpret_cast<const float*>(stage + k * T::I * 4 + ((col >> 2) ^ (half << 3)) * 16 + (col & 3) * 4);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const vec::f32x4 w = *reinterpret_cast<const vec::f32x4*>(stage + (wave * 32 + r32) * 128 +
                                                                    place(wave * 32 + r32, 4 * ks + 2 * half + h) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * h + e] = w[e];
        }
      }
      if (CAREFUL) {  // k past the end: the other operand is zero there, but zero times an infinity is not
        const int left = (TURNED ? P.rows : P.cols) - kb * 32;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 16 * ks + 8 * half + e < left ? x[e] : 0.0f;
      }
      bf16x8 p[3], q[3][T::TJ];
#pragma unroll
      for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int b = 0; b < T::TJ; ++b)
          q[n][b] = *reinterpret_cast<const bf16x8*>(stage + T::kBytesP + (n * T::J + b * 32 + r32) * 64 +
                                                     ((2 * ks + half) ^ ((r32 >> 2) & 3)) * 16);
      cut<CAREFUL>(x, p);
#pragma unroll
      for (int pair = 0; pair < kPairs; ++pair)
#pragma unroll
        for (int b = 0; b < T::TJ; ++b)
          acc[0][b] =
              __builtin_amdgcn_mfma_f32_32x32x16_bf16(p[piece_p(pair)], q[piece_q(pair)][b], acc[0][b], 0, 0, 0);
    }
  }
  arrive<0>();
}

// As product() of ews_tiles.h; k blocks are of 32. A tile with a NaN is formed once more, with care: infinities cost
// such tiles twice the time and the others nothing (told apart number by number they cost all calls 3 to 10%).
template <class T, bool TURNED>
__device__ __forceinline__ void product32(const Operand32& P, const Operand& Q, int i0, int j0, int kb0, int kb1,
                                          char* lds, f32x16 (&acc)[T::TI][T::TJ]) {
  product32_once<T, TURNED, false>(P, Q, i0, j0, kb0, kb1, lds, acc);
  bool bad = false;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad |= __builtin_isnan(acc[0][b][r]);
  int* flags = reinterpret_cast<int*>(lds);  // nobody reads a stage any more
  bad = __any(bad);
  if ((threadIdx.x & 63) == 0) flags[threadIdx.x >> 6] = bad;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T::WI * T::WJ; ++w) bad |= flags[w] != 0;
  __syncthreads();
  if (bad) product32_once<T, TURNED, true>(P, Q, i0, j0, kb0, kb1, lds, acc);
}

}  // namespace tiles
}  // namespace ews
