// Operands of the products of ews_tiles.h laid out for them: rows of whole k blocks with zeros behind their columns,
// float32 numbers as three bfloat16 planes.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ews_vec.h"

namespace ews {
namespace tiles {

using namespace ews::vec;

// The three bfloat16 planes of a float32 number, x = p0 + p1 + p2 exactly: each plane is the rest rounded to eight bits
// (cut where rounding would reach infinity), so the second is at most 2^-8 and the third 2^-16 of x. A NaN has nothing
// after its first plane. An infinity is (1, 0, infinity) with its sign: the third plane meets the other side's first
// alone, which has the sign of the whole (and is 0 where it is), while the 1 meets the third plane of an infinity on
// the other side. So infinity times w is the infinity of its sign for w other than 0, and NaN for 0, as it has to be.
__device__ __forceinline__ float plane_value(uint16_t p) { return __uint_as_float((uint32_t)p << 16); }
__device__ __forceinline__ void planes(float x, uint16_t (&p)[3]) {
  const uint32_t u = __float_as_uint(x);
  const bool finite = (u & 0x7f800000u) != 0x7f800000u;
  p[0] = round_bf16(x);
  if (finite && (p[0] & 0x7f80u) == 0x7f80u) p[0] = (uint16_t)(u >> 16);
  const float b = finite ? x - plane_value(p[0]) : 0.0f;
  p[1] = round_bf16(b);
  p[2] = round_bf16(b - plane_value(p[1]));
  if ((u & 0x7fffffffu) == 0x7f800000u) {
    p[2] = p[0];
    p[0] = (uint16_t)((u >> 16 & 0x8000u) | 0x3f80u);
  }
}
__device__ __forceinline__ void planes(bf16 x, uint16_t (&p)[1]) { p[0] = x.bits; }

struct PackArgs {
  const void* src;
  int64_t stride;
  int rows, cols;          // of the source (rows: kept[0] where there is a map)
  const int* map;          // gathers the rows; null: all of them
  const int* kept;
  uint16_t* dst;           // planes (dst_rows, ld), zero in further columns and, if any, in rows up to a multiple of 64
  int64_t ld, plane;
  int dst_rows;
  int again;               // the rows are written once more from this one on; 0: once
  int wide;
};

// A thread takes eight columns of a row; wide: rows of the source start at multiples of 16 bytes.
template <typename T>
__device__ __forceinline__ void pack_eight(const PackArgs& a, int64_t at) {
  constexpr int NP = sizeof(T) == 4 ? 3 : 1;
  const int rows = a.map ? a.kept[0] : a.rows;
  const int padded = a.again || (rows + 63) / 64 * 64 > a.dst_rows ? a.dst_rows : (rows + 63) / 64 * 64;
  const int packs = (int)(a.ld / 8);
  const int64_t row = at / packs;
  if (row >= padded) return;
  const int c0 = (int)(at % packs) * 8;
  const int64_t own = a.again && row >= a.again ? row - a.again : row;
  const int n = own >= rows ? 0 : a.cols - c0 < 8 ? a.cols - c0 : 8;
  T x[8];
  const T* src = (const T*)a.src + (n > 0 ? (int64_t)(a.map ? a.map[own] : own) * a.stride + c0 : 0);
  if (a.wide && n == 8) {
#pragma unroll
    for (int k = 0; k < 8; k += kWide<T>) *reinterpret_cast<u32x4*>(x + k) = *reinterpret_cast<const u32x4*>(src + k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = k < n ? src[k] : narrow<T>(0.0f);
  }
  uint16_t p[8][NP];
#pragma unroll
  for (int k = 0; k < 8; ++k) planes(x[k], p[k]);
#pragma unroll
  for (int q = 0; q < NP; ++q) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (uint32_t)p[2 * k][q] | ((uint32_t)p[2 * k + 1][q] << 16);
    *reinterpret_cast<u32x4*>(a.dst + q * a.plane + row * a.ld + c0) = w;
  }
}

template <typename T>
static __global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  pack_eight<T>(a, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

}  // namespace tiles
}  // namespace ews
