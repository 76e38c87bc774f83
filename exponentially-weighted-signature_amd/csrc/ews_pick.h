// Which tile a product of ews_tiles.h or ews_tiles32.h runs on, by its sizes, and what its launch needs.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ews_hip.h"
#include "ews_tiles.h"
#include "ews_tiles32.h"

namespace ews {
namespace tiles {

typedef Tile<2, 4, 4, 2> Large;   // 256 x 256, eight wavefronts
typedef Tile<2, 2, 2, 2> Medium;  // 128 x 128, four wavefronts
typedef Tile<4, 1, 2, 1> Flat;    // 256 x 32, four wavefronts: few rows
template <int BYTES>
using Few32 = Tile32<1, BYTES>;   // 128 x 32 and 128 x 64, float32 W read as it is: few rows
template <int BYTES>
using More32 = Tile32<2, BYTES>;

// A product of one stage needs no second half: more workgroups share a CU.
template <class T, int PAIRS>
__host__ __device__ constexpr int lds_bytes(int kblocks) {
  if constexpr (PAIRS == 1) {
    if (kblocks == 1) return T::kLdsBytesOne;
  }
  return T::kLdsBytes;
}

// Stages below which a 128 x 128 tile is no slower (6 stages: 86 us for 94), its CUs better shared.
constexpr int kLongProduct = 8;

enum Kind { kLarge, kMedium, kFlat, kFew32, kMore32 };

struct Product {
  Kind kind;
  int ti, tj, tile_i, tile_j, slab, splits, per, kblocks, pairs;
};

inline size_t al256x(size_t x) { return (x + 255) & ~(size_t)255; }

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// A product of I x J results over kblocks of k: 256 x 32 tiles where J fits one; 256 x 256 ones where they give (split
// over k, where that is allowed, into parts of 16 blocks at least) half the CUs work; else 128 x 128 ones, of which a
// CU holds two. Measured at float32 N=4095 H=512 V=32000, dh (30 large tiles, split by 8): 0.55 ms, 0.80 ms with the
// small. as_is: float32 W is read as it is, in k blocks of 32.
inline Product pick(int64_t I, int64_t J, int kblocks, int pairs, bool split, bool as_is) {
  Product p;
  p.kblocks = kblocks;
  p.pairs = pairs;
  const int64_t large = (int64_t)ceil_div(I, 256) * ceil_div(J, 256);
  const int parts = split ? (kblocks >= 32 ? kblocks / 16 : 1) : 1;
  if (as_is)
    p.kind = J <= 32 ? kFew32 : kMore32;
  else if (J <= 32)
    p.kind = kFlat;
  else
    p.kind = I > 128 && J > 128 && large * parts >= 128 && kblocks * pairs >= kLongProduct ? kLarge : kMedium;
  const int tile_i[] = {Large::I, Medium::I, Flat::I, Few32<16>::I, More32<16>::I};
  const int tile_j[] = {Large::J, Medium::J, Flat::J, Few32<16>::J, More32<16>::J};
  const int slab[] = {Large::kSlab, Medium::kSlab, Flat::kSlab, Few32<16>::kSlab, More32<16>::kSlab};
  p.slab = slab[p.kind];
  p.tile_i = tile_i[p.kind];
  p.tile_j = tile_j[p.kind];
  p.ti = ceil_div(I, p.tile_i);
  p.tj = ceil_div(J, p.tile_j);
  p.splits = 1;
  p.per = kblocks;
  // one round of workgroups: a CU holds one of the large tiles, two of the others
  const int64_t n = (int64_t)p.ti * p.tj, room = p.kind == kLarge ? 256 : as_is ? 1024 : 512;
  if (split && 2 * n <= room) {
    int64_t z = room / n;
    const int64_t most = p.kind == kLarge ? parts : kblocks * pairs / 4 < kblocks ? kblocks * pairs / 4 : kblocks;
    if (z > most) z = most;
    if (z > 128) z = 128;  // each split's results are written and read once more
    if (z > 1) {
      p.per = ceil_div(kblocks, z);
      p.splits = ceil_div(kblocks, p.per);
    }
  }
  return p;
}

template <class K>
inline int allow_lds(K kernel, int bytes) {
  if (bytes <= 64 << 10) return EWS_OK;  // allowed as it is
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             bytes) == hipSuccess
             ? EWS_OK
             : EWS_ERR_LAUNCH;
}

inline int rows_wide(const void* p, int64_t stride, bool f32) {
  return (uintptr_t)p % 16 == 0 && stride * (f32 ? 4 : 2) % 16 == 0;
}

}  // namespace tiles
}  // namespace ews
