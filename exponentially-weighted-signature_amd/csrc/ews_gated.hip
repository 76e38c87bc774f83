// Gated linear map of a channel stage on MI355X (gfx950), forward and backward.
//
//   v = x V^T + b      g = x G^T + c      y = v act(g)
//   dv = dy act(g)     dg = dy v act'(g)
//   dx = dv V + dg G   dV = dv^T x   dG = dg^T x   db = sum_n dv   dc = sum_n dg
//
// act: the logistic function s, g s(g), g s(2 sqrt(2/pi) (g + 0.044715 g^3)) (the tanh form of GELU), or max(g, 0).
//
// Three pairs of products of 2 N H F operations each bound all but the smallest calls; they run on the matrix cores
// (ews_tiles.h). v and g of the same output meet in a wavefront's registers: a tile's first operand is interleaved,
// half of every wavefront's rows from V and half from G, which costs nothing, as the copies to LDS can start anywhere.
// So y is formed where the sums end. A training call also writes v and g, for bfloat16 x the upper 24 bits of the sums:
// dv and dg are rounded to bfloat16 afterwards, and a second rounding of that size before it makes the gradients 1.7
// times as far off as their own rounding alone, where one makes 1.4 (16 bits would save 3% of a call). k_dz forms dv |
// dg from them, one after the other along a row, so that dx is one product over 2 F, and dV and dG are one of 2 F rows.
// What act and act' of g take is hidden there behind the memory; where the sums end it adds to the matrix cores' time.
//
// Measured (N=8192, H=2048, F=5504, bfloat16, 1.11e12 operations, 1.08 to 1.12 ms over cards, calls in a row): the
// medians of a trace, which runs slower (1.25 ms of kernels), are v and g 0.44 (0.85 PFLOP/s: 1376 tiles are 5.4 rounds
// of the CUs, and 270 MB kept are written), k_dz 0.106 (5.1 TB/s), dx 0.325 (1.14 PFLOP/s), dV and dG 0.37 (0.99).
// Float32 (N=4095, H=512, F=1365) 0.29 to 0.32 ms: 92, 78 and 84 us the three (122 to 147 TFLOP/s). One row of H=4096,
// F=11000, bfloat16: 34 us, 5.3 TB/s.
//
// Narrow maps (both widths up to 64) have kernels of their own (ews_gated_narrow.h), and keep nothing.
//
// Few rows are bound by V and G's bytes: the forward's k_few reads them straight into the matrix instructions'
// registers, many loads on their way at once, without LDS.
//
// Float32 numbers are multiplied as three bfloat16 planes and six products (ews_tiles.h), float32's accuracy. Sums are
// float32, nothing is added with atomics: the same inputs give the same bits.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "ews_hip.h"
#include "ews_pack.h"
#include "ews_pick.h"
#include "ews_tiles.h"
#include "ews_tiles32.h"
#include "ews_vec.h"

namespace ews {
namespace gated {

using namespace ews::tiles;
using namespace ews::vec;

constexpr float kLog2e = 1.44269504088896340736f;

// s(g) and s(-g), either without the other's rounding. FINE: nor that of g log2(e), |g| 2^-24 of exp(-g), which
// bfloat16 results do not show.
template <bool FINE>
__device__ __forceinline__ void logistic(float g, float& p, float& q) {
  const float y = g * -kLog2e;
  float e = __builtin_amdgcn_exp2f(y);
  if (FINE) {
    constexpr float kLog2eRest = 1.925963033500e-8f, kLn2 = 0.693147180559945309f;
    const float rest = fmaf(g, -kLog2eRest, fmaf(g, -kLog2e, -y));
    e = fabsf(y) < 126.0f ? fmaf(e, rest * kLn2, e) : e;
  }
  p = __builtin_amdgcn_rcpf(1.0f + e);
  q = y > 126.0f ? 1.0f : e * p;  // e may be infinite
}

// act(g) and act'(g) for a call of type T.
template <typename T>
__device__ __forceinline__ void activate(int kind, float g, float& act, float& slope) {
  if (kind == EWS_GATED_RELU) {
    act = g <= 0.0f ? 0.0f : g;  // a NaN stays one
    slope = g > 0.0f ? 1.0f : 0.0f;
    return;
  }
  constexpr bool kFine = sizeof(T) == 4;
  float p, q;
  if (kind == EWS_GATED_GELU) {
    const float c = g > 30.0f ? 30.0f : g < -30.0f ? -30.0f : g;  // s is 0 or 1 long before; g^3 stays finite
    const float c2 = c * c;
    logistic<kFine>(1.5957691216057308f * c * fmaf(0.044715f, c2, 1.0f), p, q);
    act = g * p;
    slope = fmaf(c * p * q, 1.5957691216057308f * fmaf(0.134145f, c2, 1.0f), p);
    return;
  }
  logistic<kFine>(g, p, q);
  act = kind == EWS_GATED_SILU ? g * p : p;
  slope = kind == EWS_GATED_SILU ? fmaf(g * p, q, p) : p * q;
}

}  // namespace gated
}  // namespace ews

#include "ews_gated_narrow.h"

namespace ews {
namespace gated {

// ------------------------------------------------------------------------------------------------------ the operands
// V and G as a tile's first operand: of every wavefront's blocks of 32 rows the first half are V's, the others the same
// rows of G. Rows start as far apart in both.
struct Pair {
  Operand v;
  int64_t to_g;  // elements from V's numbers to G's
};

template <class T>
struct CopierPair {
  static constexpr int kCopies = T::kCopiesP, kHalf = T::TI / 2;
  static_assert(T::TI % 2 == 0 && T::kThreads / 8 <= 32 * kHalf, "a copy's rows are of one side");
  const uint16_t* base;
  int64_t plane, to_g;
  uint32_t offset[kCopies];
  static constexpr __device__ __forceinline__ bool gate(int c) {
    return c * (T::kThreads / 8) / 32 % T::TI >= kHalf;
  }
  __device__ __forceinline__ CopierPair(const Pair& o, int tile) : plane(o.v.plane), to_g(o.to_g) {
    const int first = tile < o.v.rows ? tile : o.v.rows - 1;
    base = o.v.p + first * o.v.ld;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const int idx = threadIdx.x + c * T::kThreads;
      const int row = idx >> 3, block = row >> 5;
      const int own = (block / T::TI * kHalf + block % kHalf) * 32 + (row & 31);
      offset[c] = (uint32_t)(first + own < o.v.rows ? own : o.v.rows - 1 - first) * (uint32_t)o.v.ld * 2 +
                  16 * place(row, idx & 7);
    }
  }
  __device__ __forceinline__ const uint16_t* at(int piece, int kb) const {
    return base + piece * plane + (int64_t)kb * 64;
  }
  __device__ __forceinline__ void copy(int c, const uint16_t* from, char* to) const {
    copy_piece(gate(c) ? from + to_g : from, offset[c], to + c * T::kThreads * 16);
  }
};

// V and G one after the other along k, turned: k blocks of V's rows, then as many of G's (or one operand's alone). Rows
// that a last block lacks meet zeros, and have to be zero for it: an infinity in their place would make NaN. Packed
// copies have such rows; of an operand that is read as it is that block lies in a copy, V's and behind it G's.
struct Chain {
  Operand v;
  int64_t to_g;
  int blocks, whole;      // of either; of those, blocks that have all rows
  const uint16_t* tail;   // the block after them; or null
  int64_t tail_ld;
};

template <class T>
struct CopierChain {
  static constexpr int kCopies = T::kCopiesP;
  Copier<true, T::I, T::kThreads> rows;
  const uint16_t* tail;
  int64_t to_g;
  int blocks, whole;
  uint32_t ld, tail_ld;
  __device__ __forceinline__ CopierChain(const Chain& o, int tile)
      : rows(o.v, tile), tail(o.tail), to_g(o.to_g), blocks(o.blocks), whole(o.whole), ld((uint32_t)o.v.ld),
        tail_ld((uint32_t)o.tail_ld) {}
  __device__ __forceinline__ void aim(uint32_t to) {
    rows.stride = to * 2;
    rows.aim_turned(63);
  }
  // Blocks are asked for in order.
  __device__ __forceinline__ const uint16_t* at(int piece, int kb) {
    const bool second = kb >= blocks;
    const int own = second ? kb - blocks : kb;
    if (own == whole) {
      aim(tail_ld);
      return tail + (second ? 64 * tail_ld : 0);
    }
    if (second && own == 0 && tail) aim(ld);  // V's last block lay elsewhere
    return rows.base + piece * rows.plane + (int64_t)own * 64 * ld + (second ? to_g : 0);
  }
  __device__ __forceinline__ void copy(int c, const uint16_t* from, char* to) const { rows.copy(c, from, to); }
};

}  // namespace gated

namespace tiles {
template <class T>
struct CopierOf<gated::Pair, T, false> {
  typedef gated::CopierPair<T> type;
};
template <class T>
struct CopierOf<gated::Chain, T, true> {
  typedef gated::CopierChain<T> type;
};
}  // namespace tiles

namespace gated {

// x, V and G laid out in one launch, those of them that have to be.
struct Packs {
  PackArgs each[3];
  uint32_t from[3];  // first workgroups
  uint32_t blocks;
  int count;
  void add(const PackArgs& a) {
    from[count] = blocks;
    each[count++] = a;
    blocks += (uint32_t)((a.dst_rows * (a.ld / 8) + 255) / 256);
  }
};

template <typename T>
__global__ __launch_bounds__(256) void k_packs(Packs a) {
#pragma unroll
  for (int k = 2; k >= 0; --k)
    if (k < a.count && blockIdx.x >= a.from[k])
      return pack_eight<T>(a.each[k], (int64_t)(blockIdx.x - a.from[k]) * 256 + threadIdx.x);
}

// ---------------------------------------------------------------------------------------------- what a forward keeps
// Numbers that a forward keeps: float32, or for bfloat16 the upper 24 bits of float32, rounded, as 16 and 8 of them in
// two arrays one after the other. (No NaN that bfloat16 inputs give has the low bits that rounding would carry out of.)
template <typename O>
struct Kept {
  static __device__ __forceinline__ void store(void* kept, int64_t, int64_t at, const Eight& e) {
    float* to = (float*)kept + at;
    __builtin_nontemporal_store(f32x4{e.x[0], e.x[1], e.x[2], e.x[3]}, reinterpret_cast<f32x4*>(to));
    __builtin_nontemporal_store(f32x4{e.x[4], e.x[5], e.x[6], e.x[7]}, reinterpret_cast<f32x4*>(to + 4));
  }
  static __device__ __forceinline__ void store_four(void* kept, int64_t, int64_t at, const float (&x)[4]) {
    *reinterpret_cast<f32x4*>((float*)kept + at) = f32x4{x[0], x[1], x[2], x[3]};
  }
  static __device__ __forceinline__ void load(const void* kept, int64_t, int64_t at, float (&x)[8]) {
    const float* from = (const float*)kept + at;
#pragma unroll
    for (int q = 0; q < 8; q += 4) {
      const f32x4 w = *reinterpret_cast<const f32x4*>(from + q);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[q + k] = w[k];
    }
  }
};
template <>
struct Kept<bf16> {
  static __device__ __forceinline__ void store(void* kept, int64_t count, int64_t at, const Eight& e) {
    u32x4 hi;
    u32x2 lo;
#pragma unroll
    for (int q = 0; q < 8; q += 2) {
      const uint32_t a = __float_as_uint(e.x[q]) + 0x80u, b = __float_as_uint(e.x[q + 1]) + 0x80u;
      hi[q / 2] = (a >> 16) | (b & 0xffff0000u);
      const uint32_t two = ((a >> 8) & 0xffu) | (b & 0xff00u);
      lo[q / 4] = q % 4 ? lo[q / 4] | two << 16 : two;
    }
    __builtin_nontemporal_store(hi, reinterpret_cast<u32x4*>((uint16_t*)kept + at));
    __builtin_nontemporal_store(lo, reinterpret_cast<u32x2*>((uint8_t*)kept + 2 * count + at));
  }
  static __device__ __forceinline__ void store_four(void* kept, int64_t count, int64_t at, const float (&x)[4]) {
    uint32_t n[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) n[q] = __float_as_uint(x[q]) + 0x80u;
    *reinterpret_cast<u32x2*>((uint16_t*)kept + at) =
        u32x2{(n[0] >> 16) | (n[1] & 0xffff0000u), (n[2] >> 16) | (n[3] & 0xffff0000u)};
    *reinterpret_cast<uint32_t*>((uint8_t*)kept + 2 * count + at) =
        ((n[0] >> 8) & 0xffu) | (n[1] & 0xff00u) | ((n[2] >> 8) & 0xffu) << 16 | (n[3] & 0xff00u) << 16;
  }
  static __device__ __forceinline__ void load(const void* kept, int64_t count, int64_t at, float (&x)[8]) {
    const u32x4 hi = *reinterpret_cast<const u32x4*>((const uint16_t*)kept + at);
    const u32x2 lo = *reinterpret_cast<const u32x2*>((const uint8_t*)kept + 2 * count + at);
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const uint32_t h = q % 2 ? hi[q / 2] & 0xffff0000u : hi[q / 2] << 16;
      x[q] = __uint_as_float(h | ((lo[q / 4] >> (8 * (q % 4))) & 0xffu) << 8);
    }
  }
};

// ------------------------------------------------------------------------------------------------------- the forward
struct ForwardArgs {
  Pair W;
  Operand X;
  int ti, tj, kblocks;
  int N, F;
  const void* bias;        // or null
  const void* gate_bias;
  int act;
  int wide;                // rows of out start at multiples of 16 bytes and hold whole eights
  void* out;               // (N, F)
  void* kept;              // (N, 2 ld): v | g (Kept)
  int64_t ld;              // F up to a multiple of 64
};

template <typename O>
__device__ __forceinline__ void store(O* to, const Eight& e) {
#pragma unroll
  for (int q = 0; q < 8; q += kWide<O>) {
    Pack<O, kWide<O>> p;
    p.set(e.x + q);
    p.store_past(to + q);
  }
}
template <typename O>
__device__ __forceinline__ void store(O* to, const One& e) {
  *to = narrow<O>(e.x);
}

// A wavefront's 32 rows of 16 TI results each, z[a] its blocks, through its own part of LDS: f(row of the 32, column,
// W).
template <class T, typename W, class F>
__device__ __forceinline__ void rows_of_half(char* lds, const f32x16 (&z)[T::TI / 2], F f) {
  constexpr int kCols = 16 * T::TI, kRow = kCols + 4, kEach = sizeof(W) / 4;
  const int lane = threadIdx.x & 63, r32 = lane & 31, half = lane >> 5;
  float* stage = reinterpret_cast<float*>(lds) + (threadIdx.x >> 6) * 32 * T::kRowWords;
#pragma unroll
  for (int a = 0; a < T::TI / 2; ++a)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<f32x4*>(stage + r32 * kRow + a * 32 + g * 8 + half * 4) =
          f32x4{z[a][4 * g], z[a][4 * g + 1], z[a][4 * g + 2], z[a][4 * g + 3]};
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
  constexpr int kLanes = kCols / kEach < 64 ? kCols / kEach : 64;
#pragma unroll
  for (int it = 0; it < 32 * kCols / kEach / 64; ++it) {
    const int row = it * (64 / kLanes) + lane / kLanes, col = lane % kLanes * kEach;
    W w;
    if constexpr (kEach == 8) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(stage + row * kRow + col);
      const f32x4 hi = *reinterpret_cast<const f32x4*>(stage + row * kRow + col + 4);
      w = Eight{{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
    } else {
      w = One{stage[row * kRow + col]};
    }
    f(row, col, w);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
}

template <typename B>
__device__ __forceinline__ float bias_at(const void* bias, int i) {
  return bias ? widen(((const B*)bias)[i]) : 0.0f;
}

// KEEP: for a backward.
template <class T, int PAIRS, typename O, bool KEEP>
__global__ __launch_bounds__(T::kThreads, T::kWaves) void k_forward(ForwardArgs a) {
  extern __shared__ char lds[];
  int it, jt;
  tile_of(blockIdx.x, a.ti, a.tj, it, jt);
  const int i0 = it * (T::I / 2), j0 = jt * T::J;
  float* bias = reinterpret_cast<float*>(lds + lds_bytes<T, PAIRS>(a.kblocks));  // V's, then G's
  for (int t = threadIdx.x; t < T::I; t += T::kThreads) {
    const int i = i0 + t % (T::I / 2), in = i < a.F ? i : a.F - 1;
    bias[t] = bias_at<O>(t < T::I / 2 ? a.bias : a.gate_bias, in);
  }
  f32x16 acc[T::TI][T::TJ];
  product<T, PAIRS, false, false>(a.W, a.X, i0, j0, 0, a.kblocks, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave % T::WI, wj = wave / T::WI, half = lane >> 5;
  constexpr int kHalf = T::TI / 2;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) {
    f32x16 y[kHalf], v[kHalf], g[kHalf];
#pragma unroll
    for (int t = 0; t < kHalf; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int i = (wi * kHalf + t) * 32 + 8 * (r / 4) + 4 * half + r % 4;
        v[t][r] = acc[t][b][r] + bias[i];
        g[t][r] = acc[t + kHalf][b][r] + bias[T::I / 2 + i];
        float act, slope;
        activate<O>(a.act, g[t][r], act, slope);
        y[t][r] = v[t][r] * act;
      }
    const int row0 = j0 + (wj * T::TJ + b) * 32, col0 = i0 + wi * kHalf * 32;
    auto out = [&](auto each) {
      using W = decltype(each);
      rows_of_half<T, W>(lds, y, [&](int row, int col, const W& e) {
        if (row0 + row < a.N && col0 + col < a.F)
          store<O>((O*)a.out + (int64_t)(row0 + row) * a.F + col0 + col, e);
      });
    };
    if (a.wide)
      out(Eight{});
    else
      out(One{});
    if (!KEEP) continue;
    // whole eights up to ld: what lies past F is not read
    rows_of_half<T, Eight>(lds, v, [&](int row, int col, const Eight& e) {
      if (row0 + row < a.N && col0 + col < a.ld)
        Kept<O>::store(a.kept, 2 * a.ld * a.N, (int64_t)(row0 + row) * 2 * a.ld + col0 + col, e);
    });
    rows_of_half<T, Eight>(lds, g, [&](int row, int col, const Eight& e) {
      if (row0 + row < a.N && col0 + col < a.ld)
        Kept<O>::store(a.kept, 2 * a.ld * a.N, (int64_t)(row0 + row) * 2 * a.ld + a.ld + col0 + col, e);
    });
  }
}

// ------------------------------------------------------------------------------------------------------- few rows
struct FewArgs {
  const void* x;
  const void* v;
  const void* g;
  int64_t xs, ws, gs;
  int N, H, F;
  const void* bias;
  const void* gate_bias;
  int act;
  void* out;
  void* kept;              // as ForwardArgs'; or null
  int64_t ld;
};

constexpr int kFewWaves = 4;

// A lane's eight numbers of 32 k of a row from column k on, zero past the row's end: bfloat16 k + 8 q .. 8 q + 7 for q
// its fourth of the wavefront, float32 k + 4 q .. 4 q + 3 and 16 further on. Either way a load's lanes read 64 bytes of
// a row; a product's k may be in any order that its operands share.
// kAligned: rows of whole eights at multiples of 16 bytes. kInside: all 32 k lie in the row, at any address (19 rows by
// H=3761, F=6047, bfloat16: 64 us, number by number 126). kAny: neither is known.
enum Rows16 { kAny, kAligned, kInside };
template <typename T, Rows16 ROWS>
__device__ __forceinline__ void few_eight(const T* row, int k, int H, T (&x)[8]) {
  constexpr int kLoads = sizeof(T) == 4 ? 2 : 1, kEach = 8 / kLoads;
  const int q = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int h = 0; h < kLoads; ++h) {
    const int at = k + 16 * h + kEach * q;
    if (ROWS == kAligned) {
      *reinterpret_cast<u32x4*>(x + kEach * h) =
          at < H ? *reinterpret_cast<const u32x4*>(row + at) : u32x4{0, 0, 0, 0};
    } else if (ROWS == kInside || k + 32 <= H) {
      __builtin_memcpy(x + kEach * h, row + at, 16);
    } else {
#pragma unroll
      for (int e = 0; e < kEach; ++e) x[kEach * h + e] = at + e < H ? row[at + e] : narrow<T>(0.0f);
    }
  }
}

template <typename T, bool CAREFUL>
__device__ __forceinline__ void few_fragments(const T (&x)[8], bf16x8 (&f)[kPlanes<T>]) {
  if constexpr (sizeof(T) == 4)
    cut<CAREFUL>(x, f);
  else
    fragments<T>(x, f);
}

// One wavefront's part of the sums over k: of 16 of V's and G's rows and 16 COLS of x's.
template <typename T, int COLS, bool WIDE, bool CAREFUL>
__device__ __forceinline__ void few_sums(const FewArgs& a, f32x4v (&acc)[2][COLS]) {
  constexpr int kAhead = sizeof(T) == 4 ? 4 : 8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int f = blockIdx.x * 16 + (lane & 15), own = f < a.F ? f : a.F - 1;
  const T* v = (const T*)a.v + own * a.ws;
  const T* g = (const T*)a.g + own * a.gs;
#pragma unroll
  for (int c = 0; c < COLS; ++c) acc[0][c] = acc[1][c] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  auto stretch = [&](auto rows, int k0) {
    constexpr Rows16 kRows = decltype(rows)::value;
    T wv[kAhead][8], wg[kAhead][8];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      few_eight<T, kRows>(v, k0 + 32 * s, a.H, wv[s]);
      few_eight<T, kRows>(g, k0 + 32 * s, a.H, wg[s]);
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      bf16x8 fv[kPlanes<T>], fg[kPlanes<T>];
      few_fragments<T, CAREFUL>(wv[s], fv);
      few_fragments<T, CAREFUL>(wg[s], fg);
#pragma unroll
      for (int c = 0; c < COLS; ++c) {
        const int n = c * 16 + (lane & 15) < a.N ? c * 16 + (lane & 15) : a.N - 1;
        T x[8];
        bf16x8 fx[kPlanes<T>];
        few_eight<T, kRows>((const T*)a.x + n * a.xs, k0 + 32 * s, a.H, x);
        few_fragments<T, CAREFUL>(x, fx);
        mac(fv, fx, acc[0][c]);
        mac(fg, fx, acc[1][c]);
      }
    }
  };
  for (int k0 = wave * 32 * kAhead; k0 < a.H; k0 += kFewWaves * 32 * kAhead) {
    if constexpr (WIDE)
      stretch(std::integral_constant<Rows16, kAligned>{}, k0);
    else if (k0 + 32 * kAhead <= a.H)
      stretch(std::integral_constant<Rows16, kInside>{}, k0);
    else
      stretch(std::integral_constant<Rows16, kAny>{}, k0);
  }
}

// 16 outputs of up to 16 COLS rows a workgroup; its wavefronts take every fourth stretch of k and are joined in LDS.
// v_mfma_f32_16x16x32_bf16: a lane gets results column l % 16 (x's row), rows 4 (l / 16) + 0..3 (outputs). One bfloat16
// row through H=4096, F=11000 34 us (5.3 TB/s), float32 88 (4.1); 32 outputs a workgroup 46 and 106.
template <typename T, int COLS, bool WIDE>
__global__ __launch_bounds__(64 * kFewWaves) void k_few(FewArgs a) {
  __shared__ f32x4v part[kFewWaves][2 * COLS][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f32x4v acc[2][COLS];
  few_sums<T, COLS, WIDE, false>(a, acc);
  if (sizeof(T) == 4) {
    // infinities need care (ews_tiles32.h): looked for in the sums, not number by number, which took 124 us for 90
    bool bad = false;
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int c = 0; c < COLS; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) bad |= __builtin_isnan(acc[side][c][r]);
    if (__any(bad)) few_sums<T, COLS, WIDE, true>(a, acc);
  }
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int c = 0; c < COLS; ++c) part[wave][side * COLS + c][lane] = acc[side][c];
  __syncthreads();
  for (int c = wave; c < COLS; c += kFewWaves) {
    f32x4v sv = part[0][c][lane], sg = part[0][COLS + c][lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) {
      sv += part[w][c][lane];
      sg += part[w][COLS + c][lane];
    }
    const int n = c * 16 + (lane & 15), f = blockIdx.x * 16 + (lane >> 4) * 4;
    if (n >= a.N) continue;
    float v[4], g[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int in = f + r < a.F ? f + r : a.F - 1;
      v[r] = sv[r] + bias_at<T>(a.bias, in);
      g[r] = sg[r] + bias_at<T>(a.gate_bias, in);
      float act, slope;
      activate<T>(a.act, g[r], act, slope);
      if (f + r < a.F) ((T*)a.out)[(int64_t)n * a.F + f + r] = narrow<T>(v[r] * act);
    }
    if (a.kept && f < a.F) {
      Kept<T>::store_four(a.kept, 2 * a.ld * a.N, (int64_t)n * 2 * a.ld + f, v);
      Kept<T>::store_four(a.kept, 2 * a.ld * a.N, (int64_t)n * 2 * a.ld + a.ld + f, g);
    }
  }
}

// x's gradient of few float32 rows: V and G are read as they are, a lane four columns of eight rows, the eight k of
// four operands. One row by H=1066, F=14344 40 us, by the tiles 49 and 67 to pack the weights for them; 48 rows by
// H=1024, F=4096 26 (22 and 12). bfloat16, with eight columns a lane, turns too much in registers: 32 rows by H=4096,
// F=11000 78 (by the tiles 33, nothing to pack).
struct FewDxArgs {
  const uint16_t* dz;      // as DzArgs'
  int64_t plane, ld;
  const float* v;
  const float* g;
  int64_t ws, gs;
  int N, H, F;
  int blocks, per;         // of 32 rows of V and then of G; of a workgroup
  float* part;             // (workgroups along y, N, H)
};

constexpr int kDxCols = 4;

// One wavefront's part of the sums over f, of 16 ROWS rows and 64 columns.
template <int ROWS, bool CAREFUL>
__device__ __forceinline__ void few_dx_sums(const FewDxArgs& a, int b0, int b1, f32x4v (&acc)[ROWS][kDxCols]) {
  constexpr int NP = kPlanes<float>, kAhead = 2;
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int h = ((int)blockIdx.x * 16 + r16) * kDxCols, sides = a.blocks / 2;
#pragma unroll
  for (int j = 0; j < ROWS; ++j)
#pragma unroll
    for (int c = 0; c < kDxCols; ++c) acc[j][c] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
  float w[kAhead][8][kDxCols];
  auto load = [&](int s, int b) {
    const bool gate = b >= sides;
    const float* from = gate ? a.g : a.v;
    const int64_t stride = gate ? a.gs : a.ws;
    const int f = (gate ? b - sides : b) * 32 + 8 * q;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* row = from + (f + i < a.F ? f + i : a.F - 1) * stride;  // those past F meet zeros
      if (h + kDxCols <= a.H) {
        __builtin_memcpy(w[s][i], row + h, 16);
      } else {
#pragma unroll
        for (int c = 0; c < kDxCols; ++c) w[s][i][c] = h + c < a.H ? row[h + c] : 0.0f;
      }
      if (CAREFUL && f + i >= a.F)  // zero times an infinity is not
#pragma unroll
        for (int c = 0; c < kDxCols; ++c) w[s][i][c] = 0.0f;
    }
  };
  for (int b = b0; b < b1; b += kAhead) {
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
      if (b + s < b1) load(s, b + s);
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      if (b + s >= b1) break;
      const bool gate = b + s >= sides;
      const int64_t at = (gate ? a.ld : 0) + (gate ? b + s - sides : b + s) * 32 + 8 * q;
      bf16x8 z[ROWS][NP];
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
#pragma unroll
        for (int k = 0; k < NP; ++k)
          z[j][k] = *reinterpret_cast<const bf16x8*>(a.dz + k * a.plane + (int64_t)(j * 16 + r16) * 2 * a.ld + at);
#pragma unroll
      for (int c = 0; c < kDxCols; ++c) {
        float x[8];
        bf16x8 fw[NP];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = w[s][i][c];
        cut<CAREFUL>(x, fw);
#pragma unroll
        for (int j = 0; j < ROWS; ++j) mac(z[j], fw, acc[j][c]);
      }
    }
  }
}

template <int ROWS>
__global__ __launch_bounds__(64 * kFewWaves) void k_few_dx(FewDxArgs a) {
  __shared__ f32x4v part[kFewWaves - 1][ROWS * kDxCols][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int first = blockIdx.y * a.per, last = first + a.per < a.blocks ? first + a.per : a.blocks;
  const int each = (a.per + kFewWaves - 1) / kFewWaves;
  const int b0 = first + wave * each < last ? first + wave * each : last, b1 = b0 + each < last ? b0 + each : last;
  f32x4v acc[ROWS][kDxCols];
  few_dx_sums<ROWS, false>(a, b0, b1, acc);
  bool bad = false;  // as in k_few
#pragma unroll
  for (int j = 0; j < ROWS; ++j)
#pragma unroll
    for (int c = 0; c < kDxCols; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) bad |= __builtin_isnan(acc[j][c][r]);
  if (__any(bad)) few_dx_sums<ROWS, true>(a, b0, b1, acc);
  if (wave)
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
#pragma unroll
      for (int c = 0; c < kDxCols; ++c) part[wave - 1][j * kDxCols + c][lane] = acc[j][c];
  __syncthreads();
  if (wave) return;
  const int h = ((int)blockIdx.x * 16 + (lane & 15)) * kDxCols;
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
#pragma unroll
    for (int c = 0; c < kDxCols; ++c)
#pragma unroll
      for (int w = 0; w < kFewWaves - 1; ++w) acc[j][c] += part[w][j * kDxCols + c][lane];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = j * 16 + (lane >> 4) * 4 + r;
      if (n >= a.N) continue;
      float* to = a.part + ((int64_t)blockIdx.y * a.N + n) * a.H + h;
      float x[kDxCols];
#pragma unroll
      for (int c = 0; c < kDxCols; ++c) x[c] = acc[j][c][r];
      if (h + kDxCols <= a.H) {
        __builtin_memcpy(to, x, sizeof(x));
      } else {
#pragma unroll
        for (int c = 0; c < kDxCols; ++c)
          if (h + c < a.H) to[c] = x[c];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ dv | dg
struct DzArgs {
  const void* dy;          // (N, F)
  const void* kept;        // (N, 2 ld): v | g
  int act;
  int N, F, padded;        // rows; and zeros up to this one
  int64_t ld;
  int wide;                // rows of dy start at multiples of 16 bytes and hold whole eights
  uint16_t* dz;            // planes (padded, 2 ld), zero past F
  int64_t plane;
  float* sums;             // (workgroups along y, 2 ld) over the rows; or null
  int each, parts;         // rows of a workgroup; workgroups along y, but for those that lay out
  Packs tails;             // the last blocks of operands that are read as they are (bfloat16)
};

// A thread eight columns of every fourth of its workgroup's rows. SUMS: for the biases (the registers of which cost
// waves: 8192 rows by F=5504 in bfloat16 127 us with them, 105 without).
template <typename T, bool SUMS>
__global__ __launch_bounds__(256) void k_dz(DzArgs a) {
  constexpr int NP = kPlanes<T>;
  if (NP == 1 && blockIdx.y >= a.parts) {
    const uint32_t block = (blockIdx.y - a.parts) * gridDim.x + blockIdx.x;
#pragma unroll
    for (int k = 2; k >= 0; --k)
      if (k < a.tails.count && block >= a.tails.from[k])
        return pack_eight<T>(a.tails.each[k], (int64_t)(block - a.tails.from[k]) * 256 + threadIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int f = (blockIdx.x * 64 + lane) * 8;
  const int n = f >= a.F ? 0 : a.F - f < 8 ? a.F - f : 8;
  const int r1 = (int)(blockIdx.y + 1) * a.each < a.padded ? (int)(blockIdx.y + 1) * a.each : a.padded;
  float sums[2][8];
#pragma unroll
  for (int q = 0; q < 8; ++q) sums[0][q] = sums[1][q] = 0.0f;
  for (int row = blockIdx.y * a.each + wave; row < r1 && f < a.ld; row += 4) {
    float u[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) u[q] = 0.0f;
    const int live = row < a.N ? n : 0;
    const T* dy = (const T*)a.dy + (int64_t)row * a.F + f;
    if (a.wide && live) {
#pragma unroll
      for (int q = 0; q < 8; q += kWide<T>) {
        Pack<T, kWide<T>> p;
        p.load(dy + q);
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) u[q + e] = p.get(e);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < live) u[q] = widen(dy[q]);
    }
    float both[2][8];
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int q = 0; q < 8; ++q) both[side][q] = 0.0f;
    if (live) {
      Kept<T>::load(a.kept, 2 * a.ld * a.N, (int64_t)row * 2 * a.ld + f, both[0]);
      Kept<T>::load(a.kept, 2 * a.ld * a.N, (int64_t)row * 2 * a.ld + a.ld + f, both[1]);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        float act, slope;
        activate<T>(a.act, both[1][q], act, slope);
        both[1][q] = q < live ? u[q] * (both[0][q] * slope) : 0.0f;
        both[0][q] = q < live ? u[q] * act : 0.0f;
      }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      const float(&z)[8] = both[side];
      uint16_t p[8][NP];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        if (SUMS) sums[side][q] += z[q];
        planes(narrow<T>(z[q]), p[q]);
      }
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = (uint32_t)p[2 * q][k] | ((uint32_t)p[2 * q + 1][k] << 16);
        *reinterpret_cast<u32x4*>(a.dz + k * a.plane + ((int64_t)row * 2 + side) * a.ld + f) = w;
      }
    }
  }
  if (!SUMS) return;
  __shared__ float part[4][2][64][9];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int q = 0; q < 8; ++q) part[wave][side][lane][q] = sums[side][q];
  __syncthreads();
  for (int t = threadIdx.x; t < 1024; t += 256) {
    const int side = t >> 9, c = t & 511, col = blockIdx.x * 512 + c;
    if (col >= a.ld) continue;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += part[w][side][c >> 3][c & 7];
    a.sums[((int64_t)blockIdx.y * 2 + side) * a.ld + col] = s;
  }
}

// The biases' gradients: 64 columns a workgroup, its sixteen wavefronts a contiguous part of k_dz's sums each.
template <typename T>
__global__ __launch_bounds__(1024) void k_dbias(const float* sums, int parts, int64_t ld, int F, T* dv, T* dg) {
  __shared__ float joined[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, f = blockIdx.x * 64 + lane, side = blockIdx.y;
  const int each = (parts + 15) / 16, p1 = (wave + 1) * each < parts ? (wave + 1) * each : parts;
  T* out = side ? dg : dv;
  float s = 0.0f;
  if (f < F) {
#pragma unroll 8
    for (int p = wave * each; p < p1; ++p) s += sums[((int64_t)p * 2 + side) * ld + f];
  }
  joined[wave][lane] = s;
  __syncthreads();
  if (wave || f >= F || !out) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += joined[w][lane];
  out[f] = narrow<T>(s);
}

// ------------------------------------------------------------------------------------------------------ the gradients
struct GradArgs {
  Chain W;                 // dx: k along 2 F
  Chain X;                 // dV | dG: k along the rows
  Operand Z;               // dv | dg
  int ti, tj, splits, kblocks, per;
  int whole, pieces;       // tiles done by a workgroup each; workgroups that share each of the others
  int I, J;                // results along H; rows of dx, or 2 ld of dV | dG
  int F, ld;               // dV | dG: those of the J that are V's and G's
  float* part;             // (splits, J, I) where splits > 1; or the shared tiles' pieces, (tiles, pieces, tile)
  void* out;               // dx or dV
  void* gate_out;          // dG
  int wide;                // results' rows start at multiples of 16 bytes and hold whole eights
};

// Where result row j belongs; null: nowhere.
template <bool ROWS, typename O>
__device__ __forceinline__ O* result_row(const GradArgs& a, int j) {
  if (!ROWS) return j < a.J ? (O*)a.out + (int64_t)j * a.I : nullptr;
  const bool gate = j >= a.ld;
  const int f = gate ? j - a.ld : j;
  O* out = (O*)(gate ? a.gate_out : a.out);
  return f < a.F && out ? out + (int64_t)f * a.I : nullptr;
}

__device__ __forceinline__ void keep(float* to, const Eight& e) {
  *reinterpret_cast<f32x4*>(to) = f32x4{e.x[0], e.x[1], e.x[2], e.x[3]};
  *reinterpret_cast<f32x4*>(to + 4) = f32x4{e.x[4], e.x[5], e.x[6], e.x[7]};
}
__device__ __forceinline__ void keep(float* to, const One& e) { *to = e.x; }

// ROWS: dV | dG; else dx.
template <class T, int PAIRS, bool ROWS, typename O>
__global__ __launch_bounds__(T::kThreads, T::kWaves) void k_grad(GradArgs a) {
  extern __shared__ char lds[];
  const bool shared = (int)blockIdx.x >= a.whole;
  const int other = blockIdx.x - a.whole;
  const int split = shared ? other % a.pieces : blockIdx.y;
  int it, jt;
  tile_of(shared ? a.whole + other / a.pieces : blockIdx.x, a.ti, a.tj, it, jt);
  const int i0 = it * T::I, j0 = jt * T::J;
  const int per = shared ? (a.kblocks + a.pieces - 1) / a.pieces : a.per;
  const int kb0 = split * per, kb1 = kb0 + per < a.kblocks ? kb0 + per : a.kblocks;
  f32x16 acc[T::TI][T::TJ];
  if constexpr (ROWS)
    product<T, PAIRS, true, true>(a.X, a.Z, i0, j0, kb0, kb1, lds, acc);
  else
    product<T, PAIRS, true, false>(a.W, a.Z, i0, j0, kb0, kb1, lds, acc);
  auto rows = [&](auto each) {
    using W = decltype(each);
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
      rows_of<T, W>(lds, acc, b, [&](int jrow, int icol, const W& e) {
        if (shared) return keep(a.part + (int64_t)other * T::I * T::J + jrow * T::I + icol, e);
        const int j = j0 + jrow, i = i0 + icol;
        if (j >= a.J || i >= a.I) return;
        if (a.splits > 1) return keep(a.part + ((int64_t)split * a.J + j) * a.I + i, e);
        O* to = result_row<ROWS, O>(a, j);
        if (to) store<O>(to + i, e);
      });
  };
  if (a.wide)
    rows(Eight{});
  else
    rows(One{});
}

// The shared tiles' pieces added in order: 1024 results a workgroup.
template <class T, bool ROWS, typename O, typename W>
__global__ __launch_bounds__(1024 / (sizeof(W) / 4)) void k_shared(GradArgs a) {
  constexpr int kEach = sizeof(W) / 4, kOf = T::I * T::J / 1024;
  const int t = blockIdx.x / kOf, at = (blockIdx.x % kOf) * 1024 + threadIdx.x * kEach;
  int it, jt;
  tile_of(a.whole + t, a.ti, a.tj, it, jt);
  const int j = jt * T::J + at / T::I, i = it * T::I + at % T::I;
  if (j >= a.J || i >= a.I) return;
  O* to = result_row<ROWS, O>(a, j);
  if (!to) return;
  float x[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) x[q] = 0.0f;
  for (int s = 0; s < a.pieces; ++s) {
    const float* from = a.part + ((int64_t)t * a.pieces + s) * T::I * T::J + at;
#pragma unroll
    for (int q = 0; q < kEach; ++q) x[q] += from[q];
  }
  W w;
  __builtin_memcpy(&w, x, sizeof(w));
  store<O>(to + i, w);
}

// The splits' results added in order, by GROUPS groups of a workgroup's threads a contiguous part of them each; a
// thread takes one result (W: One) or eight.
template <bool ROWS, typename O, typename W, int GROUPS>
__global__ __launch_bounds__(256) void k_join(GradArgs a) {
  constexpr int kEach = sizeof(W) / 4, kThreads = 256 / GROUPS;
  __shared__ float joined[GROUPS][kThreads][kEach];
  const int group = threadIdx.x / kThreads, lane = threadIdx.x % kThreads;
  const int64_t n = (int64_t)a.J * a.I, at = ((int64_t)blockIdx.x * kThreads + lane) * kEach;
  const int per = (a.splits + GROUPS - 1) / GROUPS, s1 = (group + 1) * per < a.splits ? (group + 1) * per : a.splits;
  float x[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) x[q] = 0.0f;
  if (at < n) {
#pragma unroll 4
    for (int s = group * per; s < s1; ++s) {
      const float* from = a.part + s * n + at;
      if constexpr (kEach == 1) {
        x[0] += from[0];
      } else {
#pragma unroll
        for (int q = 0; q < kEach; q += 4) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(from + q);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[q + e] += w[e];
        }
      }
    }
  }
  if (GROUPS > 1) {
#pragma unroll
    for (int q = 0; q < kEach; ++q) joined[group][lane][q] = x[q];
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g)
#pragma unroll
      for (int q = 0; q < kEach; ++q) x[q] += joined[g][lane][q];
  }
  if (at >= n) return;
  const int j = (int)(at / a.I);
  O* to = result_row<ROWS, O>(a, j);
  W w;
  __builtin_memcpy(&w, x, sizeof(w));
  if (to) store<O>(to + (at - (int64_t)j * a.I), w);
}

}  // namespace gated
}  // namespace ews

namespace {

using namespace ews::gated;
namespace tiles = ews::tiles;
using tiles::ceil_div;
using tiles::Kind;
using tiles::Operand;
using tiles::Product;
using ews::vec::bf16;

// Rows up to which V and G go straight into registers (the measured: of a forward): 32 of H=4096, F=11000 48 us in
// bfloat16 (by the tiles 51), 33 rows 55 (48); float32, whose tiles need planes packed first, 64 rows 180 (420).
constexpr int kFewRows = 32, kFewRows32 = 64;
// Splits that one thread adds; more are added by eight groups of threads.
constexpr int kFewSplits = 8;

// A product whose tiles of the last, mostly empty round of workgroups are shared out along k.
struct GProduct : Product {
  int whole, pieces;
  size_t part_bytes(int64_t I, int64_t J) const {
    const int64_t others = (int64_t)ti * tj - whole;
    if (others) return (size_t)(others * pieces * tile_i * tile_j * 4);
    return splits > 1 ? (size_t)(splits * I * J * 4) : 0;
  }
};

// 256 large tiles are a round, one a CU. The last round's tiles are shared by two to four workgroups each where that
// shortens it by a quarter at least: 11008 x 2048 results (344 tiles) over 8192 rows 415 us, shared 361.
GProduct share(const Product& of) {
  GProduct p;
  static_cast<Product&>(p) = of;
  const int n = p.ti * p.tj, others = n % 256;
  p.whole = n;
  p.pieces = 1;
  if (p.kind != tiles::kLarge || p.splits > 1 || n < 256 || others == 0 || p.kblocks < 64) return p;
  double best = 0.75;  // of a round
  for (int z = 2; z <= 4; ++z) {
    const double took = (double)ceil_div(others * z, 256) / z;
    if (took >= best) continue;
    best = took;
    p.whole = n - others;
    p.pieces = z;
  }
  return p;
}

struct GPlan {
  int N, H, F, np;
  int64_t Hp, ld, Np;
  bool pack_x, pack_w, few, few_dx, narrow;
  Product forward;
  GProduct dx, dw;
  int dz_rows, dz_parts, narrow_groups;
  int dx_blocks, dx_per, dx_parts;  // of few_dx
  bool tail_x, tail_w;     // of a backward
  size_t xp, wp, dz, sums, part, total;
};

int narrow_pad(int n) { return n <= 32 ? 32 : 64; }

bool direct(const void* p, int64_t stride, int H) {
  return H % 64 == 0 && stride % 8 == 0 && stride <= 1 << 22 && (uintptr_t)p % 16 == 0;
}

int gated_plan(const ews_gated_desc* s, const void* x, const void* v, const void* g, bool back, bool keep, GPlan& p) {
  if (!s) return EWS_ERR_NULL;
  if (s->dtype != EWS_DTYPE_F32 && s->dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->activation < 0 || s->activation > EWS_GATED_RELU) return EWS_ERR_OPTION;
  if (s->rows < 1 || s->width < 1 || s->features < 1 || s->rows > 1 << 24 || s->width > 1 << 16 ||
      s->features > 1 << 20)
    return EWS_ERR_SHAPE;
  if (s->x_stride < s->width || s->weight_stride < s->width || s->gate_stride < s->width) return EWS_ERR_SHAPE;
  p.N = s->rows;
  p.H = s->width;
  p.F = s->features;
  p.np = s->dtype == EWS_DTYPE_F32 ? 3 : 1;
  p.Hp = (int64_t)ceil_div(p.H, 64) * 64;
  p.ld = (int64_t)ceil_div(p.F, 64) * 64;
  p.Np = (int64_t)ceil_div(p.N, 64) * 64;
  // a launch has fewer than 2^32 threads, one for eight numbers; dv | dg's rows lie within the tiles' offsets
  if (p.Np * p.Hp > (int64_t)1 << 33 || p.F * p.Hp > (int64_t)1 << 33 || p.Np * p.ld > (int64_t)1 << 34)
    return EWS_ERR_SHAPE;
  p.few = p.N <= (p.np == 3 ? kFewRows32 : kFewRows);
  p.narrow = p.H <= kNarrowWidth && p.F <= kNarrowWidth && (back || keep || !p.few);  // and keeps nothing
  if (p.narrow) {
    // 32 rows a wavefront and turn; as many workgroups as are on the CUs at a time
    const int groups = ceil_div(p.N, 32 * (p.np == 3 ? narrow_waves<float>(p.H, p.F) : narrow_waves<bf16>(p.H, p.F)));
    p.narrow_groups = groups < 512 ? groups : 512;
    p.part = 0;
    p.total = back ? (size_t)p.narrow_groups * 2 * narrow_pad(p.F) * (narrow_pad(p.H) + 1) * 4 : 0;
    return EWS_OK;
  }
  p.pack_x = p.np == 3 || !direct(x, s->x_stride, p.H);
  p.few_dx = back && p.few && p.np == 3;
  p.pack_w = !p.few_dx && (p.np == 3 || !direct(v, s->weight_stride, p.H) || !direct(g, s->gate_stride, p.H) ||
             s->weight_stride != s->gate_stride || ((uintptr_t)g - (uintptr_t)v) % 2);
  const int pairs = p.np == 3 ? tiles::kPairs : 1;
  p.forward = tiles::pick(2 * p.ld, p.N, (int)(p.Hp / 64), pairs, false, false);
  p.dx = share(tiles::pick(p.H, p.N, (int)(2 * p.ld / 64), pairs, true, false));
  p.dw = share(tiles::pick(p.H, 2 * p.ld, (int)(p.Np / 64), pairs, true, false));
  size_t off = 0;
  auto take = [&off](size_t bytes) {
    const size_t at = off;
    off += tiles::al256x(bytes);
    return at;
  };
  if (back || !p.few) {
    // whole blocks of rows, zeros past the last; or of operands that a backward reads as they are the last block alone
    p.tail_x = back && !p.pack_x && p.N % 64;
    p.tail_w = back && !p.pack_w && !p.few_dx && p.F % 64;
    p.xp = take(p.pack_x ? (size_t)(p.Np * p.Hp * p.np * 2) : p.tail_x ? (size_t)(64 * p.Hp * 2) : 0);
    p.wp = take(p.pack_w ? (size_t)(2 * p.ld * p.Hp * p.np * 2) : p.tail_w ? (size_t)(128 * p.Hp * 2) : 0);
  }
  if (back) {
    p.dz = take((size_t)(p.Np * 2 * p.ld * p.np * 2));
    // 64 rows a workgroup (the biases' partial sums stay small), fewer where that leaves CUs without one
    p.dz_rows = 64;
    while (p.dz_rows > 4 && (int64_t)ceil_div(p.Np, p.dz_rows) * ceil_div(p.ld, 512) < 1024) p.dz_rows /= 2;
    // a grid's second side, on which up to 6144 workgroups lay out tails
    while (ceil_div(p.Np, p.dz_rows) > 59000) p.dz_rows *= 2;
    p.dz_parts = ceil_div(p.Np, p.dz_rows);
    p.sums = take((size_t)p.dz_parts * 2 * p.ld * 4);
    // four workgroups a CU, of eight blocks at least
    const int wide = ceil_div(p.H, 16 * kDxCols);
    p.dx_blocks = 2 * ceil_div(p.F, 32);
    p.dx_parts = ceil_div(1024, wide);
    if (p.dx_parts > ceil_div(p.dx_blocks, 8)) p.dx_parts = ceil_div(p.dx_blocks, 8);
    p.dx_per = ceil_div(p.dx_blocks, p.dx_parts);
    p.dx_parts = ceil_div(p.dx_blocks, p.dx_per);
    const size_t dx = p.few_dx ? (size_t)p.dx_parts * p.N * p.H * 4 : p.dx.part_bytes(p.H, p.N);
    const size_t dw = p.dw.part_bytes(p.H, 2 * p.ld);
    p.part = take(dx > dw ? dx : dw);
  }
  p.total = off;
  return EWS_OK;
}

#define GATED_CHECK()                                            \
  do {                                                           \
    if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH; \
  } while (0)

struct GCall {
  const ews_gated_desc* s;
  GPlan p;
  char* w;
  hipStream_t st;
  Chain x;
  Chain weights;
  Packs tails;
};

// Rows of an operand from `first` on, as far as they go, laid out as dst_rows with zeros behind them.
tiles::PackArgs pack_args(const GPlan& p, const void* src, int64_t stride, int first, int rows, int dst_rows,
                          uint16_t* dst, int64_t plane) {
  tiles::PackArgs a{};
  a.src = (const char*)src + first * stride * (p.np == 3 ? 4 : 2);
  a.stride = stride;
  a.rows = rows - first;
  a.cols = p.H;
  a.dst = dst;
  a.ld = p.Hp;
  a.plane = plane;
  a.dst_rows = dst_rows;
  a.wide = tiles::rows_wide(src, stride, p.np == 3);
  return a;
}

// An operand, or V and G (g; else null), as the tiles read them. packed: copies of all rows (a), else tail: of the
// last, incomplete block (tails). to: where those go; want: whether the call reads them.
Chain lay_out(Packs& a, Packs& tails, const GPlan& p, const void* v, int64_t v_stride, const void* g, int64_t g_stride,
              int rows, bool packed, bool tail, char* to, bool want) {
  const int padded = ceil_div(rows, 64) * 64, sides = g ? 2 : 1;
  Chain c{};
  c.blocks = padded / 64;
  c.whole = c.blocks;
  if (packed) {
    c.v = Operand{(const uint16_t*)to, p.Hp, sides * padded * p.Hp, padded, (int)p.Hp};
    c.to_g = padded * p.Hp;
  } else {
    c.v = Operand{(const uint16_t*)v, v_stride, 0, rows, (int)p.Hp};
    c.to_g = g ? ((intptr_t)g - (intptr_t)v) / 2 : 0;
    if (!tail) return c;
    c.whole = rows / 64;
    c.tail = (const uint16_t*)to;
    c.tail_ld = p.Hp;
  }
  if (!want) return c;
  const int first = packed ? 0 : c.whole * 64, each = packed ? padded : 64;
  Packs& list = packed ? a : tails;
  list.add(pack_args(p, v, v_stride, first, rows, each, (uint16_t*)to, c.v.plane));
  if (g) list.add(pack_args(p, g, g_stride, first, rows, each, (uint16_t*)to + each * p.Hp, c.v.plane));
  return c;
}

// The operands, packed where they cannot be read as they are; tails are left to k_dz. want_x, want_w: those that the
// call reads.
int operands(GCall& c, const void* x, const void* v, const void* g, bool want_x, bool want_w) {
  const GPlan& p = c.p;
  const ews_gated_desc* s = c.s;
  Packs a{};
  c.x = lay_out(a, c.tails, p, x, s->x_stride, nullptr, 0, p.N, p.pack_x, p.tail_x, c.w + p.xp, want_x);
  c.weights = lay_out(a, c.tails, p, v, s->weight_stride, g, s->gate_stride, p.F, p.pack_w, p.tail_w, c.w + p.wp,
                      want_w);
  if (!a.blocks) return EWS_OK;
  if (p.np == 3)
    hipLaunchKernelGGL((k_packs<float>), dim3(a.blocks), dim3(256), 0, c.st, a);
  else
    hipLaunchKernelGGL((k_packs<bf16>), dim3(a.blocks), dim3(256), 0, c.st, a);
  GATED_CHECK();
  return EWS_OK;
}

template <class T, int PAIRS, typename O, bool KEEP>
int launch_forward_as(const ForwardArgs& a, hipStream_t st) {
  const int lds = tiles::lds_bytes<T, PAIRS>(a.kblocks) + T::I * 4;
  const int rc = tiles::allow_lds(k_forward<T, PAIRS, O, KEEP>, lds);
  if (rc != EWS_OK) return rc;
  hipLaunchKernelGGL((k_forward<T, PAIRS, O, KEEP>), dim3((uint32_t)(a.ti * a.tj)), dim3(T::kThreads), lds, st, a);
  GATED_CHECK();
  return EWS_OK;
}

template <typename O, bool KEEP>
int launch_forward(Kind kind, const ForwardArgs& a, hipStream_t st) {
  constexpr int kP = sizeof(O) == 4 ? tiles::kPairs : 1;
  if (kind == tiles::kLarge) return launch_forward_as<tiles::Large, kP, O, KEEP>(a, st);
  return launch_forward_as<tiles::Medium, kP, O, KEEP>(a, st);  // few rows have a kernel of their own
}

template <typename O>
int launch_forward(Kind kind, const ForwardArgs& a, hipStream_t st) {
  return a.kept ? launch_forward<O, true>(kind, a, st) : launch_forward<O, false>(kind, a, st);
}

template <typename T, bool WIDE>
int launch_few(const FewArgs& a, hipStream_t st) {
  const dim3 grid(ceil_div(a.F, 16)), block(64 * kFewWaves);
  if (a.N <= 16)
    hipLaunchKernelGGL((k_few<T, 1, WIDE>), grid, block, 0, st, a);
  else if (a.N <= 32)
    hipLaunchKernelGGL((k_few<T, 2, WIDE>), grid, block, 0, st, a);
  else if constexpr (sizeof(T) == 4)
    hipLaunchKernelGGL((k_few<T, 4, WIDE>), grid, block, 0, st, a);
  GATED_CHECK();
  return EWS_OK;
}

int launch_few_dx(const FewDxArgs& a, int parts, hipStream_t st) {
  const dim3 grid(ceil_div(a.H, 16 * kDxCols), parts), block(64 * kFewWaves);
  if (a.N <= 16)
    hipLaunchKernelGGL(k_few_dx<1>, grid, block, 0, st, a);
  else if (a.N <= 32)
    hipLaunchKernelGGL(k_few_dx<2>, grid, block, 0, st, a);
  else
    hipLaunchKernelGGL(k_few_dx<4>, grid, block, 0, st, a);
  GATED_CHECK();
  return EWS_OK;
}

template <class T, int PAIRS, bool ROWS, typename O>
int launch_grad_as(const GradArgs& a, hipStream_t st) {
  const int lds = tiles::lds_bytes<T, PAIRS>(a.per);
  const int rc = tiles::allow_lds(k_grad<T, PAIRS, ROWS, O>, lds);
  if (rc != EWS_OK) return rc;
  const int others = a.ti * a.tj - a.whole;
  hipLaunchKernelGGL((k_grad<T, PAIRS, ROWS, O>), dim3((uint32_t)(a.whole + others * a.pieces), a.splits),
                     dim3(T::kThreads), lds, st, a);
  GATED_CHECK();
  if constexpr (T::I == 256 && T::J == 256) {
    if (!others) return EWS_OK;
    const dim3 grid((uint32_t)(others * (T::I * T::J / 1024)));
    if (a.wide)
      hipLaunchKernelGGL((k_shared<T, ROWS, O, Eight>), grid, dim3(128), 0, st, a);
    else
      hipLaunchKernelGGL((k_shared<T, ROWS, O, One>), grid, dim3(1024), 0, st, a);
    GATED_CHECK();
  }
  return EWS_OK;
}

template <bool ROWS, typename O>
int launch_join(const GradArgs& a, hipStream_t st) {
  const int64_t n = (int64_t)a.J * a.I;
  if (a.splits > kFewSplits)
    hipLaunchKernelGGL((k_join<ROWS, O, One, 8>), dim3((uint32_t)((n + 31) / 32)), dim3(256), 0, st, a);
  else if (a.wide)
    hipLaunchKernelGGL((k_join<ROWS, O, Eight, 1>), dim3((uint32_t)((n / 8 + 255) / 256)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_join<ROWS, O, One, 1>), dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, st, a);
  GATED_CHECK();
  return EWS_OK;
}

template <bool ROWS, typename O>
int launch_grad(const GProduct& p, GradArgs a, hipStream_t st) {
  constexpr int kP = sizeof(O) == 4 ? tiles::kPairs : 1;
  a.ti = p.ti;
  a.tj = p.tj;
  a.splits = p.splits;
  a.kblocks = p.kblocks;
  a.per = p.per;
  a.whole = p.whole;
  a.pieces = p.pieces;
  int rc;
  if (p.kind == tiles::kLarge)
    rc = launch_grad_as<tiles::Large, kP, ROWS, O>(a, st);
  else if (ROWS || sizeof(O) == 4 || p.kind == tiles::kMedium)
    rc = launch_grad_as<tiles::Medium, kP, ROWS, O>(a, st);
  else  // the weights' gradients are 128 rows at least, and few float32 rows of x's have a kernel of their own
    rc = launch_grad_as<tiles::Flat, 1, false, bf16>(a, st);
  return rc != EWS_OK || a.splits == 1 ? rc : launch_join<ROWS, O>(a, st);
}

template <typename T, bool SUMS>
void launch_dz(const DzArgs& z, dim3 grid, hipStream_t st) {
  hipLaunchKernelGGL((k_dz<T, SUMS>), grid, dim3(256), 0, st, z);
}

// Contiguous rows of whole fours, the first at a multiple of their size.
int fours(const void* p, int cols, bool f32) { return cols % 4 == 0 && (uintptr_t)p % (f32 ? 16 : 8) == 0; }

template <typename T, int HB, int FB>
int launch_narrow_as(const NarrowArgs& a, int groups, bool back, hipStream_t st) {
  typedef Narrow<T, HB, FB> S;
  if (!back) {
    // 16 rows a wavefront and turn
    const int n = ceil_div(a.N, 16 * kNarrowWaves);
    hipLaunchKernelGGL((k_narrow_forward<T, HB, FB>), dim3(n < 2048 ? n : 2048), dim3(64 * kNarrowWaves), 0, st, a);
  } else {
    static_assert(S::kLdsBytes <= 160 << 10 && S::kWaves * 2 * S::FP * (S::HP + 1) * 4 <= S::kLdsBytes,
                  "the sums fit too");
    const int rc = tiles::allow_lds(k_narrow_backward<T, HB, FB>, S::kLdsBytes);
    if (rc != EWS_OK) return rc;
    hipLaunchKernelGGL((k_narrow_backward<T, HB, FB>), dim3(groups), dim3(64 * S::kWaves), S::kLdsBytes, st, a);
  }
  GATED_CHECK();
  return EWS_OK;
}

template <typename T>
int launch_narrow(const NarrowArgs& a, int groups, bool back, hipStream_t st) {
  if (a.H <= 32)
    return a.F <= 32 ? launch_narrow_as<T, 1, 1>(a, groups, back, st) : launch_narrow_as<T, 1, 2>(a, groups, back, st);
  return a.F <= 32 ? launch_narrow_as<T, 2, 1>(a, groups, back, st) : launch_narrow_as<T, 2, 2>(a, groups, back, st);
}

NarrowArgs narrow_args(const ews_gated_desc* s, const void* x, const void* v, const void* g, const void* bias,
                       const void* gate_bias) {
  NarrowArgs a{};
  a.x = x;
  a.v = v;
  a.g = g;
  a.xs = s->x_stride;
  a.vs = s->weight_stride;
  a.gs = s->gate_stride;
  a.N = s->rows;
  a.H = s->width;
  a.F = s->features;
  a.bias = bias;
  a.gate_bias = gate_bias;
  a.act = s->activation;
  a.wide_x = s->width % 8 == 0 && tiles::rows_wide(x, s->x_stride, s->dtype == EWS_DTYPE_F32);
  return a;
}

// Rows of results that are contiguous: whether they start at multiples of 16 bytes and hold whole eights.
int results_wide(const void* p, int cols) { return cols % 8 == 0 && (uintptr_t)p % 16 == 0; }

}  // namespace

extern "C" {

size_t ews_gated_kept_bytes(const ews_gated_desc* desc) {
  GPlan p;
  if (gated_plan(desc, nullptr, nullptr, nullptr, false, true, p) != EWS_OK) return 0;
  return p.narrow ? 0 : (size_t)(p.N * 2 * p.ld) * (p.np == 3 ? 4 : 3);
}

size_t ews_gated_workspace_bytes(const ews_gated_desc* desc, const void* x, const void* weight,
                                 const void* gate_weight, int call) {
  GPlan p;
  if (gated_plan(desc, x, weight, gate_weight, call == EWS_GATED_BACKWARD, call == EWS_GATED_KEEP, p) != EWS_OK)
    return 0;
  return p.total;
}

int ews_gated_tile(const ews_gated_desc* desc, int product, int32_t* tile) {
  GPlan p;
  const int rc = gated_plan(desc, nullptr, nullptr, nullptr, true, true, p);
  if (rc != EWS_OK) return rc;
  if (!tile) return EWS_ERR_NULL;
  if (product < 0 || product > 2) return EWS_ERR_OPTION;
  if (p.narrow || (product == 0 && p.few) || (product == 1 && p.few_dx)) {
    for (int k = 0; k < 5; ++k) tile[k] = 0;
    return EWS_OK;
  }
  const Product& q = product == 0 ? p.forward : product == 1 ? p.dx : static_cast<const Product&>(p.dw);
  tile[0] = q.tile_i;
  tile[1] = q.tile_j;
  tile[2] = q.splits;
  tile[3] = product == 0 ? q.ti * q.tj : product == 1 ? p.dx.whole : p.dw.whole;
  tile[4] = q.ti * q.tj;
  return EWS_OK;
}

int ews_gated_forward(const ews_gated_desc* desc, const void* x, const void* weight, const void* bias,
                      const void* gate_weight, const void* gate_bias, void* out, void* kept, void* workspace,
                      ews_stream_t stream) {
  GCall c{};
  int rc = gated_plan(desc, x, weight, gate_weight, false, kept != nullptr, c.p);
  if (rc != EWS_OK) return rc;
  if (!x || !weight || !gate_weight || !out || (c.p.total && !workspace)) return EWS_ERR_NULL;
  const bool f32 = c.p.np == 3;
  c.s = desc;
  c.w = (char*)workspace;
  c.st = (hipStream_t)stream;
  if (c.p.few && !c.p.narrow) {
    const FewArgs a{x,       weight,  gate_weight, desc->x_stride, desc->weight_stride, desc->gate_stride,
                    c.p.N,   c.p.H,   c.p.F,       bias,           gate_bias,           desc->activation,
                    out,     kept,    c.p.ld};
    const bool wide = c.p.H % 8 == 0 && tiles::rows_wide(x, desc->x_stride, f32) &&
                      tiles::rows_wide(weight, desc->weight_stride, f32) &&
                      tiles::rows_wide(gate_weight, desc->gate_stride, f32);
    if (f32) return wide ? launch_few<float, true>(a, c.st) : launch_few<float, false>(a, c.st);
    return wide ? launch_few<bf16, true>(a, c.st) : launch_few<bf16, false>(a, c.st);
  }
  if (c.p.narrow) {
    NarrowArgs a = narrow_args(desc, x, weight, gate_weight, bias, gate_bias);
    a.out = out;
    a.wide_f = fours(out, a.F, f32);
    return f32 ? launch_narrow<float>(a, 0, false, c.st) : launch_narrow<bf16>(a, 0, false, c.st);
  }
  rc = operands(c, x, weight, gate_weight, true, true);
  if (rc != EWS_OK) return rc;
  ForwardArgs a{};
  a.W = Pair{c.weights.v, c.weights.to_g};
  a.X = c.x.v;
  a.ti = c.p.forward.ti;
  a.tj = c.p.forward.tj;
  a.kblocks = c.p.forward.kblocks;
  a.N = c.p.N;
  a.F = c.p.F;
  a.bias = bias;
  a.gate_bias = gate_bias;
  a.act = desc->activation;
  a.wide = results_wide(out, c.p.F);
  a.out = out;
  a.kept = kept;
  a.ld = c.p.ld;
  return f32 ? launch_forward<float>(c.p.forward.kind, a, c.st) : launch_forward<bf16>(c.p.forward.kind, a, c.st);
}

int ews_gated_backward(const ews_gated_desc* desc, const void* x, const void* weight, const void* bias,
                       const void* gate_weight, const void* gate_bias, const void* kept, const void* grad_out,
                       void* grad_x, void* grad_weight, void* grad_bias, void* grad_gate_weight, void* grad_gate_bias,
                       void* workspace, ews_stream_t stream) {
  GCall c{};
  int rc = gated_plan(desc, x, weight, gate_weight, true, false, c.p);
  if (rc != EWS_OK) return rc;
  if (!x || !weight || !gate_weight || (!kept && !c.p.narrow) || !grad_out || !workspace) return EWS_ERR_NULL;
  const GPlan& p = c.p;
  const bool f32 = p.np == 3;
  c.s = desc;
  c.w = (char*)workspace;
  c.st = (hipStream_t)stream;
  const bool weights = grad_weight || grad_gate_weight, biases = grad_bias || grad_gate_bias;
  if (p.narrow) {
    NarrowArgs n = narrow_args(desc, x, weight, gate_weight, bias, gate_bias);
    n.dy = grad_out;
    n.dx = grad_x;
    n.wide_f = fours(grad_out, n.F, f32);
    n.wide_h = fours(grad_x, n.H, f32);
    n.part = weights || biases ? (float*)workspace : nullptr;
    rc = f32 ? launch_narrow<float>(n, p.narrow_groups, true, c.st)
             : launch_narrow<bf16>(n, p.narrow_groups, true, c.st);
    if (rc != EWS_OK || !n.part) return rc;
    const int FP = narrow_pad(n.F), HP = narrow_pad(n.H);
    const dim3 grid(ceil_div(2 * FP * (HP + 1), 64));
    if (f32)
      hipLaunchKernelGGL((k_join_narrow<float>), grid, dim3(1024), 0, c.st, n.part, p.narrow_groups, FP, HP, n.F, n.H,
                         (float*)grad_weight, (float*)grad_bias, (float*)grad_gate_weight, (float*)grad_gate_bias);
    else
      hipLaunchKernelGGL((k_join_narrow<bf16>), grid, dim3(1024), 0, c.st, n.part, p.narrow_groups, FP, HP, n.F, n.H,
                         (bf16*)grad_weight, (bf16*)grad_bias, (bf16*)grad_gate_weight, (bf16*)grad_gate_bias);
    GATED_CHECK();
    return EWS_OK;
  }
  rc = operands(c, x, weight, gate_weight, weights, grad_x && !p.few_dx);
  if (rc != EWS_OK) return rc;
  DzArgs z{};
  z.dy = grad_out;
  z.kept = kept;
  z.act = desc->activation;
  z.N = p.N;
  z.F = p.F;
  z.padded = (int)p.Np;
  z.ld = p.ld;
  z.wide = results_wide(grad_out, p.F);
  z.dz = (uint16_t*)(c.w + p.dz);
  z.plane = p.Np * 2 * p.ld;
  z.sums = biases ? (float*)(c.w + p.sums) : nullptr;
  z.each = p.dz_rows;
  z.parts = p.dz_parts;
  z.tails = c.tails;
  const int wide = ceil_div(p.ld, 512);
  const dim3 grid(wide, p.dz_parts + ceil_div(c.tails.blocks, wide));
  if (f32)
    z.sums ? launch_dz<float, true>(z, grid, c.st) : launch_dz<float, false>(z, grid, c.st);
  else
    z.sums ? launch_dz<bf16, true>(z, grid, c.st) : launch_dz<bf16, false>(z, grid, c.st);
  GATED_CHECK();
  if (biases) {
    const dim3 g(ceil_div(p.F, 64), 2);
    if (f32)
      hipLaunchKernelGGL((k_dbias<float>), g, dim3(1024), 0, c.st, z.sums, p.dz_parts, p.ld, p.F, (float*)grad_bias,
                         (float*)grad_gate_bias);
    else
      hipLaunchKernelGGL((k_dbias<bf16>), g, dim3(1024), 0, c.st, z.sums, p.dz_parts, p.ld, p.F, (bf16*)grad_bias,
                         (bf16*)grad_gate_bias);
    GATED_CHECK();
  }
  GradArgs a{};
  a.I = p.H;
  a.F = p.F;
  a.ld = (int)p.ld;
  a.part = (float*)(c.w + p.part);
  if (grad_x && p.few_dx) {
    const FewDxArgs d{z.dz, z.plane, p.ld, (const float*)weight, (const float*)gate_weight, desc->weight_stride,
                      desc->gate_stride, p.N, p.H, p.F, p.dx_blocks, p.dx_per, a.part};
    rc = launch_few_dx(d, p.dx_parts, c.st);
    if (rc != EWS_OK) return rc;
    a.splits = p.dx_parts;
    a.J = p.N;
    a.out = grad_x;
    a.wide = results_wide(grad_x, p.H);
    rc = launch_join<false, float>(a, c.st);
    if (rc != EWS_OK) return rc;
  } else if (grad_x) {
    a.W = c.weights;
    a.Z = Operand{z.dz, 2 * p.ld, z.plane, (int)p.Np, 0};
    a.J = p.N;
    a.out = grad_x;
    a.wide = results_wide(grad_x, p.H);
    rc = f32 ? launch_grad<false, float>(p.dx, a, c.st) : launch_grad<false, bf16>(p.dx, a, c.st);
    if (rc != EWS_OK) return rc;
  }
  if (weights) {
    a.X = c.x;
    a.Z = Operand{z.dz, 2 * p.ld, z.plane, (int)p.Np, (int)(2 * p.ld)};
    a.J = (int)(2 * p.ld);
    a.out = grad_weight;
    a.gate_out = grad_gate_weight;
    a.wide = p.H % 8 == 0 && (uintptr_t)grad_weight % 16 == 0 && (uintptr_t)grad_gate_weight % 16 == 0;
    rc = f32 ? launch_grad<true, float>(p.dw, a, c.st) : launch_grad<true, bf16>(p.dw, a, c.st);
    if (rc != EWS_OK) return rc;
  }
  return EWS_OK;
}

}  // extern "C"
