// The gated linear map of ews_gated.hip for widths up to 64: many rows through small V and G, bound by x, y, dy and
// dx's bytes. (131072 rows of 32 by 32, float32, by the tiles, forward and backward: x packed into planes, 50 MB, and
// dv | dg, 100 MB, are most of what moves, and the call takes 282 us; here the forward's kernel takes 19, the
// backward's 38 and the join 4, medians of a trace.)
//
// Nothing is kept and nothing but results is written: a wavefront holds 32 rows, and the backward forms v and g anew. V
// and G lie in LDS as the matrix instructions' fragments, cut into planes once by every workgroup, which then walks
// through rows. v_mfma_f32_16x16x32_bf16: lane l holds row (of the second operand column) l % 16 at k = 8 (l / 16) +
// 0..7, and results column l % 16, rows 4 (l / 16) + 0..3.
//
//   v, g   [f, n] = sum over h of V[f, h] x[n, h]: a lane gets four neighbouring f of one row.
//   dx     [h, n] = sum over f of V[f, h] dv[n, f] + G[f, h] dg[n, f]: dv and dg are in that layout already. A
//          product's k may be in any order that its operands share: of 32 f lane l's are 4 (l / 16) + 0..3 and 16 more,
//          which are two of its results, so only V's and G's fragments are laid out for it.
//   dV, dG [f, h] = sum over n of dv[n, f] x[n, h]: n has to run along a lane's eight, so both are turned through LDS,
//          32 rows at a time. The sums stay in registers; the wavefronts' are laid side by side in LDS at the end and
//          added in order (one after the other into the same place: 512 rows of 64 by 64 in bfloat16 63 us both ways,
//          now 35), the workgroups' by k_join_narrow in order.
//
// Float32 is multiplied as six products of bfloat16 planes; dv and dg of bfloat16 calls have two planes, which costs
// nothing here and rounds the gradients once. The second plane, of either sign or 0, must not meet an infinity: where V
// or G hold one, or the rows of x, which makes their v infinite or NaN, the products are formed with care.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "ews_hip.h"
#include "ews_pack.h"
#include "ews_tiles.h"
#include "ews_vec.h"

namespace ews {
namespace gated {

using namespace ews::tiles;
using namespace ews::vec;

constexpr int kNarrowWidth = 64;
constexpr int kNarrowWaves = 4;  // of the forward
constexpr int kTurnRow = 36;     // floats between rows of what is turned through LDS: 32 and a piece, off the banks

typedef float f32x4v __attribute__((ext_vector_type(4)));

struct NarrowArgs {
  const void* x;
  const void* v;
  const void* g;
  int64_t xs, vs, gs;
  int N, H, F;
  const void* bias;
  const void* gate_bias;
  int act;
  int wide_x;      // x's rows start at multiples of 16 bytes and hold whole eights
  int wide_f;      // rows of out, or of grad_out, hold whole fours and start at multiples of their size
  int wide_h;      // rows of grad_x
  void* out;       // forward
  const void* dy;  // backward
  void* dx;        // or null
  float* part;     // (workgroups, 2 FP, HP + 1): sums of dv, dg times x, and of dv, dg; or null
};

// Planes of a type's own numbers, and of dv and dg.
template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
template <typename T>
constexpr int kZPlanes = sizeof(T) == 4 ? 3 : 2;

template <typename T>
__device__ __forceinline__ void fragments(const T (&x)[8], bf16x8 (&f)[kPlanes<T>]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint16_t p[kPlanes<T>];
    planes(x[q], p);
#pragma unroll
    for (int n = 0; n < kPlanes<T>; ++n) f[n][q] = __builtin_bit_cast(__bf16, p[n]);
  }
}

// Float32 numbers as the planes of dv and dg.
template <int NP>
__device__ __forceinline__ void z_fragments(const float (&x)[8], bf16x8 (&f)[NP]) {
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    if constexpr (NP == 3) {
      uint16_t p[3];
      planes(x[q], p);
#pragma unroll
      for (int n = 0; n < 3; ++n) f[n][q] = __builtin_bit_cast(__bf16, p[n]);
    } else {
      f[0][q] = (__bf16)x[q];
      const float hi = (float)f[0][q];
      f[1][q] = (__bf16)(__builtin_isfinite(hi) ? x[q] - hi : 0.0f);
    }
  }
}

// acc += p q, the smallest products first.
template <int NA, int NB>
__device__ __forceinline__ void mac(const bf16x8 (&p)[NA], const bf16x8 (&q)[NB], f32x4v& acc) {
  if constexpr (NA == 3 && NB == 3) {
#pragma unroll
    for (int pair = 0; pair < kPairs; ++pair)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[piece_p(pair)], q[piece_q(pair)], acc, 0, 0, 0);
  } else {
    static_assert(NA == 1 || NB == 1, "one of the two is not cut");
#pragma unroll
    for (int n = (NA > NB ? NA : NB) - 1; n >= 0; --n)
      acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[NA > 1 ? n : 0], q[NB > 1 ? n : 0], acc, 0, 0, 0);
  }
}

// The same of one plane w, which may hold infinities, and two planes z: W_FIRST, w is the first operand.
template <bool W_FIRST, int NZ>
__device__ __forceinline__ void mac_infinite(const bf16x8& w, const bf16x8 (&z)[NZ], f32x4v& acc) {
  u32x4 u = __builtin_bit_cast(u32x4, w);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if ((u[q] & 0x7f80u) == 0x7f80u) u[q] &= 0xffff0000u;
    if ((u[q] & 0x7f800000u) == 0x7f800000u) u[q] &= 0xffffu;
  }
  const bf16x8 finite = __builtin_bit_cast(bf16x8, u);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(W_FIRST ? finite : z[1], W_FIRST ? z[1] : finite, acc, 0, 0, 0);
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(W_FIRST ? w : z[0], W_FIRST ? z[0] : w, acc, 0, 0, 0);
}

// Eight neighbouring numbers of a row from column k on, zero past the row's end.
template <typename T>
__device__ __forceinline__ void eight_of(const T* row, int k, int H, bool wide, T (&x)[8]) {
  if (wide && k < H) {  // H is a multiple of 8
#pragma unroll
    for (int q = 0; q < 8; q += kWide<T>)
      *reinterpret_cast<u32x4*>(x + q) = *reinterpret_cast<const u32x4*>(row + k + q);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = k + q < H ? row[k + q] : narrow<T>(0.0f);
  }
}

// Four neighbouring numbers, those past the row's end left alone (zero).
template <typename T>
__device__ __forceinline__ void load_four(const T* row, int k, int n, bool wide, float (&x)[4]) {
  T y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) y[q] = narrow<T>(0.0f);
  if (wide && k < n) {
    if (sizeof(T) == 4)
      *reinterpret_cast<u32x4*>(y) = *reinterpret_cast<const u32x4*>(row + k);
    else
      *reinterpret_cast<u32x2*>(y) = *reinterpret_cast<const u32x2*>(row + k);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (k + q < n) y[q] = row[k + q];
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = widen(y[q]);
}
template <typename T>
__device__ __forceinline__ void store_four(T* row, int k, int n, bool wide, const float (&x)[4]) {
  T y[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) y[q] = narrow<T>(x[q]);
  if (wide && k < n) {
    if (sizeof(T) == 4)
      *reinterpret_cast<u32x4*>(row + k) = *reinterpret_cast<const u32x4*>(y);
    else
      *reinterpret_cast<u32x2*>(row + k) = *reinterpret_cast<const u32x2*>(y);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (k + q < n) row[k + q] = y[q];
  }
}

// HB, FB: blocks of 32 of H and F.
template <typename T, int HB, int FB>
struct Narrow {
  static constexpr int NP = kPlanes<T>, HP = 32 * HB, FP = 32 * FB;
  static constexpr int kFront = NP * HB * 2 * 2 * FB;        // fragments of v and g: [plane][h block][side][16 f]
  static constexpr int kTurned = NP * 2 * FB * 2 * HB;       // of dx: [plane][side][f block][16 h]
  static constexpr int kTurn = (2 * FP + HP) * kTurnRow;     // floats that a wavefront turns: dv, dg, x by column
  static constexpr int kRest = (kFront + kTurned) * 1024 + 2 * FP * 4;
  static constexpr int kWaves = kRest + 4 * kTurn * 4 <= 160 << 10 ? 4 : 2;  // of the backward, as far as LDS goes
  static constexpr int kLdsBytes = kRest + kWaves * kTurn * 4;
  static __device__ __forceinline__ int front(int plane, int hb, int side, int f16) {
    return ((plane * HB + hb) * 2 + side) * 2 * FB + f16;
  }
  static __device__ __forceinline__ int turned(int plane, int side, int fb, int h16) {
    return kFront + ((plane * 2 + side) * FB + fb) * 2 * HB + h16;
  }
  // What of a block of 32 f a lane's e-th number of dx's k is.
  static __device__ __forceinline__ int f_of(int lane, int e) { return (e >> 2) * 16 + (lane >> 4) * 4 + (e & 3); }
};

// Wavefronts of a workgroup of the backward.
template <typename T>
int narrow_waves(int H, int F) {
  if (H <= 32) return F <= 32 ? Narrow<T, 1, 1>::kWaves : Narrow<T, 1, 2>::kWaves;
  return F <= 32 ? Narrow<T, 2, 1>::kWaves : Narrow<T, 2, 2>::kWaves;
}

// V's and G's fragments and the biases ([side][FP]) into LDS.
template <typename T, int HB, int FB, int WAVES, bool BACK>
__device__ __forceinline__ void lay_out(const NarrowArgs& a, bf16x8* frag, float* bias) {
  typedef Narrow<T, HB, FB> S;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, k8 = (lane >> 4) * 8;
  for (int n = wave; n < HB * 2 * 2 * FB; n += WAVES) {
    const int hb = n / (4 * FB), side = n / (2 * FB) % 2, f16 = n % (2 * FB);
    const int f = f16 * 16 + r16;
    const T* row = side ? (const T*)a.g + f * a.gs : (const T*)a.v + f * a.vs;
    T w[8];
    eight_of<T>(row, hb * 32 + k8, f < a.F ? a.H : 0, false, w);
    bf16x8 p[S::NP];
    fragments<T>(w, p);
#pragma unroll
    for (int q = 0; q < S::NP; ++q) frag[S::front(q, hb, side, f16) * 64 + lane] = p[q];
  }
  if (BACK) {
    for (int n = wave; n < 2 * FB * 2 * HB; n += WAVES) {
      const int side = n / (FB * 2 * HB), fb = n / (2 * HB) % FB, h16 = n % (2 * HB);
      const int h = h16 * 16 + r16;
      T w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int f = fb * 32 + S::f_of(lane, e);
        w[e] = f < a.F && h < a.H ? (side ? ((const T*)a.g)[f * a.gs + h] : ((const T*)a.v)[f * a.vs + h])
                                  : narrow<T>(0.0f);
      }
      bf16x8 p[S::NP];
      fragments<T>(w, p);
#pragma unroll
      for (int q = 0; q < S::NP; ++q) frag[S::turned(q, side, fb, h16) * 64 + lane] = p[q];
    }
  }
  for (int t = threadIdx.x; t < 2 * S::FP; t += 64 * WAVES) {
    const int f = t % S::FP;
    const T* b = (const T*)(t < S::FP ? a.bias : a.gate_bias);
    bias[t] = b && f < a.F ? widen(b[f]) : 0.0f;
  }
  __syncthreads();
}

// v and g of 16 rows, without the biases; x: their numbers as they were read.
template <typename T, int HB, int FB>
__device__ __forceinline__ void front_of(const NarrowArgs& a, const bf16x8* frag, int n0, T (&x)[HB][8],
                                         f32x4v (&z)[2][2 * FB]) {
  typedef Narrow<T, HB, FB> S;
  const int lane = threadIdx.x & 63, n = n0 + (lane & 15);
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int f16 = 0; f16 < 2 * FB; ++f16) z[side][f16] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int hb = 0; hb < HB; ++hb)
    eight_of<T>((const T*)a.x + (n < a.N ? n : 0) * a.xs, hb * 32 + (lane >> 4) * 8, n < a.N ? a.H : 0, a.wide_x,
                x[hb]);
#pragma unroll
  for (int hb = 0; hb < HB; ++hb) {
    bf16x8 p[S::NP];
    fragments<T>(x[hb], p);
#pragma unroll
    for (int side = 0; side < 2; ++side)
#pragma unroll
      for (int f16 = 0; f16 < 2 * FB; ++f16) {
        bf16x8 w[S::NP];
#pragma unroll
        for (int q = 0; q < S::NP; ++q) w[q] = frag[S::front(q, hb, side, f16) * 64 + lane];
        mac(w, p, z[side][f16]);
      }
  }
}

template <typename T, int HB, int FB>
__global__ __launch_bounds__(64 * kNarrowWaves) void k_narrow_forward(NarrowArgs a) {
  typedef Narrow<T, HB, FB> S;
  __shared__ bf16x8 frag[S::kFront * 64];
  __shared__ float bias[2 * S::FP];
  lay_out<T, HB, FB, kNarrowWaves, false>(a, frag, bias);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int step = gridDim.x * kNarrowWaves * 16;
  for (int n0 = (blockIdx.x * kNarrowWaves + wave) * 16; n0 < a.N; n0 += step) {
    T x[HB][8];
    f32x4v z[2][2 * FB];
    front_of<T, HB, FB>(a, frag, n0, x, z);
    const int n = n0 + (lane & 15);
#pragma unroll
    for (int f16 = 0; f16 < 2 * FB; ++f16) {
      const int f = f16 * 16 + (lane >> 4) * 4;
      float y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float act, slope;
        activate<T>(a.act, z[1][f16][r] + bias[S::FP + f + r], act, slope);
        y[r] = (z[0][f16][r] + bias[f + r]) * act;
      }
      if (n < a.N) store_four<T>((T*)a.out + (int64_t)n * a.F, f, a.F, a.wide_f, y);
    }
  }
}

template <typename T, int HB, int FB>
__global__ __launch_bounds__((64 * Narrow<T, HB, FB>::kWaves)) void k_narrow_backward(NarrowArgs a) {
  typedef Narrow<T, HB, FB> S;
  constexpr int NP = S::NP, NZ = kZPlanes<T>;
  extern __shared__ char lds[];
  bf16x8* frag = reinterpret_cast<bf16x8*>(lds);
  float* bias = reinterpret_cast<float*>(lds + (S::kFront + S::kTurned) * 1024);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, q4 = (lane >> 4) * 4, k8 = (lane >> 4) * 8;
  float* turn = bias + 2 * S::FP + wave * S::kTurn;
  lay_out<T, HB, FB, S::kWaves, true>(a, frag, bias);
  f32x4v dw[4 * FB][2 * HB];  // [16 f of dV, then of dG][16 h]
  float db[4 * FB][4];
#pragma unroll
  for (int i = 0; i < 4 * FB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      db[i][r] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2 * HB; ++h) dw[i][h][r] = 0.0f;
    }
  bool infinite_weights = false;
  if (NZ == 2) {
    for (int n = 0; n < S::kFront; ++n) {
      const u32x4 u = __builtin_bit_cast(u32x4, frag[n * 64 + lane]);
#pragma unroll
      for (int q = 0; q < 4; ++q)
        infinite_weights |= (u[q] & 0x7f80u) == 0x7f80u || (u[q] & 0x7f800000u) == 0x7f800000u;
    }
    infinite_weights = __any(infinite_weights);
  }
  const int step = gridDim.x * S::kWaves * 32;
  for (int n0 = (blockIdx.x * S::kWaves + wave) * 32; n0 < a.N; n0 += step) {
    bool infinite = infinite_weights;  // an operand of these rows may be
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int n = n0 + c * 16 + r16;
      T x[HB][8];
      f32x4v z[2][2 * FB];
      front_of<T, HB, FB>(a, frag, n0 + c * 16, x, z);
      if (NZ == 2) infinite |= __any(!__builtin_isfinite(z[0][0][0]));  // as with any infinity in the row of x
      // z becomes dv and dg
#pragma unroll
      for (int f16 = 0; f16 < 2 * FB; ++f16) {
        float u[4];
        load_four<T>((const T*)a.dy + (int64_t)(n < a.N ? n : 0) * a.F, f16 * 16 + q4, n < a.N ? a.F : 0, a.wide_f, u);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int f = f16 * 16 + q4 + r;
          float act, slope;
          const float v = z[0][f16][r] + bias[f];
          activate<T>(a.act, z[1][f16][r] + bias[S::FP + f], act, slope);
          z[0][f16][r] = n < a.N ? u[r] * act : 0.0f;
          z[1][f16][r] = n < a.N ? u[r] * (v * slope) : 0.0f;
        }
      }
      if (a.part) {
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int f16 = 0; f16 < 2 * FB; ++f16)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              db[side * 2 * FB + f16][r] += z[side][f16][r];
              turn[(side * S::FP + f16 * 16 + q4 + r) * kTurnRow + c * 16 + r16] = z[side][f16][r];
            }
#pragma unroll
        for (int hb = 0; hb < HB; ++hb)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            turn[(2 * S::FP + hb * 32 + k8 + e) * kTurnRow + c * 16 + r16] = widen(x[hb][e]);
      }
      auto form_dx = [&](auto careful) {
        f32x4v d[2 * HB];
#pragma unroll
        for (int h = 0; h < 2 * HB; ++h) d[h] = f32x4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int side = 0; side < 2; ++side)
#pragma unroll
          for (int fb = 0; fb < FB; ++fb) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = z[side][2 * fb + (e >> 2)][e & 3];
            bf16x8 p[NZ];
            z_fragments<NZ>(y, p);
#pragma unroll
            for (int h = 0; h < 2 * HB; ++h) {
              bf16x8 w[NP];
#pragma unroll
              for (int q = 0; q < NP; ++q) w[q] = frag[S::turned(q, side, fb, h) * 64 + lane];
              if constexpr (decltype(careful)::value)
                mac_infinite<true>(w[0], p, d[h]);
              else
                mac(w, p, d[h]);
            }
          }
        if (n < a.N) {
#pragma unroll
          for (int h = 0; h < 2 * HB; ++h) {
            const float y[4] = {d[h][0], d[h][1], d[h][2], d[h][3]};
            store_four<T>((T*)a.dx + (int64_t)n * a.H, h * 16 + q4, a.H, a.wide_h, y);
          }
        }
      };
      if (a.dx) {
        if (NZ == 2 && infinite)
          form_dx(std::bool_constant<NZ == 2>{});
        else
          form_dx(std::false_type{});
      }
    }
    if (!a.part) continue;
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    bf16x8 px[2 * HB][NP];
#pragma unroll
    for (int h = 0; h < 2 * HB; ++h) {
      const float* from = turn + (2 * S::FP + h * 16 + r16) * kTurnRow + k8;
      T y[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(from + e);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[e + k] = narrow<T>(w[k]);
      }
      fragments<T>(y, px[h]);
    }
    auto add_dw = [&](auto careful) {
#pragma unroll
      for (int i = 0; i < 4 * FB; ++i) {
        const float* from = turn + (i * 16 + r16) * kTurnRow + k8;
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          const f32x4 w = *reinterpret_cast<const f32x4*>(from + e);
#pragma unroll
          for (int k = 0; k < 4; ++k) y[e + k] = w[k];
        }
        bf16x8 pz[NZ];
        z_fragments<NZ>(y, pz);
#pragma unroll
        for (int h = 0; h < 2 * HB; ++h) {
          if constexpr (decltype(careful)::value)
            mac_infinite<false>(px[h][0], pz, dw[i][h]);
          else
            mac(pz, px[h], dw[i][h]);
        }
      }
    };
    if (NZ == 2 && infinite)
      add_dw(std::bool_constant<NZ == 2>{});
    else
      add_dw(std::false_type{});
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  if (!a.part) return;
  // the wavefronts' sums side by side into LDS, then added in order and out
  constexpr int kRow = S::HP + 1, kSums = 2 * S::FP * kRow;
  float* sum = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int i = 0; i < 4 * FB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int d = 8; d; d >>= 1) db[i][r] += __shfl_xor(db[i][r], d);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4 * FB; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float* to = sum + wave * kSums + (i * 16 + q4 + r) * kRow;
#pragma unroll
      for (int h = 0; h < 2 * HB; ++h) to[h * 16 + r16] = dw[i][h][r];
      if (r16 == 0) to[S::HP] = db[i][r];
    }
  __syncthreads();
  for (int t = threadIdx.x; t < kSums; t += 64 * S::kWaves) {
    float s = sum[t];
#pragma unroll
    for (int w = 1; w < S::kWaves; ++w) s += sum[w * kSums + t];
    a.part[(int64_t)blockIdx.x * kSums + t] = s;
  }
}

// The workgroups' sums added in order: 64 of them at a time by a workgroup, its sixteen wavefronts a contiguous part of
// the workgroups each.
template <typename T>
__global__ __launch_bounds__(1024) void k_join_narrow(const float* part, int parts, int FP, int HP, int F, int H, T* dv,
                                                      T* dbv, T* dg, T* dbg) {
  __shared__ float joined[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = HP + 1, n = 2 * FP * row;
  const int at = blockIdx.x * 64 + lane;
  const int each = (parts + 15) / 16, p1 = (wave + 1) * each < parts ? (wave + 1) * each : parts;
  float s = 0.0f;
  if (at < n) {
#pragma unroll 8
    for (int p = wave * each; p < p1; ++p) s += part[(int64_t)p * n + at];
  }
  joined[wave][lane] = s;
  __syncthreads();
  if (wave || at >= n) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += joined[w][lane];
  const int h = at % row, fs = at / row, side = fs / FP, f = fs % FP;
  if (f >= F) return;
  if (h == HP) {
    T* to = side ? dbg : dbv;
    if (to) to[f] = narrow<T>(s);
  } else if (h < H) {
    T* to = side ? dg : dv;
    if (to) to[f * H + h] = narrow<T>(s);
  }
}

}  // namespace gated
}  // namespace ews
