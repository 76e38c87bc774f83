// Rows of float32 or bfloat16 numbers read and written sixteen bytes a lane, for the kernels around a token model's
// blocks (ews_embed.hip, ews_clip.hip, ews_loss.hip). Arithmetic is float32; a store rounds once, to nearest even.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ews {
namespace vec {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float widen(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
__device__ __forceinline__ float widen(float x) { return x; }

__device__ __forceinline__ uint16_t round_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

// Two numbers rounded to bfloat16 in one word, `lo` in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return (uint32_t)round_bf16(lo) | ((uint32_t)round_bf16(hi) << 16);
}

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ bf16 narrow<bf16>(float x) {
  return bf16{round_bf16(x)};
}

// V consecutive numbers: V = 16 / sizeof(T) as one 16-byte access (the address a multiple of 16), V = 1 as one number.
// store_past: for results that nobody reads soon, past the caches where whole pieces are written.
template <typename T, int V>
struct Pack;

template <>
struct Pack<float, 4> {
  f32x4 w;
  __device__ __forceinline__ void load(const float* p) { w = *reinterpret_cast<const f32x4*>(p); }
  __device__ __forceinline__ float get(int i) const { return w[i]; }
  __device__ __forceinline__ void set(const float* x) { w = f32x4{x[0], x[1], x[2], x[3]}; }
  __device__ __forceinline__ void store(float* p) const { *reinterpret_cast<f32x4*>(p) = w; }
  __device__ __forceinline__ void store_past(float* p) const {
    __builtin_nontemporal_store(w, reinterpret_cast<f32x4*>(p));
  }
};

template <>
struct Pack<bf16, 8> {
  u32x4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = w[i >> 1];
    return __uint_as_float((i & 1) ? (u & 0xffff0000u) : (u << 16));
  }
  __device__ __forceinline__ void set(const float* x) {
    w = u32x4{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
  }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<u32x4*>(p) = w; }
  __device__ __forceinline__ void store_past(bf16* p) const {
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p));
  }
};

template <typename T>
struct Pack<T, 1> {
  T w;
  __device__ __forceinline__ void load(const T* p) { w = *p; }
  __device__ __forceinline__ float get(int) const { return widen(w); }
  __device__ __forceinline__ void set(const float* x) { w = narrow<T>(x[0]); }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
  __device__ __forceinline__ void store_past(T* p) const { *p = w; }
};

template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);

}  // namespace vec
}  // namespace ews
