// Gated linear recurrence over sequences on MI355X (gfx950), forward and backward.
//
//   convex   a_t = sigmoid(g_t), h_t = a_t h_{t-1} + (1 - a_t) x_t
//   linear   a_t = g_t,          h_t = a_t h_{t-1} + x_t
//
// for every channel by itself, h_0 given or zero. A step off the mask has a = 1 and no input (h stays), and nothing
// that its x and g hold is used. With l_t the gradient of h_t and m_t = a_t l_t that of h_{t-1}:
//
//   l_t = dh_t + m_{t+1} (m after the last step: the last state's own gradient)
//   convex   dx_t = l_t (1 - a_t),   dg_t = l_t (h_{t-1} - x_t) a_t (1 - a_t)
//   linear   dx_t = l_t,             dg_t = l_t h_{t-1}
//
// 1 - a is formed as e a with e = exp(-g), so neither side of the gate loses digits. States are float32.
//
// A few operations a number: memory bounds it. The forward reads x and g and writes h; the backward reads x, g and dh
// and writes dx and dg. It forms the states anew from those at the starts of tiles, which the forward leaves in float32
// (one state in the 8 steps of a thread that walks alone, 8% more bytes of a bfloat16 forward and 5% of its backward;
// in 64 to 512 of a strip's tile): h in bfloat16 would be as large as x, and dg would lose what h - x cancels.
//
// A step is the map h -> a h + b, and maps compose: (a2, b2) after (a1, b1) is (a2 a1, a2 b1 + b2). A workgroup owns a
// strip of channels of one sequence and walks it in tiles of steps, a thread kSteps steps of its channels: it composes
// its own steps, its wavefront's by shuffles, the workgroup's through LDS, and then applies them to the state before.
// Loads of the next tile are on their way meanwhile. Where there are channels enough to fill the chip, a thread walks
// its channels alone and nothing is exchanged. Where there are few, sequences are cut into segments: a first launch
// composes each segment's steps (k_ends), and each workgroup of the second applies those before its own.
//
// Medians of a trace of ten calls, bfloat16: 8 x 4095 x 2048 (strips) forward 106 us (3.8 TB/s with the tiles' states),
// backward 155 (4.4), one workgroup a CU and the VALU busy for half of it; 1 x 131071 x 1024 (segments, which read x
// and g, backward g and dh, twice) 143 + 164 and 139 + 299; a step of 8 x 1 x 2048 3.6. (Calls in a row, untraced, take
// a twentieth less.)
#include <hip/hip_runtime.h>

#include "ews_hip.h"
#include "ews_vec.h"

namespace ews {
namespace gscan {

using namespace ews::vec;

constexpr int kSteps = 8;           // of a thread in a tile
constexpr int kWaves = 8;           // of a strip's workgroup
constexpr float kLog2e = 1.44269504088896340736f;

struct Args {
  const void* x;
  const void* g;
  const uint8_t* mask;              // (B, L) or null
  const float* state;               // (B, D) or null: zero
  int64_t xb, xs, gb, gs, mb;       // elements between sequences and steps
  int B, L, D;
  int lanes, shift;                 // of a row of channels; log2
  int tile;                         // steps
  int tiles, seg_tiles, segs;       // of a sequence; of a segment; segments
  int strips;
  float* starts;                    // (B, tiles, D) the state before every tile; or null
  float* ends;                      // (2, segs, B, D) the segments' composed maps
  float* first;                     // (B, D) a copy of state where segments read it: last may be written over it
  void* h;                          // (B, L, D)
  float* last;                      // (B, D)
  const void* dh;                   // (B, L, D) or null
  const float* dlast;               // (B, D) or null
  void* dx;
  void* dg;
  float* dstate;                    // (B, D) or null
};

// V neighbouring numbers as they lie in memory.
template <typename T, int V>
struct Raw {
  T n[V];
};
template <>
struct Raw<bf16, 2> {
  uint32_t w;
};

template <typename T, int V>
__device__ __forceinline__ void widen_raw(const Raw<T, V>& r, float (&x)[V]) {
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = widen(r.n[v]);
}
__device__ __forceinline__ void widen_raw(const Raw<bf16, 2>& r, float (&x)[2]) {
  x[0] = __uint_as_float(r.w << 16);
  x[1] = __uint_as_float(r.w & 0xffff0000u);
}
template <typename T, int V>
__device__ __forceinline__ void narrow_raw(const float (&x)[V], Raw<T, V>& r) {
#pragma unroll
  for (int v = 0; v < V; ++v) r.n[v] = narrow<T>(x[v]);
}
__device__ __forceinline__ void narrow_raw(const float (&x)[2], Raw<bf16, 2>& r) { r.w = pack_bf16(x[0], x[1]); }

// A gate's factor a and what it lets in. exp(-g) is held below infinity, where its product with a is 1 all the same.
template <bool CONVEX>
__device__ __forceinline__ void open(float g, float& a, float& take) {
  if (!CONVEX) {
    a = g;
    take = 1.0f;
    return;
  }
  float y = g * -kLog2e;
  y = y > 126.0f ? 126.0f : y;  // a NaN stays one
  const float e = __builtin_amdgcn_exp2f(y);
  a = __builtin_amdgcn_rcpf(1.0f + e);
  take = e * a;
}

// Where a thread stands: its channels, its place in the tile.
template <int V>
struct Place {
  int b, c, slot, seg, first, end;  // first tile and last + 1 of the segment
  bool live;
  __device__ __forceinline__ explicit Place(const Args& a) {
    const int at = blockIdx.x % (a.strips * a.B);
    seg = blockIdx.x / (a.strips * a.B);
    b = at / a.strips;
    c = ((at % a.strips) * a.lanes + (int)(threadIdx.x & (a.lanes - 1))) * V;
    slot = threadIdx.x >> a.shift;
    live = c < a.D;
    if (!live) c = a.D - V;
    first = seg * a.seg_tiles;
    end = first + a.seg_tiles < a.tiles ? first + a.seg_tiles : a.tiles;
  }
};

// A thread's steps of one array. Steps past the sequence's end read the last one.
template <typename T, int V>
__device__ __forceinline__ void fetch(Raw<T, V> (&r)[kSteps], const void* base, int64_t batch, int64_t step, int b, int c,
                                      int t0, int L) {
  const T* p = (const T*)base + b * batch + c;
  if (t0 + kSteps <= L) {
    p += t0 * step;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) r[i] = *reinterpret_cast<const Raw<T, V>*>(p + i * step);
  } else {
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
      r[i] = *reinterpret_cast<const Raw<T, V>*>(p + (t0 + i < L ? t0 + i : L - 1) * step);
  }
}

// A thread's steps of the mask, a byte each; steps past the sequence's end are off.
__device__ __forceinline__ uint64_t fetch_mask(const Args& a, int b, int t0) {
  if (!a.mask) return ~0ull;
  const uint8_t* m = a.mask + b * a.mb;
  uint64_t w = 0;
  if (t0 + kSteps <= a.L) {
    __builtin_memcpy(&w, m + t0, 8);
  } else {
#pragma unroll
    for (int i = 0; i < kSteps; ++i) w |= (uint64_t)(t0 + i < a.L ? m[t0 + i] : 0) << (8 * i);
  }
  return w;
}

// Bit i: step t0 + i is in the sequence (bit 8 + i: and on the mask).
constexpr uint32_t kWhole = 0xffffu;
__device__ __forceinline__ uint32_t steps_on(const Args& a, uint64_t mask, int t0) {
  const int left = a.L - t0;
  const uint32_t in = left >= kSteps ? 0xffu : left > 0 ? (1u << left) - 1 : 0;
  // bytes that are not 0 to their lowest bit, and those bits side by side
  const uint64_t low = 0x7f7f7f7f7f7f7f7full;
  const uint64_t one = (((mask & low) + low) | mask) >> 7 & 0x0101010101010101ull;
  return in | ((uint32_t)(one * 0x0102040810204080ull >> 56) & in) << 8;
}
static_assert(kSteps == 8, "two bits a step in one word, a byte of the mask each in another");

// A product of convex gates is 0 by underflow alone, but zero times an infinite state, which the steps one by one would
// keep, is NaN. So such products are held at float32's least number: of a finite state that is 2^-149 of it in place of
// less, which is nothing beside float32's roundings unless it was beyond 2^100 (looking for NaN and composing again
// with care took 3 to 5% of strips).
template <bool CONVEX>
__device__ __forceinline__ float above_zero(float a) {
  return CONVEX ? fmaxf(a, 1.40129846e-45f) : a;
}

// (a, b) = (a2, b2) after (a, b).
__device__ __forceinline__ void then(float& a, float& b, float a2, float b2) {
  b = fmaf(a2, b, b2);
  a *= a2;
}

// ------------------------------------------------------------------------------------------------------- the forward
template <typename T, int V, bool CONVEX, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_forward(Args a) {
  constexpr bool kAlone = WAVES == 1;
  __shared__ float2 ends[2][WAVES][64 * V];
  const Place<V> at(a);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = a.lanes;
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = a.state ? a.state[(int64_t)at.b * a.D + at.c + v] : 0.0f;
#pragma unroll 8
  for (int s = 0; s < at.seg; ++s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t e = ((int64_t)s * a.B + at.b) * a.D + at.c + v;
      carry[v] = fmaf(a.ends[e], carry[v], a.ends[(int64_t)a.segs * a.B * a.D + e]);
    }
  Raw<T, V> rx[kSteps], rg[kSteps];
  uint64_t mask;
  auto load = [&](int tile) {
    const int t0 = tile * a.tile + at.slot * kSteps;
    fetch(rx, a.x, a.xb, a.xs, at.b, at.c, t0, a.L);
    fetch(rg, a.g, a.gb, a.gs, at.b, at.c, t0, a.L);
    mask = fetch_mask(a, at.b, t0);
  };
  load(at.first);
  for (int tile = at.first; tile < at.end; ++tile) {
    const int t0 = tile * a.tile + at.slot * kSteps;
    const uint32_t on = steps_on(a, mask, t0);
    const bool whole = __all(on == kWhole);
    float ka[kSteps][V], kb[kSteps][V], A[V], H[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float x[V], g[V];
      widen_raw(rx[i], x);
      widen_raw(rg[i], g);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float take;
        open<CONVEX>(g[v], ka[i][v], take);
        kb[i][v] = take * x[v];
        if (!whole) {
          const bool kept = on & (256u << i);
          ka[i][v] = kept ? ka[i][v] : 1.0f;
          kb[i][v] = kept ? kb[i][v] : 0.0f;
        }
        then(A[v], H[v], ka[i][v], kb[i][v]);
      }
    }
    if (tile + 1 < at.end) load(tile + 1);
    float h[V];
    if (kAlone) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = carry[v];
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) A[v] = above_zero<CONVEX>(A[v]);
      for (int d = row; d < 64; d <<= 1)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a0 = __shfl_up(A[v], d), h0 = __shfl_up(H[v], d);
          if (lane >= d) {
            then(a0, h0, A[v], H[v]);
            A[v] = above_zero<CONVEX>(a0);
            H[v] = h0;
          }
        }
      const int buf = tile & 1;
      if (lane >= 64 - row)
#pragma unroll
        for (int v = 0; v < V; ++v) ends[buf][wave][(lane & (row - 1)) * V + v] = make_float2(A[v], H[v]);
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float state = carry[v];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          if (w == wave) h[v] = state;
          const float2 e = ends[buf][w][(lane & (row - 1)) * V + v];
          state = fmaf(e.x, state, e.y);
        }
        carry[v] = state;
        const float a0 = __shfl_up(A[v], row & 63), h0 = __shfl_up(H[v], row & 63);
        if (lane >= row) h[v] = fmaf(a0, h[v], h0);
      }
    }
    if (a.starts && at.slot == 0 && at.live)
#pragma unroll
      for (int v = 0; v < V; ++v) a.starts[((int64_t)at.b * a.tiles + tile) * a.D + at.c + v] = h[v];
    T* out = (T*)a.h + ((int64_t)at.b * a.L + t0) * a.D + at.c;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = fmaf(ka[i][v], h[v], kb[i][v]);
      Raw<T, V> r;
      narrow_raw(h, r);
      if (at.live && (whole || (on & (1u << i)))) *reinterpret_cast<Raw<T, V>*>(out + (int64_t)i * a.D) = r;
    }
    if (kAlone)
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = h[v];
  }
  if (at.end == a.tiles && at.slot == 0 && at.live)
#pragma unroll
    for (int v = 0; v < V; ++v) a.last[(int64_t)at.b * a.D + at.c + v] = carry[v];
}

// ------------------------------------------------------------------------------------------------------ the backward
template <typename T, int V, bool CONVEX, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_backward(Args a) {
  constexpr bool kAlone = WAVES == 1;
  __shared__ float ends[2][WAVES][3][64 * V];
  const Place<V> at(a);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = a.lanes;
  float carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = a.dlast ? a.dlast[(int64_t)at.b * a.D + at.c + v] : 0.0f;
#pragma unroll 8
  for (int s = a.segs - 1; s > at.seg; --s)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t e = ((int64_t)s * a.B + at.b) * a.D + at.c + v;
      carry[v] = fmaf(a.ends[e], carry[v], a.ends[(int64_t)a.segs * a.B * a.D + e]);
    }
  Raw<T, V> rx[kSteps], rg[kSteps], ru[kSteps];
  uint64_t mask;
  float start[V];
  auto load = [&](int tile) {
    const int t0 = tile * a.tile + at.slot * kSteps;
    fetch(rx, a.x, a.xb, a.xs, at.b, at.c, t0, a.L);
    fetch(rg, a.g, a.gb, a.gs, at.b, at.c, t0, a.L);
    if (a.dh) fetch(ru, a.dh, (int64_t)a.L * a.D, a.D, at.b, at.c, t0, a.L);
    mask = fetch_mask(a, at.b, t0);
#pragma unroll
    for (int v = 0; v < V; ++v) start[v] = a.starts[((int64_t)at.b * a.tiles + tile) * a.D + at.c + v];
  };
  load(at.end - 1);
  for (int tile = at.end - 1; tile >= at.first; --tile) {
    const int t0 = tile * a.tile + at.slot * kSteps;
    const uint32_t on = steps_on(a, mask, t0);
    const bool whole = __all(on == kWhole);
    float ka[kSteps][V], take[kSteps][V], x[kSteps][V], u[kSteps][V], state[V];
#pragma unroll
    for (int v = 0; v < V; ++v) state[v] = start[v];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      float g[V];
      widen_raw(rx[i], x[i]);
      widen_raw(rg[i], g);
      if (a.dh) widen_raw(ru[i], u[i]);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        open<CONVEX>(g[v], ka[i][v], take[i][v]);
        if (!a.dh) u[i][v] = 0.0f;
        if (!whole) {
          const bool kept = on & (256u << i);
          ka[i][v] = kept ? ka[i][v] : 1.0f;
          take[i][v] = kept ? take[i][v] : 0.0f;
          x[i][v] = kept ? x[i][v] : 0.0f;
          u[i][v] = on & (1u << i) ? u[i][v] : 0.0f;
        }
      }
    }
    if (tile > at.first) load(tile - 1);
    float h[V], m[V];
    if (kAlone) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = state[v], m[v] = carry[v];
    } else {
      // A, H: the thread's steps composed; A, M: the same for m, from its last step to its first
      float A[V], H[V], M[V], B[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        A[v] = 1.0f, H[v] = 0.0f, M[v] = 0.0f;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) then(A[v], H[v], ka[i][v], take[i][v] * x[i][v]);
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) M[v] = ka[i][v] * (u[i][v] + M[v]);
        B[v] = A[v] = above_zero<CONVEX>(A[v]);
      }
      for (int d = row; d < 64; d <<= 1)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a0 = __shfl_up(A[v], d), h0 = __shfl_up(H[v], d);
          if (lane >= d) {
            then(a0, h0, A[v], H[v]);
            A[v] = above_zero<CONVEX>(a0);
            H[v] = h0;
          }
          float b0 = __shfl_down(B[v], d), m0 = __shfl_down(M[v], d);
          if (lane + d < 64) {
            then(b0, m0, B[v], M[v]);
            B[v] = above_zero<CONVEX>(b0);
            M[v] = m0;
          }
        }
      // the last slot's (A, H) are its wavefront's, the first's M
      const int buf = tile & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int cell = (lane & (row - 1)) * V + v;
        if (lane >= 64 - row) {
          ends[buf][wave][0][cell] = A[v];
          ends[buf][wave][1][cell] = H[v];
        }
        if (lane < row) ends[buf][wave][2][cell] = M[v];
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int cell = (lane & (row - 1)) * V + v;
        float here = state[v], back = carry[v];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          if (w == wave) h[v] = here;
          here = fmaf(ends[buf][w][0][cell], here, ends[buf][w][1][cell]);
        }
#pragma unroll
        for (int w = WAVES - 1; w >= 0; --w) {
          if (w == wave) m[v] = back;
          back = fmaf(ends[buf][w][0][cell], back, ends[buf][w][2][cell]);
        }
        carry[v] = back;
        const float a0 = __shfl_up(A[v], row & 63), h0 = __shfl_up(H[v], row & 63);
        if (lane >= row) h[v] = fmaf(a0, h[v], h0);
        const float b0 = __shfl_down(B[v], row & 63), m0 = __shfl_down(M[v], row & 63);
        if (lane + row < 64) m[v] = fmaf(b0, m[v], m0);
      }
    }
    float before[kSteps][V];
#pragma unroll
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        before[i][v] = h[v];
        h[v] = fmaf(ka[i][v], h[v], take[i][v] * x[i][v]);
      }
    const int64_t to = ((int64_t)at.b * a.L + t0) * a.D + at.c;
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      float dx[V], dg[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float l = u[i][v] + m[v];
        dx[v] = l * take[i][v];
        dg[v] = CONVEX ? dx[v] * ka[i][v] * (before[i][v] - x[i][v]) : l * before[i][v];
        if (!whole && !(on & (256u << i))) dx[v] = dg[v] = 0.0f;
        m[v] = ka[i][v] * l;
      }
      if (at.live && (whole || (on & (1u << i)))) {
        Raw<T, V> r;
        narrow_raw(dx, r);
        *reinterpret_cast<Raw<T, V>*>((T*)a.dx + to + (int64_t)i * a.D) = r;
        narrow_raw(dg, r);
        *reinterpret_cast<Raw<T, V>*>((T*)a.dg + to + (int64_t)i * a.D) = r;
      }
    }
    if (kAlone)
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = m[v];
  }
  if (a.dstate && at.first == 0 && at.slot == 0 && at.live)
#pragma unroll
    for (int v = 0; v < V; ++v) a.dstate[(int64_t)at.b * a.D + at.c + v] = carry[v];
}

// ---------------------------------------------------------------------------------------------------- segments' maps
// A segment's steps composed (BACK: those of m, from its last step to its first). A slot goes over a stretch of the
// segment by itself; the stretches are joined at the end.
template <typename T, int V, bool CONVEX, bool BACK>
__global__ __launch_bounds__(512) void k_ends(Args a) {
  __shared__ float2 parts[512][V];
  const Place<V> at(a);
  const int slots = 512 >> a.shift;
  const int begin = at.first * a.tile, end = at.end * a.tile < a.L ? at.end * a.tile : a.L;
  const int each = ((end - begin + slots - 1) / slots + kSteps - 1) / kSteps * kSteps;
  const int lo = begin + at.slot * each < end ? begin + at.slot * each : end;
  const int hi = lo + each < end ? lo + each : end;
  float A[V], H[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = 1.0f, H[v] = 0.0f;
  for (int n = 0; n < each; n += kSteps) {
    const int t0 = BACK ? lo + each - kSteps - n : lo + n;  // the whole stretch in eights from its first step on
    if (t0 >= hi) continue;
    Raw<T, V> r[kSteps], rg[kSteps];
    fetch(rg, a.g, a.gb, a.gs, at.b, at.c, t0, a.L);
    if (!BACK) fetch(r, a.x, a.xb, a.xs, at.b, at.c, t0, a.L);
    if (BACK && a.dh) fetch(r, a.dh, (int64_t)a.L * a.D, a.D, at.b, at.c, t0, a.L);
    uint32_t on = steps_on(a, fetch_mask(a, at.b, t0), t0);
    if (t0 + kSteps > hi) on &= ((1u << (hi - t0)) - 1) * 257u;  // steps of the next stretch
    const bool whole = __all(on == kWhole);
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      const int i = BACK ? kSteps - 1 - k : k;
      float x[V], g[V];
      widen_raw(rg[i], g);
      if (!BACK || a.dh) widen_raw(r[i], x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float f, take;
        open<CONVEX>(g[v], f, take);
        if (BACK && !a.dh) x[v] = 0.0f;
        if (!whole) {
          const bool in = on & (1u << i), kept = on & (256u << i);
          f = kept ? f : 1.0f;
          x[v] = (BACK ? in : kept) ? x[v] : 0.0f;
          take = kept ? take : 0.0f;
        }
        if (BACK)
          H[v] = f * (x[v] + H[v]);
        else
          H[v] = fmaf(f, H[v], take * x[v]);
        A[v] = above_zero<CONVEX>(A[v] * f);
      }
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) parts[threadIdx.x][v] = make_float2(A[v], H[v]);
  __syncthreads();
  if (at.slot || !at.live) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.0f, H[v] = 0.0f;
    for (int n = 0; n < slots; ++n) {
      const float2 e = parts[((BACK ? slots - 1 - n : n) << a.shift) + threadIdx.x][v];
      then(A[v], H[v], e.x, e.y);
      A[v] = above_zero<CONVEX>(A[v]);
    }
    const int64_t to = ((int64_t)at.seg * a.B + at.b) * a.D + at.c + v;
    if (!BACK && a.state && at.seg == 0) a.first[to] = a.state[to];
    a.ends[to] = A[v];
    a.ends[(int64_t)a.segs * a.B * a.D + to] = H[v];
  }
}

}  // namespace gscan
}  // namespace ews

namespace {

using namespace ews::gscan;
using ews::vec::bf16;

constexpr int kFill = 192;  // workgroups that give most CUs work

struct SPlan {
  int lanes, shift, waves, tile, tiles, seg_tiles, segs, pairs;  // pairs: two bfloat16 channels a thread
};

int s_ceil(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

int scan_plan(const ews_gated_scan_desc* s, SPlan& p) {
  if (!s) return EWS_ERR_NULL;
  if (s->dtype != EWS_DTYPE_F32 && s->dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->form != EWS_GATED_SCAN_CONVEX && s->form != EWS_GATED_SCAN_LINEAR) return EWS_ERR_OPTION;
  if (s->batch < 1 || s->length < 1 || s->dim < 1 || s->batch > 1 << 20 || s->length > 1 << 28 || s->dim > 1 << 20)
    return EWS_ERR_SHAPE;
  if (s->x_step < 0 || s->gate_step < 0 || s->x_batch < 0 || s->gate_batch < 0 || s->mask_batch < 0)
    return EWS_ERR_SHAPE;
  // The plan asks for sizes and types alone, so that a backward finds the forward's tiles in the residual whatever x's
  // and gate's strides have become; rows of pairs that do not start at whole words are read number by number.
  p.pairs = s->dtype == EWS_DTYPE_BF16 && s->dim % 2 == 0;
  const int cells = p.pairs ? s->dim / 2 : s->dim;  // threads that the channels need
  // threads that walk alone: where sixteen wavefronts a CU can (bfloat16 64 x 512 x 4096 both ways: 437 us, by strips
  // 455; half as many wavefronts: 510, by strips 456), or a sequence is but one or two of their tiles
  if ((int64_t)s->batch * s_ceil(cells, 64) >= 4096 || s->length <= 2 * kSteps) {
    p.waves = 1;
    p.lanes = 64;
    p.shift = 6;
  } else {
    // else eight wavefronts a strip: 64 lanes wide (8 x 2048 x 4096: 231 us, with 32 lanes 242), or 32, a cache line
    // of float32 or of bfloat16 pairs, where those fill the CUs and the wider ones do not
    p.waves = kWaves;
    const int64_t wide = (int64_t)s->batch * s_ceil(cells, 64), narrow = (int64_t)s->batch * s_ceil(cells, 32);
    p.shift = wide < kFill && narrow >= kFill ? 5 : 6;
    while (p.shift > 3 && cells <= 1 << (p.shift - 1)) --p.shift;
    p.lanes = 1 << p.shift;
  }
  p.tile = (64 * p.waves >> p.shift) * kSteps;
  p.tiles = s_ceil(s->length, p.tile);
  p.segs = 1;
  p.seg_tiles = p.tiles;
  const int64_t groups = (int64_t)s->batch * s_ceil(cells, p.lanes);
  if (p.waves > 1 && groups < kFill) {  // segments: two workgroups a CU
    int64_t z = 512 / groups;
    if (z > p.tiles / 2) z = p.tiles / 2;  // each reads x and g once more
    if (z > 1) {
      p.seg_tiles = s_ceil(p.tiles, z);
      p.segs = s_ceil(p.tiles, p.seg_tiles);
    }
  }
  const int64_t blocks = (int64_t)s->batch * s_ceil(s->dim, p.lanes) * p.segs;
  if (blocks > 1 << 25) return EWS_ERR_SHAPE;
  return EWS_OK;
}

Args scan_args(const ews_gated_scan_desc* s, const SPlan& p, bool pairs, const void* x, const void* gate,
               const uint8_t* mask, void* workspace) {
  Args a{};
  a.x = x;
  a.g = gate;
  a.mask = mask;
  a.xb = s->x_batch;
  a.xs = s->x_step;
  a.gb = s->gate_batch;
  a.gs = s->gate_step;
  a.mb = s->mask_batch;
  a.B = s->batch;
  a.L = s->length;
  a.D = s->dim;
  a.lanes = p.lanes;
  a.shift = p.shift;
  a.tile = p.tile;
  a.tiles = p.tiles;
  a.seg_tiles = p.seg_tiles;
  a.segs = p.segs;
  a.strips = s_ceil(s->dim, p.lanes * (pairs ? 2 : 1));
  a.ends = (float*)workspace;
  a.first = a.ends + (int64_t)2 * p.segs * s->batch * s->dim;
  return a;
}

template <typename T, int V, bool CONVEX>
int scan_launch(Args a, const SPlan& p, bool back, hipStream_t st) {
  const dim3 grid((uint32_t)(a.strips * a.B * a.segs));
  if (a.segs > 1) {
    if (back)
      hipLaunchKernelGGL((k_ends<T, V, CONVEX, true>), grid, dim3(512), 0, st, a);
    else
      hipLaunchKernelGGL((k_ends<T, V, CONVEX, false>), grid, dim3(512), 0, st, a);
    if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
    if (a.state) a.state = a.first;
  }
  if (back && p.waves == 1)
    hipLaunchKernelGGL((k_backward<T, V, CONVEX, 1>), grid, dim3(64), 0, st, a);
  else if (back)
    hipLaunchKernelGGL((k_backward<T, V, CONVEX, kWaves>), grid, dim3(64 * kWaves), 0, st, a);
  else if (p.waves == 1)
    hipLaunchKernelGGL((k_forward<T, V, CONVEX, 1>), grid, dim3(64), 0, st, a);
  else
    hipLaunchKernelGGL((k_forward<T, V, CONVEX, kWaves>), grid, dim3(64 * kWaves), 0, st, a);
  return hipGetLastError() == hipSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <bool CONVEX>
int scan_launch(const ews_gated_scan_desc* s, const Args& a, const SPlan& p, bool pairs, bool back, hipStream_t st) {
  if (s->dtype == EWS_DTYPE_F32) return scan_launch<float, 1, CONVEX>(a, p, back, st);
  return pairs ? scan_launch<bf16, 2, CONVEX>(a, p, back, st) : scan_launch<bf16, 1, CONVEX>(a, p, back, st);
}

int scan_launch(const ews_gated_scan_desc* s, const Args& a, const SPlan& p, bool pairs, bool back, hipStream_t st) {
  return s->form == EWS_GATED_SCAN_CONVEX ? scan_launch<true>(s, a, p, pairs, back, st)
                                          : scan_launch<false>(s, a, p, pairs, back, st);
}

bool words(const void* p) { return (uintptr_t)p % 4 == 0; }

// Whether x's and gate's steps start at whole words.
bool word_steps(const ews_gated_scan_desc* s, const void* x, const void* gate) {
  return s->x_step % 2 == 0 && s->gate_step % 2 == 0 && s->x_batch % 2 == 0 && s->gate_batch % 2 == 0 && words(x) &&
         words(gate);
}

}  // namespace

extern "C" {

size_t ews_gated_scan_residual_bytes(const ews_gated_scan_desc* desc) {
  SPlan p;
  if (scan_plan(desc, p) != EWS_OK) return 0;
  return (size_t)desc->batch * p.tiles * desc->dim * 4;
}

size_t ews_gated_scan_workspace_bytes(const ews_gated_scan_desc* desc) {
  SPlan p;
  if (scan_plan(desc, p) != EWS_OK || p.segs == 1) return 0;
  return (size_t)(2 * p.segs + 1) * desc->batch * desc->dim * 4;
}

int ews_gated_scan_forward(const ews_gated_scan_desc* desc, const void* x, const void* gate, const uint8_t* mask,
                           const float* state, void* out, float* last, void* residual, void* workspace,
                           ews_stream_t stream) {
  SPlan p;
  const int rc = scan_plan(desc, p);
  if (rc != EWS_OK) return rc;
  if (!x || !gate || !out || !last || (p.segs > 1 && !workspace)) return EWS_ERR_NULL;
  const bool pairs = p.pairs && word_steps(desc, x, gate) && words(out);
  Args a = scan_args(desc, p, pairs, x, gate, mask, workspace);
  a.state = state;
  a.h = out;
  a.last = last;
  a.starts = (float*)residual;
  return scan_launch(desc, a, p, pairs, false, (hipStream_t)stream);
}

int ews_gated_scan_backward(const ews_gated_scan_desc* desc, const void* x, const void* gate, const uint8_t* mask,
                            const void* residual, const void* grad_out, const float* grad_last, void* grad_x,
                            void* grad_gate, float* grad_state, void* workspace, ews_stream_t stream) {
  SPlan p;
  const int rc = scan_plan(desc, p);
  if (rc != EWS_OK) return rc;
  if (!x || !gate || !residual || !grad_x || !grad_gate || (p.segs > 1 && !workspace)) return EWS_ERR_NULL;
  const bool pairs =
      p.pairs && word_steps(desc, x, gate) && words(grad_out) && words(grad_x) && words(grad_gate);
  Args a = scan_args(desc, p, pairs, x, gate, mask, workspace);
  a.starts = (float*)residual;
  a.dh = grad_out;
  a.dlast = grad_last;
  a.dx = grad_x;
  a.dg = grad_gate;
  a.dstate = grad_state;
  return scan_launch(desc, a, p, pairs, true, (hipStream_t)stream);
}

}  // extern "C"
