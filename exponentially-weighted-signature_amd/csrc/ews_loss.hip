// Softmax cross entropy of a language model's head on MI355X (gfx950), with its gradients, without the logits in
// memory.
//
//   z[n, v] = h[n] . W[v] + b[v]        l[n] = log sum_v exp z[n, v] - z[n, t_n]
//   dz[n, v] = g_n (exp(z[n, v]) / sum_u exp(z[n, u]) - [v = t_n])
//   dh = dz W        dW = dz^T h        db[v] = sum_n dz[n, v]
//
// Rows whose target is the ignored index are taken out first (k_prepare), so nothing they hold is read and they cost
// nothing; their loss and their row of dh are zero. A target outside the vocabulary makes its row's loss NaN.
//
// The head's three products are 2 N V H operations each and run on the matrix cores (ews_tiles.h); they bound the
// call for all but the smallest N. What is between them:
//
//   k_logits  a tile of z in registers; every wavefront takes the maximum m and the sum of exp(z - m) of its slab of
//             the vocabulary for each of its rows. A training call also writes exp(z - m), for bfloat16 inputs as 16
//             bits of (m - z) log2 e in steps of 1/512: off by less than 2^-10.5 of exp(z - m) whatever its size, a
//             fifth of what dz loses in bfloat16 afterwards (bfloat16 itself would lose as much again, and a logit
//             rounded to it more than its probability).
//   k_join    joins a row's slabs: the row's maximum M and sum, its loss.
//   k_dz      dz = exp(z - m) exp(m - M) g / sum, in place; the target's entry from its own float32
//             logit, so a target of probability near one loses nothing. The mean's factor stays out of it: most
//             targets' entries are near -1, which bfloat16 holds, while their common factor's rounding would scale
//             the whole gradient.
//   k_grad    dh and dW, sums in float32, reading W, h and dz as they are, with k along their rows. Few tiles are
//             split over k and joined in order by k_reduce.
//
// 8192 rows (a tenth of them ignored), H=2048, V=32000, bfloat16, in a trace of ten calls: k_logits 0.94 ms (1.0
// PFLOP/s), k_dz 0.20 (4.6 TB/s), dh and dW 0.83 each (1.16), all else 0.035; calls in a row, untraced, take 2.69 ms in
// all. One row by V=100003, H=4096: k_logits 0.15 ms, 5.6 TB/s of W.
//
// The probabilities are kept for kChunkBytes of rows at a time; dW is summed over the chunks in float32. Nothing is
// added with atomics: the same inputs give the same bits.
//
// Float32 inputs are multiplied as three bfloat16 planes (ews_tiles.h): float32's accuracy at the bfloat16 rate over
// six, against one sixteenth for the float32 matrix instructions.
#include <hip/hip_runtime.h>

#include "ews_hip.h"
#include "ews_tiles.h"
#include "ews_tiles32.h"
#include "ews_vec.h"

namespace ews {
namespace loss {

using namespace ews::vec;
using namespace ews::tiles;

typedef Tile<2, 4, 4, 2> Large;   // 256 x 256, eight wavefronts
typedef Tile<2, 2, 2, 2> Medium;  // 128 x 128, four wavefronts
typedef Tile<4, 1, 2, 1> Flat;    // 256 x 32, four wavefronts: few rows
template <int BYTES>
using Few32 = Tile32<1, BYTES>;   // 128 x 32 and 128 x 64, float32 W read as it is: few rows
template <int BYTES>
using More32 = Tile32<2, BYTES>;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kOctaves = 128.0f;  // 16-bit logarithms: 65535 is 2^-128 and stands for a probability of 0

struct Rows {
  int* map;       // (N) the kept rows' places, in order
  int* target;    // (N) their targets; -1 outside the vocabulary
  int* kept;      // [0]: how many
  float* scale;   // [0]: 1 / max(kept, 1) for the mean, 1 for the sum
};

// Logits are kept in units of a factor of two: z log2 e.
struct Stats {
  float2* slab;   // (slabs, chunk rows) maximum and sum of 2^(z - maximum) of one wavefront's slab
  float* zt;      // (N) the target's logit
  float* top;     // (N) the row's maximum
  float* inv;     // (N) one over its sum
  float* loss;    // (N) the kept rows' losses
};

// ------------------------------------------------------------------------------------------------- rows and planes
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
__global__ __launch_bounds__(256) void k_pack(PackArgs a) {
  pack_eight<T>(a, (int64_t)blockIdx.x * 256 + threadIdx.x);
}

// ------------------------------------------------------------------------------------------------------ preparation
struct PrepareArgs {
  const int64_t* targets;
  int n, vocab, padded, mean, H;
  int64_t ignore;
  Rows rows;
  float* loss_rows;        // (N) or null: the ignored rows' zeros
  const void* bias;        // or null
  int bias_bf16;
  float* bias_out;         // (padded)
  void* grad_hidden;       // or null: the ignored rows' zeros
  int each, kept_blocks;   // rows that a workgroup lists, and those workgroups
  int bias_blocks, ignored_blocks;
  PackArgs weight;         // packed by the further workgroups
  PackArgs few;            // the hidden rows, where the first workgroup packs them too; dst null: k_pack does
};

// Lists the kept ones of `each` rows. A workgroup counts those of all rows before its own by itself (the targets stay
// in L2), its wavefronts those of their own stretches, and so every one knows where its first goes. 131072 rows by 16
// workgroups: 21 us; 100000 by one: 43.
__device__ __forceinline__ void keep_rows(const PrepareArgs& a) {
  __shared__ int counts[16], earlier[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int start = (int)blockIdx.x * a.each, end = start + a.each < a.n ? start + a.each : a.n;
  const int part = (end - start + 1023) / 1024 * 64;
  const int lo = start + wave * part < end ? start + wave * part : end;
  const int hi = lo + part < end ? lo + part : end;
  int before = 0, m = 0;
  for (int i = tid; i < start; i += 8 * 1024) {  // `each` is a multiple of that where there is more than one workgroup
    int64_t t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = a.targets[i + k * 1024];
#pragma unroll
    for (int k = 0; k < 8; ++k) before += t[k] != a.ignore;
  }
#pragma unroll 8
  for (int i = lo + lane; i < hi; i += 64) m += a.targets[i] != a.ignore;
#pragma unroll
  for (int s = 32; s; s >>= 1) {
    m += __shfl_xor(m, s);
    before += __shfl_xor(before, s);
  }
  if (lane == 0) {
    counts[wave] = m;
    earlier[wave] = before;
  }
  __syncthreads();
  int total = 0, at = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < wave) at += counts[w];
    at += earlier[w];
    total += counts[w] + earlier[w];
  }
#pragma unroll 4
  for (int i0 = lo; i0 < hi; i0 += 64) {
    const int i = i0 + lane;
    const int64_t t = i < hi ? a.targets[i] : a.ignore;
    const bool keep = t != a.ignore;
    const uint64_t kept = __ballot(keep);
    if (keep) {
      const int to = at + __popcll(kept & ((1ull << lane) - 1ull));
      a.rows.map[to] = i;
      a.rows.target[to] = t >= 0 && t < a.vocab ? (int)t : -1;
    } else if (i < hi && a.loss_rows) {
      a.loss_rows[i] = 0.0f;
    }
    at += __popcll(kept);
  }
  if (tid == 0 && end == a.n) {
    a.rows.kept[0] = total;
    a.rows.scale[0] = a.mean ? 1.0f / (float)(total > 0 ? total : 1) : 1.0f;
  }
}

// The bias in float32 times log2 e, -inf past the vocabulary: those columns of a tile then have no weight in any row. A
// finite bias stays finite (a mask of the type's lowest value is not -inf: a row of nothing else is uniform).
__device__ __forceinline__ void scale_bias(const PrepareArgs& a, int v) {
  if (v >= a.padded) return;
  float b = -__builtin_inff();
  if (v < a.vocab) {
    const float x = !a.bias ? 0.0f : a.bias_bf16 ? widen(((const bf16*)a.bias)[v]) : ((const float*)a.bias)[v];
    b = x * kLog2e;
    if (__builtin_isinf(b) && !__builtin_isinf(x)) b = copysignf(3.402823466e+38f, x);
  }
  a.bias_out[v] = b;
}

// What needs nothing of the others, in one launch: the first workgroups list the kept rows (one packs a few), some
// write the bias, some (16 rows each) zero the ignored rows of dh, the others pack W where it is not read as it is.
template <typename T>
__global__ __launch_bounds__(1024) void k_prepare(PrepareArgs a) {
  if ((int)blockIdx.x < a.kept_blocks) {
    keep_rows(a);
    if (!a.few.dst) return;  // else there is one such workgroup
    __threadfence_block();
    __syncthreads();  // the list is this workgroup's own
    const int64_t packs = (int64_t)a.few.dst_rows * (a.few.ld / 8);
    for (int64_t at = threadIdx.x; at < packs; at += 1024) pack_eight<T>(a.few, at);
    return;
  }
  const int b = blockIdx.x - a.kept_blocks;
  if (b < a.bias_blocks) return scale_bias(a, b * 1024 + threadIdx.x);
  if (b >= a.bias_blocks + a.ignored_blocks)
    return pack_eight<T>(a.weight, (int64_t)(b - a.bias_blocks - a.ignored_blocks) * 1024 + threadIdx.x);
  const int row = (b - a.bias_blocks) * 16 + (threadIdx.x >> 6);
  if (row >= a.n || a.targets[row] != a.ignore) return;
  for (int c = threadIdx.x & 63; c < a.H; c += 64) ((T*)a.grad_hidden)[(int64_t)row * a.H + c] = narrow<T>(0.0f);
}

// ------------------------------------------------------------------------------------------------------ the logits
struct LogitArgs {
  Operand W, X;
  Operand32 W32;          // float32 W where it is read as it is
  int ti, tj;             // tiles along the vocabulary and along the chunk's rows
  int kblocks;
  int c0, chunk;          // the chunk's first row, its rows
  const float* bias;
  Rows rows;
  Stats st;
  void* prob;             // exp(z - m) (chunk, ldp): a 16-bit logarithm, or float32 where there are three planes
  int64_t ldp;
};

// A product of one stage needs no second half: more workgroups share a CU.
template <class T, int PAIRS>
__host__ __device__ constexpr int lds_bytes(int kblocks) {
  if constexpr (PAIRS == 1) {
    if (kblocks == 1) return T::kLdsBytesOne;
  }
  return T::kLdsBytes;
}

// PAIRS: 1, kPairs for planes, or 0 for float32 W. KEEP: 0 the loss alone, 1 also 16-bit logarithms, 2 also float32
// probabilities.
template <class T, int PAIRS, int KEEP>
__global__ __launch_bounds__(T::kThreads, T::kWaves) void k_logits(LogitArgs a) {
  extern __shared__ char lds[];
  int it, jt;
  tile_of(blockIdx.x, a.ti, a.tj, it, jt);
  const int i0 = it * T::I, j0 = jt * T::J;
  const int live = a.rows.kept[0] - a.c0 < a.chunk ? a.rows.kept[0] - a.c0 : a.chunk;
  if (j0 >= live) return;
  // the epilogue's operands, where it need not wait for them
  float* tile_bias = reinterpret_cast<float*>(lds + lds_bytes<T, PAIRS>(a.kblocks));
  int* tile_target = reinterpret_cast<int*>(tile_bias + T::I);
  for (int t = threadIdx.x; t < T::I + T::J; t += T::kThreads) {
    if (t < T::I)
      tile_bias[t] = a.bias[i0 + t];
    else
      tile_target[t - T::I] = j0 + t - T::I < live ? a.rows.target[a.c0 + j0 + t - T::I] : -1;
  }
  f32x16 acc[T::TI][T::TJ];
  if constexpr (PAIRS == 0)
    product32<T, false>(a.W32, a.X, i0, j0 + a.c0, 0, a.kblocks, lds, acc);
  else
    product<T, PAIRS, false, false>(a.W, a.X, i0, j0 + a.c0, 0, a.kblocks, lds, acc);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wi = wave % T::WI, wj = wave / T::WI;
  const int r32 = lane & 31, half = lane >> 5;
  const int ibase = i0 + wi * T::kSlab;
  const float* bias = tile_bias + wi * T::kSlab + half * 4;
#pragma unroll
  for (int b = 0; b < T::TJ; ++b) {
    const int j = j0 + (wj * T::TJ + b) * 32 + r32;
    float m = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < T::TI; ++t)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 add = *reinterpret_cast<const f32x4*>(bias + t * 32 + g * 8);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float z = fmaf(acc[t][b][4 * g + q], kLog2e, add[q]);
          acc[t][b][4 * g + q] = z;
          m = fmaxf(m, z);
        }
      }
    m = fmaxf(m, __shfl_xor(m, 32));
    // the target's logit, from the one lane that holds it
    const int want = tile_target[(wj * T::TJ + b) * 32 + r32] - ibase;
    const bool mine = want >= 0 && want < T::kSlab && ((want >> 2) & 1) == half;
    if (__any(mine)) {
      float zt = 0.0f;
#pragma unroll
      for (int t = 0; t < T::TI; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * 32 + 8 * (r / 4) + 4 * half + r % 4 == want) zt = acc[t][b][r];
      if (mine) a.st.zt[a.c0 + j] = zt;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;  // a slab of -inf alone has the sum 0
    float s = 0.0f;
#pragma unroll
    for (int t = 0; t < T::TI; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float y = acc[t][b][r] - ref;
        const float e = __builtin_amdgcn_exp2f(y);
        s += e;
        if (KEEP == 1) acc[t][b][r] = y * (-1.0f / kOctaves);
        if (KEEP == 2) acc[t][b][r] = e;
      }
    s += __shfl_xor(s, 32);
    if (half == 0 && j < live) a.st.slab[(int64_t)(it * T::WI + wi) * a.chunk + j] = make_float2(m, s);
    if (KEEP == 1) {
      rows_of<T, uint16_t>(lds, acc, b, [&](int jrow, int i, const u32x4& w) {
        const int j = j0 + jrow;
        if (j < live && i0 + i < a.ldp) *reinterpret_cast<u32x4*>((uint16_t*)a.prob + j * a.ldp + i0 + i) = w;
      });
    } else if (KEEP == 2) {
      rows_of<T, float>(lds, acc, b, [&](int jrow, int i, const u32x4& w) {
        const int j = j0 + jrow;
        if (j < live && i0 + i < a.ldp) *reinterpret_cast<u32x4*>((float*)a.prob + j * a.ldp + i0 + i) = w;
      });
    }
  }
}

// Maximum and sum of two parts of a row.
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  s = s * __builtin_amdgcn_exp2f(m - ref) + s2 * __builtin_amdgcn_exp2f(m2 - ref);
  m = top;
}

// ROWS rows a workgroup, the other threads along the slabs; joined as a tree.
template <int ROWS>
__global__ __launch_bounds__(1024) void k_join(Stats st, Rows rows, int slabs, int c0, int chunk, float* loss_rows) {
  constexpr int kGroups = 1024 / ROWS;
  __shared__ float ms[1024], ss[1024];
  const int tid = threadIdx.x, group = tid / ROWS;
  const int live = rows.kept[0] - c0 < chunk ? rows.kept[0] - c0 : chunk;
  const int j = blockIdx.x * ROWS + tid % ROWS;
  if (blockIdx.x * ROWS >= live) return;
  float m = -__builtin_inff(), s = 0.0f;
  if (j < live) {
#pragma unroll 4
    for (int k = group; k < slabs; k += kGroups) {
      const float2 x = st.slab[(int64_t)k * chunk + j];
      join(m, s, x.x, x.y);
    }
  }
#pragma unroll
  for (int g = kGroups / 2; g; g >>= 1) {
    ms[tid] = m;
    ss[tid] = s;
    __syncthreads();
    if (group < g) join(m, s, ms[tid + g * ROWS], ss[tid + g * ROWS]);
    __syncthreads();
  }
  if (group || j >= live) return;
  const int row = c0 + j;
  st.top[row] = m;
  st.inv[row] = 1.0f / s;
  const float l = rows.target[row] < 0 ? __builtin_nanf("") : logf(s) + (m - st.zt[row]) * kLn2;
  st.loss[row] = l;
  if (loss_rows) loss_rows[rows.map[row]] = l;
}

// The sum or mean of the kept rows' losses, by one workgroup of up to 1024 threads.
__device__ __forceinline__ void total_loss(const Stats& st, const Rows& rows, float* out) {
  __shared__ double part[16];
  double s = 0.0;
  const int n = rows.kept[0], threads = blockDim.x;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += threads) s += (double)st.loss[i];
#pragma unroll
  for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = 0.0;
  for (int w = 0; w < threads / 64; ++w) s += part[w];
  out[0] = (float)(s * (double)rows.scale[0]);
}

__global__ __launch_bounds__(1024) void k_total(Stats st, Rows rows, float* out) { total_loss(st, rows, out); }

// ---------------------------------------------------------------------------------------------------------- dz
struct DzArgs {
  Rows rows;
  Stats st;
  const float* upstream;  // (N) or null: 1 (k_grad applies the reduction's factor)
  int c0, chunk, slab;
  void* prob;
  int64_t ld;             // the vocabulary padded to a multiple of 64
  uint16_t* dz;           // planes (chunk, ld): in bfloat16 the first is prob itself; zero rows up to a multiple of 64
  int64_t plane;
  float* bias;            // (ceil(chunk / each), ld) sums over the rows; may be null
  int each;               // rows a workgroup goes over, one wavefront a row, 512 columns wide
  int lanes;              // narrow: so many lanes a row, 64 / lanes rows a wavefront; a power of two
  float* loss;            // or null: the call's loss, by one further workgroup
};

// NP planes: 3 of float32 inputs, 1 or (few rows) 2 of bfloat16 ones. NARROW: a row fills half a wavefront at most, so
// several rows share one (131072 rows by V=8: 94 -> 38 us).
template <int NP, bool NARROW>
__global__ __launch_bounds__(256) void k_dz(DzArgs a) {
  if (blockIdx.x * 512 >= a.ld) {
    if (blockIdx.y == 0) total_loss(a.st, a.rows, a.loss);
    return;
  }
  __shared__ float part[4][64][9];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lanes = NARROW ? a.lanes : 64, abreast = NARROW ? 64 / lanes : 1;
  const int v = NARROW ? (lane & (lanes - 1)) * 8 : (blockIdx.x * 64 + lane) * 8;
  const int live = a.rows.kept[0] - a.c0 < a.chunk ? a.rows.kept[0] - a.c0 : a.chunk;
  const int padded = NP == 2 ? a.chunk : (live + 63) / 64 * 64;
  const bool in = v < a.ld;
  const int slab = in ? v / a.slab : 0;
  const int r0 = blockIdx.y * a.each, r1 = r0 + a.each < padded ? r0 + a.each : padded;
  float sums[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) sums[q] = 0.0f;
  for (int j = NARROW ? r0 + wave * abreast + lane / lanes : r0 + wave; j < r1; j += 4 * abreast) {
    float x[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = 0.0f;
    if (j < live && in) {
      const int row = a.c0 + j;
      const int t = a.rows.target[row];
      const float top = a.st.top[row], inv = a.st.inv[row];
      const float g = a.upstream ? a.upstream[a.rows.map[row]] : 1.0f;
      const float m = a.st.slab[(int64_t)slab * a.chunk + j].x;
      const float f = t < 0 ? __builtin_nanf("") : __builtin_amdgcn_exp2f(m - top) * inv * g;
      if (NP != 3) {
        const u32x4 w = *reinterpret_cast<const u32x4*>((const uint16_t*)a.prob + j * a.ld + v);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t y = (w[q >> 1] >> (16 * (q & 1))) & 0xffffu;
          x[q] = y == 65535u ? 0.0f * f : __builtin_amdgcn_exp2f((float)y * (-kOctaves / 65535.0f)) * f;
        }
      } else {
        Pack<float, 4> lo, hi;
        lo.load((const float*)a.prob + j * a.ld + v);
        hi.load((const float*)a.prob + j * a.ld + v + 4);
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = (q < 4 ? lo.get(q) : hi.get(q - 4)) * f;
      }
      if (t >= v && t < v + 8) {
        const float own = (__builtin_amdgcn_exp2f(a.st.zt[row] - top) * inv - 1.0f) * g;
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = t == v + q ? own : x[q];
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) sums[q] += x[q];
    }
    if (!in) continue;
    if (NP != 3) {
      Pack<bf16, 8> p;
      p.set(x);
      p.store((bf16*)a.dz + j * a.ld + v);
      if (NP == 2) {
#pragma unroll
        for (int q = 0; q < 8; ++q) x[q] = __builtin_isfinite(p.get(q)) ? x[q] - p.get(q) : 0.0f;
        p.set(x);
        p.store((bf16*)a.dz + a.plane + j * a.ld + v);
      }
    } else {
      uint16_t p[8][3];
#pragma unroll
      for (int q = 0; q < 8; ++q) planes(x[q], p[q]);
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = (uint32_t)p[2 * q][k] | ((uint32_t)p[2 * q + 1][k] << 16);
        *reinterpret_cast<u32x4*>(a.dz + k * a.plane + j * a.ld + v) = w;
      }
    }
  }
  if (!a.bias) return;
#pragma unroll
  for (int q = 0; q < 8; ++q) part[wave][lane][q] = sums[q];
  __syncthreads();
  for (int c = threadIdx.x; c < 8 * lanes; c += 256) {
    const int col = blockIdx.x * 512 + c;
    if (col >= a.ld) break;
    float s = 0.0f;
    for (int r = 0; r < 64; r += lanes)
#pragma unroll
      for (int w = 0; w < 4; ++w) s += part[w][r + (c >> 3)][c & 7];
    a.bias[(int64_t)blockIdx.y * a.ld + col] = s;
  }
}

// The bias's gradient: k_dz's sums over rows, added to those of the chunks before; the last chunk writes it. 64 columns
// a workgroup, its sixteen wavefronts a contiguous part of the sums each (4096 of them by V=200: 6 us, by one thread a
// column 44).
template <typename T>
__global__ __launch_bounds__(1024) void k_dbias(const float* part, int parts, int64_t ld, int vocab, float* sum,
                                                int add, const float* factor, T* out) {
  __shared__ float joined[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v = blockIdx.x * 64 + lane;
  const int each = (parts + 15) / 16, p1 = (wave + 1) * each < parts ? (wave + 1) * each : parts;
  float s = 0.0f;
  if (v < vocab) {
#pragma unroll 8
    for (int p = wave * each; p < p1; ++p) s += part[p * ld + v];
  }
  joined[wave][lane] = s;
  __syncthreads();
  if (wave || v >= vocab) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) s += joined[w][lane];
  s = (factor ? s * factor[0] : s) + (add ? sum[v] : 0.0f);
  if (out)
    out[v] = narrow<T>(s);
  else
    sum[v] = s;
}

// ------------------------------------------------------------------------------------------------------ the gradients
struct GradArgs {
  Operand P, Q;
  Operand32 P32;          // float32 W where it is read as it is
  int ti, tj, splits;
  int kblocks, per;       // k blocks, and those of one split
  int by_rows;            // 1: k is the chunk's kept rows (dW); 0: the result's rows are (dh)
  int twice;              // dW of few rows: k is the rows of both planes of dz, all of them
  int c0, chunk;
  Rows rows;
  int I, J;               // the result's columns and (where by_rows) rows
  float* part;            // (splits, J or chunk, I) where splits > 1
  float* sum;             // float32 sums over the chunks, or null
  int add;                // sum holds those of earlier chunks
  void* out;              // the result, or null before the last chunk
  int wide;               // the result's rows start at multiples of 16 bytes and hold whole eights
  const float* factor;    // of every result; null: 1
};

// Eight consecutive results of result row `row`, from column i on; all in the row, at a multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ void finish(const GradArgs& a, int64_t row, int i, const Eight& e) {
  const int64_t at = row * a.I + i;
  const float f = a.factor ? a.factor[0] : 1.0f;
  float y[8];
#pragma unroll
  for (int q = 0; q < 8; ++q) y[q] = e.x[q] * f + (a.add ? a.sum[at + q] : 0.0f);
  if (!a.out) {
#pragma unroll
    for (int q = 0; q < 8; ++q) a.sum[at + q] = y[q];
    return;
  }
#pragma unroll
  for (int q = 0; q < 8; q += kWide<T>) {
    Pack<T, kWide<T>> p;
    p.set(y + q);
    p.store_past((T*)a.out + at + q);
  }
}

// One result.
template <typename T>
__device__ __forceinline__ void finish(const GradArgs& a, int64_t row, int i, const One& e) {
  const int64_t at = row * a.I + i;
  const float y = e.x * (a.factor ? a.factor[0] : 1.0f) + (a.add ? a.sum[at] : 0.0f);
  if (a.out)
    ((T*)a.out)[at] = narrow<T>(y);
  else
    a.sum[at] = y;
}

// Results of a split, kept for k_reduce.
__device__ __forceinline__ void keep(float* to, const Eight& e) {
  Pack<float, 4> lo, hi;
  lo.set(e.x);
  hi.set(e.x + 4);
  lo.store(to);
  hi.store(to + 4);
}
__device__ __forceinline__ void keep(float* to, const One& e) { *to = e.x; }

// ROWS: dW, whose k is the chunk's kept rows and whose operands are both turned; else dh, whose rows they are.
template <class T, int PAIRS, bool ROWS, typename O>
__global__ __launch_bounds__(T::kThreads, T::kWaves) void k_grad(GradArgs a) {
  extern __shared__ char lds[];
  const int split = blockIdx.y;
  int it, jt;
  tile_of(blockIdx.x, a.ti, a.tj, it, jt);
  const int i0 = it * T::I, j0 = jt * T::J;
  int live = a.rows.kept[0] - a.c0 < a.chunk ? a.rows.kept[0] - a.c0 : a.chunk;
  live = live > 0 ? live : 0;
  const int nj = ROWS ? a.J : live;
  if (j0 >= nj) return;
  int kb0 = split * a.per, kb1 = kb0 + a.per < a.kblocks ? kb0 + a.per : a.kblocks;
  if (ROWS && !a.twice && kb1 > (live + 63) / 64) kb1 = (live + 63) / 64;
  f32x16 acc[T::TI][T::TJ];
  if constexpr (PAIRS == 0)
    product32<T, true>(a.P32, a.Q, i0, j0, kb0, kb1, lds, acc);
  else
    product<T, PAIRS, true, ROWS>(a.P, a.Q, i0, j0, kb0, kb1, lds, acc);
  auto rows = [&](auto each) {
    using W = decltype(each);
#pragma unroll
    for (int b = 0; b < T::TJ; ++b)
      rows_of<T, W>(lds, acc, b, [&](int jrow, int icol, const W& e) {
        const int j = j0 + jrow, i = i0 + icol;
        if (j >= nj || i >= a.I) return;
        if (a.splits > 1)
          keep(a.part + ((int64_t)split * (ROWS ? a.J : a.chunk) + j) * a.I + i, e);
        else
          finish<O>(a, ROWS ? j : a.rows.map[a.c0 + j], i, e);
      });
  };
  // rows of other lengths are written one number a lane: 64 neighbours at a time, not eight apart
  if (a.wide)
    rows(Eight{});
  else
    rows(One{});
}

// The splits' results added in order. Many splits: 32 results a workgroup, its eight groups of lanes a contiguous part
// of the splits each, joined in LDS.
template <typename O>
__global__ __launch_bounds__(256) void k_reduce(GradArgs a) {
  __shared__ float parts[8][32];
  const int live = a.rows.kept[0] - a.c0 < a.chunk ? a.rows.kept[0] - a.c0 : a.chunk;
  const int nj = a.by_rows ? a.J : live;
  const int64_t stride = (int64_t)(a.by_rows ? a.J : a.chunk) * a.I;
  const int64_t at = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
  const int group = threadIdx.x >> 5;
  const bool in = at < (int64_t)nj * a.I;
  const int per = (a.splits + 7) / 8;
  const int s0 = group * per, s1 = s0 + per < a.splits ? s0 + per : a.splits;
  float x = 0.0f;
  if (in) {
#pragma unroll 8
    for (int s = s0; s < s1; ++s) x += a.part[s * stride + at];
  }
  parts[group][threadIdx.x & 31] = x;
  __syncthreads();
  if (group || !in) return;
#pragma unroll
  for (int g = 1; g < 8; ++g) x += parts[g][threadIdx.x];
  const int64_t j = at / a.I;
  finish<O>(a, a.by_rows ? j : a.rows.map[a.c0 + j], (int)(at - j * a.I), One{x});
}

// Few splits: a thread adds one result's (W: One) or, where rows are wide, eight results'.
template <typename O, typename W>
__global__ __launch_bounds__(256) void k_reduce_few(GradArgs a) {
  constexpr int kEach = sizeof(W) / 4;
  const int live = a.rows.kept[0] - a.c0 < a.chunk ? a.rows.kept[0] - a.c0 : a.chunk;
  const int nj = a.by_rows ? a.J : live;
  const int64_t stride = (int64_t)(a.by_rows ? a.J : a.chunk) * a.I;
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * kEach;
  if (at >= (int64_t)nj * a.I) return;
  float x[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) x[q] = 0.0f;
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) {
    const float* from = a.part + s * stride + at;
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
  W w;
  __builtin_memcpy(&w, x, sizeof(w));
  const int64_t j = at / a.I;
  finish<O>(a, a.by_rows ? j : a.rows.map[a.c0 + j], (int)(at - j * a.I), w);
}

}  // namespace loss
}  // namespace ews

namespace {

using namespace ews::loss;

// Rows kept at a time: exp(z - m), and dz in its place (float32: dz in three planes beside it), of as many as fit here.
constexpr int64_t kChunkBytes = (int64_t)2 << 30;
// float32 W is read as it is for up to so many rows or logits, else packed into planes first. H=2048 V=30000, packing,
// logits and dh: N=128 0.25 ms as it is, 0.51 packed; N=256 0.50 and 0.54. Packing and logits alone, H=1772 V=45646:
// N=260 0.34 and 0.61, N=400 0.50 and 0.67; H=1024 V=32000: N=520 0.26 and 0.32, N=800 0.38 and 0.35. Few logits give
// few tiles, which six products a stage serve better: packing, logits, dh and dW of N=645 H=3904 V=1037 0.22 and 0.31
// ms, of N=2000 H=1024 V=1000 0.11 and 0.12, of N=3000 H=333 V=2000 0.13 and 0.13.
constexpr int kFewRows32 = 512;
constexpr int64_t kFewLogits32 = 1 << 22;
// A call without gradients keeps eight bytes for every row's slabs (64 of the vocabulary at least) of as many rows as
// fit here. Float32 W read as it is has slabs of 32, but few rows or logits: half as much at most.
constexpr int64_t kScoreBytes = (int64_t)256 << 20;

// Stages below which a 128 x 128 tile is no slower (6 stages: 86 us for 94), its CUs better shared.
constexpr int kLongProduct = 8;

// Splits that one thread adds: two of 2000 x 256 by 32000 13 us (eight groups of lanes: 60), eight of 4095 x 512 13
// (36).
constexpr int kFewSplits = 8;

// Up to so many rows of bfloat16, dz is kept in two planes: where few rows add up, the rounding of dz to eight bits
// (most of it that of the targets' entries, g (p - 1)) does not average out. Against the results' own rounding alone,
// dh and dW are up to 2.5 times as far off at 2 rows and 1.8 at 16 with one plane, 1.0 with two; from 256 rows on 1.4
// to 1.5. Where g stays out of dz (the mean and the sum) the targets' entries are near -1 and lose less: up to 2.2
// times at 2 rows, 1.4 at 16. The planes lie one behind the other, and so do two copies of h: dW's k is twice the rows,
// and dh takes two products a stage.
constexpr int kFewRowsNone = 256, kFewRowsMean = 16;

enum Kind { kLarge, kMedium, kFlat, kFew32, kMore32 };

struct Product {
  Kind kind;
  int ti, tj, tile_i, tile_j, slab, splits, per, kblocks, pairs;
};

struct LPlan {
  int N, H, V, np;
  int64_t Hp, Vp, Np, chunk;
  int chunks, slabs, bias_pad, dz_rows;
  bool train, packed, as_is, twice;
  Product logits, dh, dw;
  size_t map, target, meta, zt, top, inv, loss, xp, wp, bias, slab, prob, dz, dbias, dbsum, part, acc;
  size_t total;
};

size_t al256x(size_t x) { return (x + 255) & ~(size_t)255; }

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// A product of I x J results over kblocks of k: 256 x 32 tiles where J fits one; 256 x 256 ones where they give (split
// over k, where that is allowed, into parts of 16 blocks at least) half the CUs work; else 128 x 128 ones, of which a
// CU holds two. Measured at float32 N=4095 H=512 V=32000, dh (30 large tiles, split by 8): 0.55 ms, 0.80 ms with the
// small. as_is: float32 W is read as it is, in k blocks of 32.
Product pick(int64_t I, int64_t J, int kblocks, int pairs, bool split, bool as_is) {
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

int loss_plan(const ews_loss_desc* s, bool train, bool direct, LPlan& p) {
  if (!s) return EWS_ERR_NULL;
  if (s->dtype != EWS_DTYPE_F32 && s->dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->bias_dtype != EWS_DTYPE_F32 && s->bias_dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->reduction < 0 || s->reduction > 2) return EWS_ERR_OPTION;
  if (s->rows < 1 || s->hidden < 1 || s->vocab < 1 || s->rows > 1 << 22 || s->hidden > 1 << 16 || s->vocab > 1 << 22)
    return EWS_ERR_SHAPE;
  if (s->hidden_stride < s->hidden || s->weight_stride < s->hidden) return EWS_ERR_SHAPE;
  // a launch has fewer than 2^32 threads, one for eight numbers of either operand
  const int64_t wide = (s->hidden + 63) / 64 * 64;
  if (s->rows * wide > (int64_t)1 << 34 || s->vocab * wide > (int64_t)1 << 34) return EWS_ERR_SHAPE;
  p.N = s->rows;
  p.H = s->hidden;
  p.V = s->vocab;
  p.np = s->dtype == EWS_DTYPE_F32 ? 3 : 1;
  p.train = train;
  p.packed = !direct;
  p.Hp = (int64_t)ceil_div(p.H, 64) * 64;
  p.Vp = (int64_t)ceil_div(p.V, 64) * 64;
  p.Np = train ? (int64_t)ceil_div(p.N, 64) * 64 : p.N;  // dW's k goes in blocks of 64 rows
  const int64_t each = p.Vp * (p.np == 3 ? 10 : 2);
  int64_t fit = train ? kChunkBytes / each / 256 * 256 : kScoreBytes / (p.Vp / 8) / 256 * 256;
  if (fit < 256) fit = 256;
  p.chunk = p.Np < fit ? p.Np : fit;
  // equal chunks: the last one's tiles fill the CUs as the others' do
  p.chunks = ceil_div(p.Np, p.chunk);
  if (p.chunks > 1) p.chunk = (int64_t)ceil_div(ceil_div(p.Np, p.chunks), 256) * 256;
  p.chunks = ceil_div(p.Np, p.chunk);
  p.twice = train && p.np == 1 && p.N <= (s->reduction == EWS_LOSS_NONE ? kFewRowsNone : kFewRowsMean);
  if (p.twice) {
    p.chunk = (int64_t)ceil_div(p.N, 32) * 32;
    p.Np = 2 * p.chunk;
  }
  const int64_t most = p.chunk < p.N ? p.chunk : p.N;  // rows of a chunk
  const int pairs = p.np == 3 ? kPairs : 1;
  p.as_is = p.np == 3 && direct;
  p.logits = pick(p.V, most, p.as_is ? ceil_div(p.H, 32) : (int)(p.Hp / 64), pairs, false, p.as_is);
  p.dh = pick(p.H, most, p.as_is ? ceil_div(p.V, 32) : (int)(p.Vp / 64), p.twice ? 2 : pairs, true, p.as_is);
  p.dw = pick(p.H, p.V, (int)((p.twice ? p.Np : p.chunk) / 64), pairs, true, false);
  p.bias_pad = p.logits.ti * p.logits.tile_i;
  p.slabs = p.bias_pad / p.logits.slab;
  size_t off = 0;
  auto take = [&off](size_t bytes) {
    const size_t at = off;
    off += al256x(bytes);
    return at;
  };
  p.map = take((size_t)p.N * 4);
  p.target = take((size_t)p.N * 4);
  p.meta = take(8);
  p.zt = take((size_t)p.N * 4);
  p.top = take((size_t)p.N * 4);
  p.inv = take((size_t)p.N * 4);
  p.loss = take((size_t)p.N * 4);
  p.xp = take((size_t)(p.Np * p.Hp * p.np * 2));
  p.wp = take(p.packed ? (size_t)(p.V * p.Hp * p.np * 2) : 0);
  p.bias = take((size_t)p.bias_pad * 4);
  p.slab = take((size_t)p.slabs * p.chunk * 8);
  if (train) {
    p.prob = take((size_t)(p.chunk * p.Vp) * (p.np == 3 || p.twice ? 4 : 2));
    p.dz = p.np == 3 ? take((size_t)(p.chunk * p.Vp) * 6) : p.prob;
    // 128 rows a workgroup (the bias's partial sums stay small), fewer where that leaves CUs without one
    p.dz_rows = 128;
    while (p.dz_rows > 4 && (int64_t)ceil_div(p.chunk, p.dz_rows) * ceil_div(p.Vp, 512) < 1024) p.dz_rows /= 2;
    p.dbias = take((size_t)(ceil_div(p.chunk, p.dz_rows) * p.Vp) * 4);
    p.dbsum = take((size_t)p.V * 4);
    size_t part = 0;
    if (p.dh.splits > 1) part = (size_t)p.dh.splits * p.chunk * p.H * 4;
    if (p.dw.splits > 1 && (size_t)p.dw.splits * p.V * p.H * 4 > part) part = (size_t)p.dw.splits * p.V * p.H * 4;
    p.part = take(part);
    p.acc = take(p.chunks > 1 && s->dtype == EWS_DTYPE_BF16 ? (size_t)p.V * p.H * 4 : 0);
  }
  p.total = off;
  return EWS_OK;
}

// bfloat16 weights whose rows start at multiples of 16 bytes and fill whole k blocks are read where they are, and
// float32 weights for few rows (of a stride that the tiles' offsets hold). Here what the sizes allow; bfloat16's
// address has to fit too.
bool may_read_direct(const ews_loss_desc* s) {
  if (s->weight_stride > 1 << 22) return false;
  if (s->dtype == EWS_DTYPE_F32) {
    // the three planes of h, and of a chunk's dz, lie within 32-bit offsets
    if ((s->rows + 63) * (int64_t)(s->hidden + 63) > 1 << 29 || s->vocab > 1 << 20) return false;
    return s->rows <= kFewRows32 || s->rows * (int64_t)s->vocab <= kFewLogits32;
  }
  return s->hidden % 64 == 0 && s->weight_stride % 8 == 0;
}

bool reads_direct(const ews_loss_desc* s, const void* weight) {
  return may_read_direct(s) && (s->dtype == EWS_DTYPE_F32 || (uintptr_t)weight % 16 == 0);
}

struct Call {
  const ews_loss_desc* s;
  LPlan p;
  char* w;
  hipStream_t st;
  Rows rows;
  Stats stats;
};

#define LOSS_CHECK()                                             \
  do {                                                           \
    if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH; \
  } while (0)

template <class K>
int allow_lds(K kernel, int bytes) {
  if (bytes <= 64 << 10) return EWS_OK;  // allowed as it is
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                             bytes) == hipSuccess
             ? EWS_OK
             : EWS_ERR_LAUNCH;
}

// Whether a float32 operand can be copied 16 bytes a lane.
bool pieces(const Operand32& o) { return (uintptr_t)o.p % 16 == 0 && o.ld % 4 == 0 && o.cols % 4 == 0; }

template <class T, int PAIRS, int KEEP>
int launch_logits_as(const LogitArgs& a, hipStream_t st) {
  const int lds = lds_bytes<T, PAIRS>(a.kblocks) + (T::I + T::J) * 4;
  const int rc = allow_lds(k_logits<T, PAIRS, KEEP>, lds);
  if (rc != EWS_OK) return rc;
  hipLaunchKernelGGL((k_logits<T, PAIRS, KEEP>), dim3((uint32_t)(a.ti * a.tj)), dim3(T::kThreads), lds, st, a);
  LOSS_CHECK();
  return EWS_OK;
}

template <int PAIRS, int KEEP>
int launch_logits(Kind kind, const LogitArgs& a, hipStream_t st) {
  if constexpr (KEEP != 1 && PAIRS != 1) {
    if (kind == kFew32)
      return pieces(a.W32) ? launch_logits_as<Few32<16>, 0, KEEP>(a, st) : launch_logits_as<Few32<4>, 0, KEEP>(a, st);
    if (kind == kMore32)
      return pieces(a.W32) ? launch_logits_as<More32<16>, 0, KEEP>(a, st) : launch_logits_as<More32<4>, 0, KEEP>(a, st);
  }
  if (kind == kLarge) return launch_logits_as<Large, PAIRS, KEEP>(a, st);
  return kind == kMedium ? launch_logits_as<Medium, PAIRS, KEEP>(a, st) : launch_logits_as<Flat, PAIRS, KEEP>(a, st);
}

// kP: float32 gradients are those of float32 operands
template <class T, bool ROWS, typename O, int kP>
int launch_grad_as(const GradArgs& a, hipStream_t st) {
  const int lds = lds_bytes<T, kP>(a.per);
  const int rc = allow_lds(k_grad<T, kP, ROWS, O>, lds);
  if (rc != EWS_OK) return rc;
  hipLaunchKernelGGL((k_grad<T, kP, ROWS, O>), dim3((uint32_t)(a.ti * a.tj), a.splits), dim3(T::kThreads), lds, st, a);
  LOSS_CHECK();
  if (a.splits > 1) {
    const int64_t n = (int64_t)(a.by_rows ? a.J : a.chunk) * a.I;
    if (a.splits > kFewSplits)
      hipLaunchKernelGGL((k_reduce<O>), dim3((uint32_t)((n + 31) / 32)), dim3(256), 0, st, a);
    else if (a.wide)
      hipLaunchKernelGGL((k_reduce_few<O, Eight>), dim3((uint32_t)((n / 8 + 255) / 256)), dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((k_reduce_few<O, One>), dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, st, a);
    LOSS_CHECK();
  }
  return EWS_OK;
}

template <bool ROWS, typename O>
int launch_grad(const Product& p, const GradArgs& a, hipStream_t st) {
  constexpr int kP = sizeof(O) == 4 ? kPairs : 1;
  if constexpr (!ROWS && kP == kPairs) {
    if (p.kind == kFew32)
      return pieces(a.P32) ? launch_grad_as<Few32<16>, ROWS, O, 0>(a, st) : launch_grad_as<Few32<4>, ROWS, O, 0>(a, st);
    if (p.kind == kMore32)
      return pieces(a.P32) ? launch_grad_as<More32<16>, ROWS, O, 0>(a, st)
                           : launch_grad_as<More32<4>, ROWS, O, 0>(a, st);
  }
  if constexpr (!ROWS && kP == 1) {
    if (p.pairs == 2) {
      if (p.kind == kLarge) return launch_grad_as<Large, ROWS, O, 2>(a, st);
      return p.kind == kMedium ? launch_grad_as<Medium, ROWS, O, 2>(a, st) : launch_grad_as<Flat, ROWS, O, 2>(a, st);
    }
  }
  if (p.kind == kLarge) return launch_grad_as<Large, ROWS, O, kP>(a, st);
  return p.kind == kMedium ? launch_grad_as<Medium, ROWS, O, kP>(a, st) : launch_grad_as<Flat, ROWS, O, kP>(a, st);
}

int rows_wide(const void* p, int64_t stride, bool f32) {
  return (uintptr_t)p % 16 == 0 && stride * (f32 ? 4 : 2) % 16 == 0;
}

// What every call begins with: the kept rows, the operands' planes, the bias.
int begin(Call& c, const void* hidden, const void* weight, const void* bias, const int64_t* targets, float* loss_rows,
          void* grad_hidden) {
  const LPlan& p = c.p;
  const bool f32 = p.np == 3;
  PackArgs x{};
  x.src = hidden;
  x.stride = c.s->hidden_stride;
  x.rows = p.N;
  x.cols = p.H;
  x.map = c.rows.map;
  x.kept = c.rows.kept;
  x.dst = (uint16_t*)(c.w + p.xp);
  x.ld = p.Hp;
  x.plane = p.Np * p.Hp;
  x.dst_rows = (int)p.Np;
  x.again = p.twice ? (int)p.chunk : 0;
  x.wide = rows_wide(x.src, x.stride, f32);
  PrepareArgs r{};
  r.targets = targets;
  r.n = p.N;
  r.vocab = p.V;
  r.padded = p.bias_pad;
  r.mean = c.s->reduction == EWS_LOSS_MEAN ? 1 : 0;
  r.H = p.H;
  r.ignore = c.s->ignore_index;
  r.rows = c.rows;
  r.loss_rows = loss_rows;
  r.bias = bias;
  r.bias_bf16 = c.s->bias_dtype == EWS_DTYPE_BF16;
  r.bias_out = (float*)(c.w + p.bias);
  r.grad_hidden = grad_hidden;
  // 64 workgroups at most list rows, 8192 or a multiple each
  r.each = ceil_div(ceil_div(p.N, 64), 8192) * 8192;
  r.kept_blocks = ceil_div(p.N, r.each);
  r.bias_blocks = ceil_div(p.bias_pad, 1024);
  r.ignored_blocks = grad_hidden ? ceil_div(p.N, 16) : 0;
  int64_t blocks = r.kept_blocks + r.bias_blocks + r.ignored_blocks;
  if (p.packed) {
    PackArgs& w = r.weight;
    w.src = weight;
    w.stride = c.s->weight_stride;
    w.rows = p.V;
    w.cols = p.H;
    w.dst = (uint16_t*)(c.w + p.wp);
    w.ld = p.Hp;
    w.plane = p.V * p.Hp;
    w.dst_rows = p.V;
    w.wide = rows_wide(w.src, w.stride, f32);
    blocks += ceil_div(p.V * (p.Hp / 8), 1024);
  }
  // up to eight sixteen-byte packs a thread cost less there than a launch does
  const bool few = p.Np * (p.Hp / 8) <= 8192;
  if (few) r.few = x;
  if (f32)
    hipLaunchKernelGGL((k_prepare<float>), dim3((uint32_t)blocks), dim3(1024), 0, c.st, r);
  else
    hipLaunchKernelGGL((k_prepare<bf16>), dim3((uint32_t)blocks), dim3(1024), 0, c.st, r);
  LOSS_CHECK();
  if (few) return EWS_OK;
  const uint32_t packs = (uint32_t)((p.Np * (p.Hp / 8) + 255) / 256);
  if (f32)
    hipLaunchKernelGGL((k_pack<float>), dim3(packs), dim3(256), 0, c.st, x);
  else
    hipLaunchKernelGGL((k_pack<bf16>), dim3(packs), dim3(256), 0, c.st, x);
  LOSS_CHECK();
  return EWS_OK;
}

Operand32 weight_operand32(const Call& c, const void* weight) {
  const LPlan& p = c.p;
  return Operand32{(const float*)weight, c.s->weight_stride, p.V, p.H};
}

Operand weight_operand(const Call& c, const void* weight) {
  const LPlan& p = c.p;
  if (p.packed) return Operand{(const uint16_t*)(c.w + p.wp), p.Hp, p.V * p.Hp, p.V, (int)p.Hp};
  return Operand{(const uint16_t*)weight, c.s->weight_stride, 0, p.V, (int)p.Hp};
}

Operand hidden_operand(const Call& c) {
  const LPlan& p = c.p;
  return Operand{(const uint16_t*)(c.w + p.xp), p.Hp, p.Np * p.Hp, (int)p.Np, (int)p.Hp};
}

int logits(const Call& c, const void* weight, int chunk, float* loss_rows) {
  const LPlan& p = c.p;
  LogitArgs a{};
  if (p.as_is)
    a.W32 = weight_operand32(c, weight);
  else
    a.W = weight_operand(c, weight);
  a.X = hidden_operand(c);
  a.ti = p.logits.ti;
  a.tj = p.logits.tj;
  a.kblocks = p.logits.kblocks;
  a.c0 = (int)(chunk * p.chunk);
  a.chunk = (int)p.chunk;
  a.bias = (const float*)(c.w + p.bias);
  a.rows = c.rows;
  a.st = c.stats;
  int rc;
  if (p.train) {
    a.prob = c.w + p.prob;
    a.ldp = p.Vp;
    rc = p.np == 3 ? launch_logits<kPairs, 2>(p.logits.kind, a, c.st) : launch_logits<1, 1>(p.logits.kind, a, c.st);
  } else {
    rc = p.np == 3 ? launch_logits<kPairs, 0>(p.logits.kind, a, c.st) : launch_logits<1, 0>(p.logits.kind, a, c.st);
  }
  if (rc != EWS_OK) return rc;
  // one row's slabs by a workgroup's threads where there are few rows: N=1, V=100003: 23 us with 16 threads a row
  if (p.N <= 256)
    hipLaunchKernelGGL((k_join<4>), dim3(ceil_div(p.chunk, 4)), dim3(1024), 0, c.st, c.stats, c.rows, p.slabs, a.c0,
                       a.chunk, loss_rows);
  else
    hipLaunchKernelGGL((k_join<64>), dim3(ceil_div(p.chunk, 64)), dim3(1024), 0, c.st, c.stats, c.rows, p.slabs, a.c0,
                       a.chunk, loss_rows);
  LOSS_CHECK();
  return EWS_OK;
}

Call make_call(const ews_loss_desc* s, const LPlan& p, void* workspace, ews_stream_t stream) {
  Call c{};
  c.s = s;
  c.p = p;
  c.w = (char*)workspace;
  c.st = (hipStream_t)stream;
  c.rows.map = (int*)(c.w + p.map);
  c.rows.target = (int*)(c.w + p.target);
  c.rows.kept = (int*)(c.w + p.meta);
  c.rows.scale = (float*)(c.w + p.meta + 4);
  c.stats.slab = (float2*)(c.w + p.slab);
  c.stats.zt = (float*)(c.w + p.zt);
  c.stats.top = (float*)(c.w + p.top);
  c.stats.inv = (float*)(c.w + p.inv);
  c.stats.loss = (float*)(c.w + p.loss);
  return c;
}

int launch_total(const Call& c, float* loss) {
  hipLaunchKernelGGL(k_total, dim3(1), dim3(1024), 0, c.st, c.stats, c.rows, loss);
  LOSS_CHECK();
  return EWS_OK;
}

// Chunk k's gradients from what logits() kept of it; the last chunk writes the call's loss too, where asked.
int gradients(const Call& c, const void* weight, int k, const float* upstream, float* loss, void* grad_hidden,
              void* grad_weight, void* grad_bias) {
  const LPlan& p = c.p;
  const bool f32 = p.np == 3, last = k + 1 == p.chunks;
  const int wide = p.H % 8 == 0 && (uintptr_t)grad_hidden % 16 == 0 && (uintptr_t)grad_weight % 16 == 0;
  const float* factor = upstream ? nullptr : c.rows.scale;
  int rc;
  DzArgs z{};
  z.rows = c.rows;
  z.st = c.stats;
  z.upstream = upstream;
  z.c0 = (int)(k * p.chunk);
  z.chunk = (int)p.chunk;
  z.slab = p.logits.slab;
  z.prob = c.w + p.prob;
  z.ld = p.Vp;
  z.dz = (uint16_t*)(c.w + p.dz);
  z.plane = p.chunk * p.Vp;
  z.bias = grad_bias ? (float*)(c.w + p.dbias) : nullptr;
  z.each = p.dz_rows;
  z.loss = last ? loss : nullptr;
  const dim3 grid(ceil_div(p.Vp, 512) + (z.loss ? 1 : 0), ceil_div(p.chunk, p.dz_rows));
  if (p.Vp <= 256) {
    z.lanes = p.Vp <= 64 ? 8 : p.Vp <= 128 ? 16 : 32;
    if (f32)
      hipLaunchKernelGGL((k_dz<3, true>), grid, dim3(256), 0, c.st, z);
    else if (p.twice)
      hipLaunchKernelGGL((k_dz<2, true>), grid, dim3(256), 0, c.st, z);
    else
      hipLaunchKernelGGL((k_dz<1, true>), grid, dim3(256), 0, c.st, z);
  } else if (f32) {
    hipLaunchKernelGGL((k_dz<3, false>), grid, dim3(256), 0, c.st, z);
  } else if (p.twice) {
    hipLaunchKernelGGL((k_dz<2, false>), grid, dim3(256), 0, c.st, z);
  } else {
    hipLaunchKernelGGL((k_dz<1, false>), grid, dim3(256), 0, c.st, z);
  }
  LOSS_CHECK();
  if (grad_bias) {
    float* sum = (float*)(c.w + p.dbsum);
    const dim3 g(ceil_div(p.V, 64));
    if (c.s->bias_dtype == EWS_DTYPE_BF16)
      hipLaunchKernelGGL((k_dbias<bf16>), g, dim3(1024), 0, c.st, z.bias, (int)grid.y, p.Vp, p.V, sum, k > 0 ? 1 : 0,
                         factor, last ? (bf16*)grad_bias : nullptr);
    else
      hipLaunchKernelGGL((k_dbias<float>), g, dim3(1024), 0, c.st, z.bias, (int)grid.y, p.Vp, p.V, sum, k > 0 ? 1 : 0,
                         factor, last ? (float*)grad_bias : nullptr);
    LOSS_CHECK();
  }
  GradArgs g{};
  g.c0 = z.c0;
  g.chunk = z.chunk;
  g.rows = c.rows;
  g.wide = wide;
  g.factor = factor;
  g.part = (float*)(c.w + p.part);
  if (grad_hidden) {
    if (p.as_is)
      g.P32 = weight_operand32(c, weight);
    else
      g.P = weight_operand(c, weight);
    g.Q = Operand{z.dz, p.Vp, z.plane, (int)p.chunk, 0};
    g.ti = p.dh.ti;
    g.tj = p.dh.tj;
    g.splits = p.dh.splits;
    g.kblocks = p.dh.kblocks;
    g.per = p.dh.per;
    g.by_rows = 0;
    g.I = p.H;
    g.J = (int)p.chunk;
    g.sum = nullptr;
    g.add = 0;
    g.out = grad_hidden;
    rc = f32 ? launch_grad<false, float>(p.dh, g, c.st) : launch_grad<false, bf16>(p.dh, g, c.st);
    if (rc != EWS_OK) return rc;
  }
  if (grad_weight) {
    g.P = hidden_operand(c);
    g.P.p += z.c0 * p.Hp;
    g.P.rows -= z.c0;
    g.Q = Operand{z.dz, p.Vp, z.plane, (int)(p.twice ? 2 * p.chunk : p.chunk), (int)p.Vp};
    g.twice = p.twice;
    g.ti = p.dw.ti;
    g.tj = p.dw.tj;
    g.splits = p.dw.splits;
    g.kblocks = p.dw.kblocks;
    g.per = p.dw.per;
    g.by_rows = 1;
    g.I = p.H;
    g.J = p.V;
    g.sum = f32 ? (float*)grad_weight : (float*)(c.w + p.acc);
    g.add = k > 0 ? 1 : 0;
    g.out = last || f32 ? grad_weight : nullptr;
    rc = f32 ? launch_grad<true, float>(p.dw, g, c.st) : launch_grad<true, bf16>(p.dw, g, c.st);
    if (rc != EWS_OK) return rc;
  }
  return EWS_OK;
}

}  // namespace

extern "C" {

size_t ews_loss_workspace_bytes(const ews_loss_desc* desc, int train) {
  LPlan p;
  if (loss_plan(desc, train != 0, false, p) != EWS_OK) return 0;
  if (!may_read_direct(desc)) return p.total;
  // read as it is W needs no packed copy; bfloat16's address, which is not known here, may ask for one all the same
  const size_t packed = desc->dtype == EWS_DTYPE_F32 ? 0 : p.total;
  loss_plan(desc, train != 0, true, p);
  return p.total > packed ? p.total : packed;
}

size_t ews_loss_workspace_bytes_for(const ews_loss_desc* desc, const void* weight, int train) {
  LPlan p;
  return loss_plan(desc, train != 0, desc && reads_direct(desc, weight), p) == EWS_OK ? p.total : 0;
}

int ews_loss_tile(const ews_loss_desc* desc, const void* weight, int train, int product, int32_t* tile) {
  LPlan p;
  const int rc = loss_plan(desc, train != 0, desc && reads_direct(desc, weight), p);
  if (rc != EWS_OK) return rc;
  if (!tile) return EWS_ERR_NULL;
  if (product < 0 || product > (train ? 2 : 0)) return EWS_ERR_OPTION;
  const Product& q = product == 0 ? p.logits : product == 1 ? p.dh : p.dw;
  tile[0] = q.tile_i;
  tile[1] = q.tile_j;
  tile[2] = q.splits;
  tile[3] = p.chunks;
  return EWS_OK;
}

int ews_loss_forward(const ews_loss_desc* desc, const void* hidden, const void* weight, const void* bias,
                     const int64_t* targets, float* loss, void* workspace, ews_stream_t stream) {
  LPlan p;
  int rc = loss_plan(desc, false, desc && reads_direct(desc, weight), p);
  if (rc != EWS_OK) return rc;
  if (!hidden || !weight || !targets || !loss || !workspace) return EWS_ERR_NULL;
  Call c = make_call(desc, p, workspace, stream);
  float* rows = desc->reduction == EWS_LOSS_NONE ? loss : nullptr;
  rc = begin(c, hidden, weight, bias, targets, rows, nullptr);
  if (rc != EWS_OK) return rc;
  for (int k = 0; k < p.chunks; ++k) {
    rc = logits(c, weight, k, rows);
    if (rc != EWS_OK) return rc;
  }
  return rows ? EWS_OK : launch_total(c, loss);
}

int ews_loss_train(const ews_loss_desc* desc, const void* hidden, const void* weight, const void* bias,
                   const int64_t* targets, const float* upstream, float* loss, void* grad_hidden, void* grad_weight,
                   void* grad_bias, void* workspace, ews_stream_t stream) {
  LPlan p;
  int rc = loss_plan(desc, true, desc && reads_direct(desc, weight), p);
  if (rc != EWS_OK) return rc;
  if (!hidden || !weight || !targets || !workspace || (grad_bias && !bias)) return EWS_ERR_NULL;
  Call c = make_call(desc, p, workspace, stream);
  float* rows = desc->reduction == EWS_LOSS_NONE ? loss : nullptr;
  rc = begin(c, hidden, weight, bias, targets, rows, grad_hidden);
  for (int k = 0; k < p.chunks && rc == EWS_OK; ++k) {
    rc = logits(c, weight, k, rows);
    if (rc == EWS_OK)
      rc = gradients(c, weight, k, upstream, rows ? nullptr : loss, grad_hidden, grad_weight, grad_bias);
  }
  return rc;
}

int ews_loss_keeps(const ews_loss_desc* desc) {
  LPlan p;
  return loss_plan(desc, true, false, p) == EWS_OK && p.chunks == 1;
}

int ews_loss_keep(const ews_loss_desc* desc, const void* hidden, const void* weight, const void* bias,
                  const int64_t* targets, float* loss, void* grad_hidden, void* workspace, ews_stream_t stream) {
  LPlan p;
  int rc = loss_plan(desc, true, desc && reads_direct(desc, weight), p);
  if (rc != EWS_OK) return rc;
  if (p.chunks > 1) return EWS_ERR_SHAPE;
  if (!hidden || !weight || !targets || !loss || !workspace) return EWS_ERR_NULL;
  Call c = make_call(desc, p, workspace, stream);
  float* rows = desc->reduction == EWS_LOSS_NONE ? loss : nullptr;
  rc = begin(c, hidden, weight, bias, targets, rows, grad_hidden);
  if (rc == EWS_OK) rc = logits(c, weight, 0, rows);
  return rc != EWS_OK || rows ? rc : launch_total(c, loss);
}

int ews_loss_kept(const ews_loss_desc* desc, const void* weight, const float* upstream, void* grad_hidden,
                  void* grad_weight, void* grad_bias, void* workspace, ews_stream_t stream) {
  LPlan p;
  const int rc = loss_plan(desc, true, desc && reads_direct(desc, weight), p);
  if (rc != EWS_OK) return rc;
  if (p.chunks > 1) return EWS_ERR_SHAPE;
  if (!weight || !workspace) return EWS_ERR_NULL;
  return gradients(make_call(desc, p, workspace, stream), weight, 0, upstream, nullptr, grad_hidden, grad_weight,
                   grad_bias);
}

}  // extern "C"
