// Norm over many tensors on MI355X (gfx950), and the scaling of all of them by one coefficient: gradient clipping.
//
//   norm = sqrt(sum over tensors and elements of g^2),  c = min(1, max_norm / (norm + 1e-6)),  out = c g
//
// Memory bounds it: everything is read for the norm before any number can be scaled, so clipping reads twice and
// writes once. The tensors go by value in a launch's arguments (kMany to a launch): no table is copied to the device
// and the host waits for nothing. A workgroup takes one chunk of one tensor; squares are added in float64, so no
// gradient that float32 holds overflows or vanishes, and the chunks' sums are added in a fixed order.
// A scaling launch walks its chunks backwards: of a set in one launch the data read last by the norm is read first,
// while it is in the caches. The launches of a larger set go in the norm's order: backwards too they measured the same
// (196 tensors, 1.2 GB: 656 us for 659; 132 tensors, 6.4 GB: 3480 for 3475). In place with c = 1 nothing is read or
// written again.
//
// 3.2 G bfloat16 numbers in 132 tensors: read for the norm in 1.07 ms (6.1 TB/s), scaled in 2.35 (5.5 TB/s).
#include <hip/hip_runtime.h>

#include "ews_hip.h"
#include "ews_vec.h"

namespace ews {
namespace clip {

using namespace ews::vec;

constexpr int kMany = 128;        // tensors of one launch
constexpr int kThreads = 256;
constexpr int kChunk = 16384;     // elements a workgroup takes

struct Table {
  const void* in[kMany];
  void* out[kMany];
  int64_t count[kMany];           // elements; negated for bfloat16
  uint32_t first[kMany + 1];      // the first chunk of every tensor
  int n;
};
static_assert(sizeof(Table) < 4000, "a launch's arguments hold 4 KB");

// The tensor of a chunk: the last whose first chunk is not past it.
__device__ __forceinline__ int find(const Table& t, uint32_t chunk) {
  int lo = 0, hi = t.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename T, int V>
__device__ __forceinline__ double chunk_squares(const T* p, int n) {
  double s = 0.0;
  constexpr int kAhead = 4;
  const int packs = n / V;
  int c = threadIdx.x;
  for (; c + (kAhead - 1) * kThreads < packs; c += kAhead * kThreads) {
    Pack<T, V> x[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) x[q].load(p + (int64_t)(c + q * kThreads) * V);
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const double v = (double)x[q].get(i);
        s = fma(v, v, s);
      }
  }
  for (; c < packs; c += kThreads) {
    Pack<T, V> x;
    x.load(p + (int64_t)c * V);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double v = (double)x.get(i);
      s = fma(v, v, s);
    }
  }
  if (V > 1 && (int)threadIdx.x < n - packs * V) {
    const double v = (double)widen(p[packs * V + threadIdx.x]);
    s = fma(v, v, s);
  }
  return s;
}

__device__ __forceinline__ double block_sum(double s, double* sums, int waves) {
#pragma unroll
  for (int m = 32; m; m >>= 1) s += __shfl_xor(s, m);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < waves; ++w) s += sums[w];
  return s;
}

__global__ __launch_bounds__(kThreads) void k_squares(Table t, double* sums) {
  __shared__ double part[kThreads / 64];
  const int k = find(t, blockIdx.x);
  const int64_t off = (int64_t)(blockIdx.x - t.first[k]) * kChunk;
  const bool half = t.count[k] < 0;
  const int64_t count = half ? -t.count[k] : t.count[k];
  const int n = (int)(count - off < kChunk ? count - off : kChunk);
  double s;
  if (half) {
    const bf16* p = (const bf16*)t.in[k] + off;
    s = (uintptr_t)p % 16 == 0 ? chunk_squares<bf16, 8>(p, n) : chunk_squares<bf16, 1>(p, n);
  } else {
    const float* p = (const float*)t.in[k] + off;
    s = (uintptr_t)p % 16 == 0 ? chunk_squares<float, 4>(p, n) : chunk_squares<float, 1>(p, n);
  }
  s = block_sum(s, part, kThreads / 64);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// result[0] = norm, result[1] = the coefficient (NaN where the norm is NaN, 0 where it is infinite)
__global__ __launch_bounds__(1024) void k_norm(const double* sums, int64_t n, float max_norm, float* result) {
  __shared__ double part[16];
  double s = 0.0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += sums[i];
  s = block_sum(s, part, 16);
  if (threadIdx.x == 0) {
    const double norm = sqrt(s);
    const double c = (double)max_norm / (norm + 1e-6);
    result[0] = (float)norm;
    result[1] = c > 1.0 ? 1.0f : (float)c;
  }
}

template <typename T, int V>
__device__ __forceinline__ void chunk_scale(const T* p, T* o, int n, float c) {
  constexpr int kAhead = 4;
  const int packs = n / V;
  int k = threadIdx.x;
  for (; k + (kAhead - 1) * kThreads < packs; k += kAhead * kThreads) {
    Pack<T, V> x[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) x[q].load(p + (int64_t)(k + q * kThreads) * V);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      float y[V];
#pragma unroll
      for (int i = 0; i < V; ++i) y[i] = x[q].get(i) * c;
      x[q].set(y);
      x[q].store(o + (int64_t)(k + q * kThreads) * V);
    }
  }
  for (; k < packs; k += kThreads) {
    Pack<T, V> x;
    float y[V];
    x.load(p + (int64_t)k * V);
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = x.get(i) * c;
    x.set(y);
    x.store(o + (int64_t)k * V);
  }
  if (V > 1 && (int)threadIdx.x < n - packs * V) {
    const int i = packs * V + threadIdx.x;
    o[i] = narrow<T>(widen(p[i]) * c);
  }
}

__global__ __launch_bounds__(kThreads) void k_scale(Table t, const float* factor) {
  const uint32_t chunk = gridDim.x - 1 - blockIdx.x;
  const int k = find(t, chunk);
  const float c = *factor;
  if (c == 1.0f && t.in[k] == t.out[k]) return;
  const int64_t off = (int64_t)(chunk - t.first[k]) * kChunk;
  const bool half = t.count[k] < 0;
  const int64_t count = half ? -t.count[k] : t.count[k];
  const int n = (int)(count - off < kChunk ? count - off : kChunk);
  if (half) {
    const bf16* p = (const bf16*)t.in[k] + off;
    bf16* o = (bf16*)t.out[k] + off;
    if (((uintptr_t)p | (uintptr_t)o) % 16 == 0)
      chunk_scale<bf16, 8>(p, o, n, c);
    else
      chunk_scale<bf16, 1>(p, o, n, c);
  } else {
    const float* p = (const float*)t.in[k] + off;
    float* o = (float*)t.out[k] + off;
    if (((uintptr_t)p | (uintptr_t)o) % 16 == 0)
      chunk_scale<float, 4>(p, o, n, c);
    else
      chunk_scale<float, 1>(p, o, n, c);
  }
}

}  // namespace clip
}  // namespace ews

namespace {

using namespace ews::clip;

// Chunks of one tensor; 0 for an empty one, which no launch names.
int64_t chunks_of(int64_t count) { return (count + kChunk - 1) / kChunk; }

// The next launch's tensors, from `at` on: as many as the table and the grid hold. Returns its chunks.
uint32_t fill(Table& t, int n, int& at, const uint64_t* in, const uint64_t* out, const int64_t* counts,
              const int32_t* dtypes) {
  t.n = 0;
  int64_t chunks = 0;
  for (; at < n && t.n < kMany; ++at) {
    if (counts[at] == 0) continue;
    const int64_t more = chunks_of(counts[at]);
    if (t.n > 0 && chunks + more > 1 << 23) break;  // a launch has fewer than 2^32 threads
    t.in[t.n] = (const void*)in[at];
    t.out[t.n] = out ? (void*)out[at] : (void*)in[at];
    t.count[t.n] = dtypes[at] == EWS_DTYPE_BF16 ? -counts[at] : counts[at];
    t.first[t.n++] = (uint32_t)chunks;
    chunks += more;
  }
  t.first[t.n] = (uint32_t)chunks;
  return (uint32_t)chunks;
}

int check(int n, const uint64_t* in, const uint64_t* out, const int64_t* counts, const int32_t* dtypes) {
  if (n < 0) return EWS_ERR_SHAPE;
  if (n > 0 && (!in || !counts || !dtypes)) return EWS_ERR_NULL;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0 || chunks_of(counts[i]) > 1 << 23) return EWS_ERR_SHAPE;
    if (dtypes[i] != EWS_DTYPE_F32 && dtypes[i] != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
    if (counts[i] > 0 && (!in[i] || (out && !out[i]))) return EWS_ERR_NULL;
  }
  return EWS_OK;
}

int scale_all(int n, const uint64_t* in, const uint64_t* out, const int64_t* counts, const int32_t* dtypes,
              const float* factor, hipStream_t st) {
  Table t;
  for (int at = 0; at < n;) {
    const uint32_t chunks = fill(t, n, at, in, out, counts, dtypes);
    if (!chunks) continue;
    hipLaunchKernelGGL(k_scale, dim3(chunks), dim3(kThreads), 0, st, t, factor);
    if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  }
  return EWS_OK;
}

}  // namespace

extern "C" {

size_t ews_clip_workspace_bytes(int n, const int64_t* counts) {
  if (n < 0 || (n > 0 && !counts)) return 0;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (counts[i] < 0) return 0;
    chunks += chunks_of(counts[i]);
  }
  return (size_t)(chunks > 0 ? chunks : 1) * 8;
}

int ews_clip(int n, const uint64_t* in, const uint64_t* out, const int64_t* counts, const int32_t* dtypes,
             float max_norm, int32_t scale, float* result, void* workspace, ews_stream_t stream) {
  const int rc = check(n, in, scale ? out : nullptr, counts, dtypes);
  if (rc != EWS_OK) return rc;
  if (!result || !workspace || (scale && n > 0 && !out)) return EWS_ERR_NULL;
  hipStream_t st = (hipStream_t)stream;
  double* sums = (double*)workspace;
  int64_t done = 0;
  Table t;
  for (int at = 0; at < n;) {
    const uint32_t chunks = fill(t, n, at, in, nullptr, counts, dtypes);
    if (!chunks) continue;
    hipLaunchKernelGGL(k_squares, dim3(chunks), dim3(kThreads), 0, st, t, sums + done);
    if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
    done += chunks;
  }
  hipLaunchKernelGGL(k_norm, dim3(1), dim3(1024), 0, st, sums, done, max_norm, result);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  return scale ? scale_all(n, in, out, counts, dtypes, result + 1, st) : EWS_OK;
}

// The gradients of ews_loss_train, scaled in place as a clipped set is. They have been rounded to their type already: a
// factor that is no power of two rounds bfloat16 ones again (half a unit each time). Kept in float32 for this they
// would take twice the memory and be read and written once more in every step, where a factor of 1 now reads nothing.
int ews_loss_scale(const ews_loss_desc* desc, void* grad_hidden, void* grad_weight, void* grad_bias,
                   const float* factor, ews_stream_t stream) {
  if (!desc || !factor) return EWS_ERR_NULL;
  if (ews_loss_workspace_bytes(desc, 0) == 0) return EWS_ERR_SHAPE;
  uint64_t at[3];
  int64_t counts[3];
  int32_t dtypes[3];
  int n = 0;
  auto take = [&](void* p, int64_t count, int32_t dtype) {
    if (!p) return;
    at[n] = (uint64_t)p;
    counts[n] = count;
    dtypes[n++] = dtype;
  };
  take(grad_hidden, (int64_t)desc->rows * desc->hidden, desc->dtype);
  take(grad_weight, (int64_t)desc->vocab * desc->hidden, desc->dtype);
  take(grad_bias, desc->vocab, desc->bias_dtype);
  const int rc = check(n, at, at, counts, dtypes);
  return rc != EWS_OK ? rc : scale_all(n, at, at, counts, dtypes, factor, (hipStream_t)stream);
}

}  // extern "C"
