// Embedding lookup of a token model on MI355X (gfx950), and its gradient.
//
//   forward   out[n, :] = s W[t_n, :]
//   backward  dW[v, :] = s sum_{n : t_n = v} g[n, :], zero for a token that does not occur and for the padding token
//
// Both only move rows, so memory bounds them. The backward adds no number with an atomic: it sorts the positions by
// token (stable, so a token's rows are added in the order of the text) and sums runs of equal tokens, in float32,
// rounding each row of dW once. The same inputs give the same bits.
//
//   k_sort   a workgroup owns a range of the vocabulary, reads every token twice (the ids stay in L2) and writes the
//            sorted positions of its own ones: counts first, then the places. No workgroup waits for another.
//   k_runs   a wavefront takes kRun sorted positions and one column tile, whatever tokens they are, so a frequent
//            token costs no more than rare ones: rows of runs that lie inside are written, the ends of runs that go on
//            in a neighbour's positions are kept as float32 partial rows.
//   k_join   adds the partial rows of the runs that were cut, in order.
//   k_absent zeroes the rows of dW without a token.
//
// An id outside [0, vocab) reads nothing: its output row is NaN and it has no gradient.
#include <hip/hip_runtime.h>

#include "ews_hip.h"
#include "ews_vec.h"

namespace ews {
namespace embed {

using namespace ews::vec;

constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kPerThread = 4;                        // consecutive tokens a thread reads at a time
constexpr int kPiece = kSortThreads * kPerThread;    // tokens a workgroup looks through at a time
constexpr int kMaxRange = 1024;                      // vocabulary entries a workgroup of k_sort may own
constexpr int kRun = 32;                             // sorted positions a wavefront of k_runs adds up
constexpr int kJoinWaves = 4;

struct Args {
  int64_t n, stride, pad;
  int H, V, R;     // R: vocabulary entries per workgroup of k_sort
  int lanes;       // lanes a row of the lookup is spread over
  float scale;
  const void* tokens;
  const void* weight;
  void* out;
  const void* gout;
  void* gweight;
  int* order;      // (n) positions, sorted by token
  int* sorted;     // (n) their tokens
  int* start;      // (V + 1) first sorted position of every token; start[V]: positions that count
  float* part;     // (runs, 2, H) sums of the runs cut at a wavefront's first and last position
};

template <typename T, int V, typename Tok>
__global__ __launch_bounds__(256) void k_lookup(Args a) {
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid / a.lanes;
  if (row >= a.n) return;
  const int lane = (int)(gid % a.lanes);
  const int64_t t = (int64_t)((const Tok*)a.tokens)[row];
  const bool known = t >= 0 && t < a.V;
  const T* src = (const T*)a.weight + (known ? t * a.stride : 0);
  T* dst = (T*)a.out + row * a.H;
  const int packs = a.H / V;
  for (int c = lane; c < packs; c += a.lanes) {
    Pack<T, V> p;
    float x[V];
    if (known) p.load(src + (int64_t)c * V);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = known ? p.get(i) * a.scale : __builtin_nanf("");
    p.set(x);
    p.store(dst + (int64_t)c * V);
  }
}

template <typename Tok>
__device__ __forceinline__ int local_id(const Tok* tokens, int64_t i, int64_t n, int64_t lo, int64_t hi, int64_t pad,
                                        int64_t vocab, int& below) {
  if (i >= n) return -1;
  const int64_t t = (int64_t)tokens[i];
  if (t < 0 || t >= vocab || t == pad) return -1;
  if (t < lo) ++below;
  return (t >= lo && t < hi) ? (int)(t - lo) : -1;
}

template <typename Tok>
__global__ __launch_bounds__(kSortThreads) void k_sort(Args a) {
  __shared__ int cnt[kMaxRange];             // occurrences, then the next free place, of every own token
  __shared__ int wsum[kSortWaves];
  __shared__ int lpos[kPiece];               // own positions of a piece, in the order of the text
  __shared__ uint16_t lid[kPiece];
  __shared__ int base;
  const Tok* tokens = (const Tok*)a.tokens;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t lo = (int64_t)blockIdx.x * a.R;
  const int64_t hi = lo + a.R < a.V ? lo + a.R : a.V;
  const int range = (int)(hi - lo);
  for (int i = tid; i < range; i += kSortThreads) cnt[i] = 0;
  if (tid == 0) base = 0;
  __syncthreads();

  // how often each own token occurs, and how many positions the smaller tokens take
  int below = 0;
  for (int64_t p0 = 0; p0 < a.n; p0 += kPiece) {
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) {
      const int id = local_id(tokens, p0 + (int64_t)q * kSortThreads + tid, a.n, lo, hi, a.pad, a.V, below);
      if (id >= 0) atomicAdd(&cnt[id], 1);
    }
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) below += __shfl_xor(below, s);
  if (lane == 0) atomicAdd(&base, below);
  __syncthreads();

  // the first place of every own token (exclusive sums of the counts; range <= kMaxRange = one per thread)
  const int mine = tid < range ? cnt[tid] : 0;
  int incl = mine;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int up = __shfl_up(incl, s);
    if (lane >= s) incl += up;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  int first = base + incl - mine;
  for (int w = 0; w < wave; ++w) first += wsum[w];
  if (tid < range) {
    cnt[tid] = first;
    a.start[lo + tid] = first;
    if (lo + tid == a.V - 1) a.start[a.V] = first + mine;
  }
  __syncthreads();

  for (int64_t p0 = 0; p0 < a.n; p0 += kPiece) {
    int ids[kPerThread], m = 0, unused = 0;
    const int64_t i0 = p0 + (int64_t)tid * kPerThread;
#pragma unroll
    for (int q = 0; q < kPerThread; ++q) {
      ids[q] = local_id(tokens, i0 + q, a.n, lo, hi, a.pad, a.V, unused);
      m += ids[q] >= 0;
    }
    int at = m;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int up = __shfl_up(at, s);
      if (lane >= s) at += up;
    }
    if (lane == 63) wsum[wave] = at;
    at -= m;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      if (w < wave) at += wsum[w];
      total += wsum[w];
    }
#pragma unroll
    for (int q = 0; q < kPerThread; ++q)
      if (ids[q] >= 0) {
        lpos[at] = (int)(i0 + q);
        lid[at] = (uint16_t)ids[q];
        ++at;
      }
    __syncthreads();
    // tokens are dealt to the wavefronts, so a token's next place has one owner; equal tokens of 64 keep their order
    for (int l0 = 0; l0 < total; l0 += 64) {
      const int l = l0 + lane;
      const int id = l < total ? (int)lid[l] : -1;
      uint64_t left = __ballot(id >= 0 && id % kSortWaves == wave);
      while (left) {
        const int leader = __ffsll((unsigned long long)left) - 1;
        const int same_id = __shfl(id, leader);
        const uint64_t same = __ballot(id == same_id);
        const int place = cnt[same_id];
        if (id == same_id) {
          const int rank = __popcll(same & ((1ull << lane) - 1ull));
          a.order[place + rank] = lpos[l];
          a.sorted[place + rank] = (int)lo + id;
        }
        if (lane == leader) cnt[same_id] = place + __popcll(same);
        left &= ~same;
      }
    }
    __syncthreads();
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void k_runs(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t run = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int col = ((int)blockIdx.y * 64 + lane) * V;
  const int total = a.start[a.V];
  const int64_t b = run * kRun;
  if (b >= total) return;
  const int j0 = (int)b, j1 = j0 + kRun < total ? j0 + kRun : total;
  const bool in = col < a.H;
  const T* g = (const T*)a.gout + (in ? col : 0);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  constexpr int kAhead = 8;
  for (int j = j0; j < j1; j += kAhead) {
    Pack<T, V> p[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int jj = j + q < j1 ? j + q : j1 - 1;
      p[q].load(g + (int64_t)a.order[jj] * a.H);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (j + q >= j1) break;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += p[q].get(i);
      const int t = a.sorted[j + q];
      const bool last = j + q + 1 == j1;
      if (!last && a.sorted[j + q + 1] == t) continue;
      const int s0 = a.start[t], s1 = a.start[t + 1];
      if (in) {
        if (s0 >= j0 && s1 <= j1) {
          Pack<T, V> o;
          float x[V];
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = acc[i] * a.scale;
          o.set(x);
          o.store((T*)a.gweight + (int64_t)t * a.H + col);
        } else {
          float* part = a.part + (run * 2 + (s0 < j0 ? 0 : 1)) * a.H + col;
#pragma unroll
          for (int i = 0; i < V; ++i) part[i] = acc[i];
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    }
  }
}

// One workgroup per run of kRun positions and 64 columns; only those whose last token starts in them and goes on work.
// The wavefronts add contiguous quarters of the partial rows, the first one joins them.
template <typename T>
__global__ __launch_bounds__(64 * kJoinWaves) void k_join(Args a) {
  __shared__ float sums[kJoinWaves][64];
  const int total = a.start[a.V];
  const int64_t run = blockIdx.x;
  const int64_t b = run * kRun;
  if (b >= total) return;
  const int j0 = (int)b, j1 = j0 + kRun < total ? j0 + kRun : total;
  const int t = a.sorted[j1 - 1];
  const int s0 = a.start[t], s1 = a.start[t + 1];
  if (s0 < j0 || s1 <= j1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t last = (int64_t)(s1 - 1) / kRun;  // the last run that holds the token
  const int64_t per = (last - run + kJoinWaves - 1) / kJoinWaves;
  const int64_t c0 = run + 1 + wave * per;
  const int64_t c1 = c0 + per < last + 1 ? c0 + per : last + 1;
  for (int col0 = blockIdx.y * 64; col0 < a.H; col0 += gridDim.y * 64) {
    const int col = col0 + lane;
    float s = 0.0f;
    if (col < a.H) {
      if (wave == 0) s = a.part[(run * 2 + 1) * a.H + col];
#pragma unroll 8
      for (int64_t c = c0; c < c1; ++c) s += a.part[c * 2 * a.H + col];
    }
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < a.H) {
      for (int w = 1; w < kJoinWaves; ++w) s += sums[w][lane];
      ((T*)a.gweight)[(int64_t)t * a.H + col] = narrow<T>(s * a.scale);
    }
    __syncthreads();
  }
}

template <typename T, int V>
__global__ __launch_bounds__(256) void k_absent(Args a) {
  const int64_t v = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v >= a.V || a.start[v] != a.start[v + 1]) return;
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = 0.0f;
  Pack<T, V> z;
  z.set(x);
  T* row = (T*)a.gweight + v * a.H;
  for (int c = (threadIdx.x & 63) * V; c < a.H; c += 64 * V) z.store(row + c);
}

}  // namespace embed
}  // namespace ews

namespace {

using namespace ews::embed;

struct EPlan {
  int64_t runs;
  int groups, R;
  size_t order, sorted, start, part, total;
};

size_t al256e(size_t x) { return (x + 255) & ~(size_t)255; }

int embed_plan(const ews_embed_desc* s, EPlan& p) {
  if (!s) return EWS_ERR_NULL;
  if (s->dtype != EWS_DTYPE_F32 && s->dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->token_bytes != 4 && s->token_bytes != 8) return EWS_ERR_OPTION;
  // a launch has fewer than 2^32 threads along x and 2^16 workgroups along y
  if (s->count < 1 || s->count > 1 << 25 || s->width < 1 || s->vocab < 1) return EWS_ERR_SHAPE;
  if (s->width > 1 << 20 || s->vocab > 1 << 25 || s->weight_stride < s->width) return EWS_ERR_SHAPE;
  // one workgroup of k_sort per CU where the vocabulary allows it; each reads all the ids
  int groups = s->vocab < 256 ? s->vocab : 256;
  const int least = (s->vocab + kMaxRange - 1) / kMaxRange;
  if (groups < least) groups = least;
  p.R = (s->vocab + groups - 1) / groups;
  p.groups = (s->vocab + p.R - 1) / p.R;
  p.runs = (s->count + kRun - 1) / kRun;
  size_t off = 0;
  p.order = off; off += al256e((size_t)s->count * 4);
  p.sorted = off; off += al256e((size_t)s->count * 4);
  p.start = off; off += al256e(((size_t)s->vocab + 1) * 4);
  p.part = off; off += al256e((size_t)p.runs * 2 * s->width * 4);
  p.total = off;
  return EWS_OK;
}

Args embed_args(const ews_embed_desc* s) {
  Args a{};
  a.n = s->count;
  a.H = s->width;
  a.V = s->vocab;
  a.stride = s->weight_stride;
  a.pad = s->padding;
  a.scale = s->scale;
  return a;
}

// Sixteen-byte accesses need every row of both sides to start at a multiple of 16 bytes.
bool rows_aligned(const ews_embed_desc* s, const void* x, const void* y, int64_t stride_x) {
  const int64_t e = s->dtype == EWS_DTYPE_F32 ? 4 : 2;
  return ((uintptr_t)x | (uintptr_t)y) % 16 == 0 && (s->width * e) % 16 == 0 && (stride_x * e) % 16 == 0;
}

template <typename T, int V>
int launch_lookup(const ews_embed_desc* s, Args a, hipStream_t st) {
  const int packs = a.H / V;
  a.lanes = 1;
  while (a.lanes < 64 && a.lanes < packs) a.lanes *= 2;
  const int64_t blocks = (a.n * a.lanes + 255) / 256;
  if (s->token_bytes == 8)
    hipLaunchKernelGGL((k_lookup<T, V, int64_t>), dim3((uint32_t)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_lookup<T, V, int32_t>), dim3((uint32_t)blocks), dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T, int V>
int launch_sums(const EPlan& p, const Args& a, hipStream_t st) {
  const int tiles = (a.H + 64 * V - 1) / (64 * V);
  hipLaunchKernelGGL((k_runs<T, V>), dim3((uint32_t)((p.runs + 3) / 4), tiles), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  const int ctiles = (a.H + 63) / 64;
  hipLaunchKernelGGL((k_join<T>), dim3((uint32_t)p.runs, ctiles < 64 ? ctiles : 64), dim3(64 * kJoinWaves), 0, st, a);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  hipLaunchKernelGGL((k_absent<T, V>), dim3((uint32_t)((a.V + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int ews_embed_forward(const ews_embed_desc* desc, const void* tokens, const void* weight, void* out,
                      ews_stream_t stream) {
  EPlan p;
  const int rc = embed_plan(desc, p);
  if (rc != EWS_OK) return rc;
  if (!tokens || !weight || !out) return EWS_ERR_NULL;
  Args a = embed_args(desc);
  a.tokens = tokens;
  a.weight = weight;
  a.out = out;
  hipStream_t st = (hipStream_t)stream;
  const bool wide = rows_aligned(desc, weight, out, desc->weight_stride);
  if (desc->dtype == EWS_DTYPE_F32)
    return wide ? launch_lookup<float, 4>(desc, a, st) : launch_lookup<float, 1>(desc, a, st);
  return wide ? launch_lookup<bf16, 8>(desc, a, st) : launch_lookup<bf16, 1>(desc, a, st);
}

size_t ews_embed_workspace_bytes(const ews_embed_desc* desc) {
  EPlan p;
  return embed_plan(desc, p) == EWS_OK ? p.total : 0;
}

int ews_embed_backward(const ews_embed_desc* desc, const void* tokens, const void* grad_out, void* grad_weight,
                       void* workspace, ews_stream_t stream) {
  EPlan p;
  const int rc = embed_plan(desc, p);
  if (rc != EWS_OK) return rc;
  if (!tokens || !grad_out || !grad_weight || !workspace) return EWS_ERR_NULL;
  Args a = embed_args(desc);
  char* w = (char*)workspace;
  a.tokens = tokens;
  a.gout = grad_out;
  a.gweight = grad_weight;
  a.R = p.R;
  a.order = (int*)(w + p.order);
  a.sorted = (int*)(w + p.sorted);
  a.start = (int*)(w + p.start);
  a.part = (float*)(w + p.part);
  hipStream_t st = (hipStream_t)stream;
  if (desc->token_bytes == 8)
    hipLaunchKernelGGL((k_sort<int64_t>), dim3(p.groups), dim3(kSortThreads), 0, st, a);
  else
    hipLaunchKernelGGL((k_sort<int32_t>), dim3(p.groups), dim3(kSortThreads), 0, st, a);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  const bool wide = rows_aligned(desc, grad_out, grad_weight, desc->width);
  if (desc->dtype == EWS_DTYPE_F32)
    return wide ? launch_sums<float, 4>(p, a, st) : launch_sums<float, 1>(p, a, st);
  return wide ? launch_sums<bf16, 8>(p, a, st) : launch_sums<bf16, 1>(p, a, st);
}

}  // extern "C"
