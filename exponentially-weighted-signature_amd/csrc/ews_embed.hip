// Embedding lookup of a token model on MI355X (gfx950), and its gradient.
//
//   forward   out[n, :] = s W[t_n, :]
//   backward  dW[v, :] = s sum_{n : t_n = v} g[n, :], zero for a token that does not occur and for the padding token
//
// Both only move rows, so memory bounds them: 131071 tokens of width 2048 in bfloat16 are looked up in 132 us, summed
// in 230 (k_runs, the bulk of it, moves 5.2 TB/s). Rows are stored past the caches, which hold what is read again
// (k_lookup 159 -> 148 us, k_runs 190 -> 158). The backward adds no number with an atomic: it sorts the positions by
// token (stable, so a token's rows are added in the order of the text) and sums runs of equal tokens, in float32,
// rounding each row of dW once. The same inputs give the same bits.
//
//   k_sort   the vocabulary is dealt to the workgroups one token at a time (frequent tokens are often neighbours). Each
//            looks through all the tokens (the ids stay in L2): its wavefronts count their own stretch's own tokens and
//            list them in LDS; from the counts every wavefront knows where its first one of each token goes. No
//            workgroup waits for another.
//   k_runs   a wavefront takes a run of sorted positions and one column tile, whatever tokens they are, so a frequent
//            token costs no more than rare ones: rows of tokens that lie inside are written, the ends of tokens that go
//            on in a neighbour's positions are kept as float32 partial rows. Further workgroups of the same launch zero
//            the rows of dW without a token.
//   k_join   adds the partial rows of the tokens that were cut, in order.
//
// Up to kFewTokens tokens need no order: k_few gives a wavefront a row of dW and a column tile, which looks through all
// the tokens and adds its own ones' rows. One launch for three and no scratch (n=64, V=100, H=64: 7 us on the host for
// 15).
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
constexpr int kListed = 640;      // own tokens a wavefront lists: of 131071, 32 where all are alike rare
constexpr int kMaxRange = 512;    // vocabulary entries a workgroup of k_sort may own
constexpr int kJoinWaves = 4;
constexpr int kFewTokens = 256;   // one wavefront would add them all in about 30 us
constexpr int kFewRows = 16;

struct Args {
  int64_t n, stride, pad;
  int H, V;
  int deal, range; // token t is entry t >> deal of workgroup t % 2^deal of k_sort, which owns 2^range (its slot)
  int lanes;       // lanes a row of the lookup is spread over
  int run;         // sorted positions a wavefront of k_runs adds up
  int runs;        // how many there are
  uint32_t tiles;  // column tiles of a row
  float scale;
  const void* tokens;
  const void* weight;
  void* out;
  const void* gout;
  void* gweight;
  int* order;      // (n) positions, sorted by token
  int* sorted;     // (n) their tokens' slots
  int* start;      // (slots + 1) first sorted position of every slot; the last: positions that count
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
  constexpr int kAhead = 4;  // loads on their way: 148 -> 132 us with four for one
  for (int c0 = lane; c0 < packs; c0 += kAhead * a.lanes) {
    Pack<T, V> p[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (known && c0 + k * a.lanes < packs) p[k].load(src + (int64_t)(c0 + k * a.lanes) * V);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int c = c0 + k * a.lanes;
      if (c >= packs) break;
      float x[V];
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = known ? p[k].get(i) * a.scale : __builtin_nanf("");
      p[k].set(x);
      p[k].store_past(dst + (int64_t)c * V);
    }
  }
}

// A token that counts, or kNone.
constexpr uint32_t kNone = ~0u;
__device__ __forceinline__ uint32_t counted(int64_t t, const Args& a) {
  return (uint64_t)t < (uint64_t)a.V && t != a.pad ? (uint32_t)t : kNone;
}

__device__ __forceinline__ int token_of(const Args& a, int slot) {
  return (slot & ((1 << a.range) - 1)) << a.deal | slot >> a.range;
}

// Places 64 positions of own tokens (entry < 0: none); equal tokens keep their order.
__device__ __forceinline__ void place(const Args& a, int entry, int position, int* next) {
  const int lane = threadIdx.x & 63;
  uint64_t left = __ballot(entry >= 0);
  while (left) {
    const int leader = __ffsll((unsigned long long)left) - 1;
    const int one = __builtin_amdgcn_readlane(entry, leader);
    const uint64_t same = __ballot(entry == one);
    const int first = next[one];
    if (entry == one) {
      const int to = first + __popcll(same & ((1ull << lane) - 1ull));
      a.order[to] = position;
      a.sorted[to] = ((int)blockIdx.x << a.range) + entry;
    }
    if (lane == leader) next[one] = first + __popcll(same);
    left &= ~same;
  }
}

template <typename Tok>
__global__ __launch_bounds__(kSortThreads) void k_sort(Args a) {
  __shared__ int next[kSortWaves][kMaxRange];    // a wavefront's occurrences, then its next place, of every own token
  __shared__ int pos[kSortWaves][kListed];       // own positions, in the order of the text
  __shared__ uint16_t ids[kSortWaves][kListed];
  __shared__ int wsum[kSortWaves];
  __shared__ int base;
  const Tok* tokens = (const Tok*)a.tokens;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t group = blockIdx.x, mask = (1u << a.deal) - 1u;
  const int range = 1 << a.range;
  for (int i = tid; i < kSortWaves * range; i += kSortThreads) next[i >> a.range][i & (range - 1)] = 0;
  if (tid == 0) base = 0;
  __syncthreads();

  // a wavefront looks through a stretch of the text: how often each own token occurs, how many tokens go to smaller
  // groups, and where its own ones are, as far as its list goes
  const int64_t each = (a.n + kSortThreads - 1) / kSortThreads * 64;
  const int64_t from = wave * each, to = from + each < a.n ? from + each : a.n;
  int below = 0, m = 0;
  constexpr int kAhead = 8;
  for (int64_t i0 = from; i0 < to; i0 += 64 * kAhead) {
    Tok t[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int64_t i = i0 + 64 * q + lane;
      t[q] = i < to ? tokens[i] : (Tok)-1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const uint32_t x = counted(t[q], a);
      below += (x & mask) < group && x != kNone;
      const bool own = (x & mask) == group && x != kNone;
      const uint64_t mine = __ballot(own);
      if (!mine) continue;
      const int at = m + __popcll(mine & ((1ull << lane) - 1ull));
      if (own) {
        const int entry = (int)(x >> a.deal);
        atomicAdd(&next[wave][entry], 1);
        if (at < kListed) {
          pos[wave][at] = (int)(i0 + 64 * q + lane);
          ids[wave][at] = (uint16_t)entry;
        }
      }
      m += __popcll(mine);
    }
  }
#pragma unroll
  for (int s = 32; s; s >>= 1) below += __shfl_xor(below, s);
  if (lane == 0) atomicAdd(&base, below);
  __syncthreads();

  // every wavefront's first place of every own token: by token, then by wavefront (one thread a token)
  int count = 0;
  if (tid < range)
    for (int w = 0; w < kSortWaves; ++w) count += next[w][tid];
  int incl = count;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int up = __shfl_up(incl, s);
    if (lane >= s) incl += up;
  }
  if (lane == 63) wsum[wave] = incl;
  __syncthreads();
  if (tid < range) {
    int first = base + incl - count;
    for (int w = 0; w < wave; ++w) first += wsum[w];
    a.start[group * range + tid] = first;
    if (group == mask && tid == range - 1) a.start[(group + 1) * range] = first + count;
    for (int w = 0; w < kSortWaves; ++w) {
      const int k = next[w][tid];
      next[w][tid] = first;
      first += k;
    }
  }
  __syncthreads();

  if (m <= kListed) {
    for (int l = lane; l - lane < m; l += 64)
      place(a, l < m ? (int)ids[wave][l] : -1, l < m ? pos[wave][l] : 0, next[wave]);
    return;
  }
  for (int64_t i0 = from; i0 < to; i0 += 64 * kAhead) {  // more than its list holds: the stretch again
    Tok t[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int64_t i = i0 + 64 * q + lane;
      t[q] = i < to ? tokens[i] : (Tok)-1;
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const uint32_t x = counted(t[q], a);
      const bool own = (x & mask) == group && x != kNone;
      place(a, own ? (int)(x >> a.deal) : -1, (int)(i0 + 64 * q + lane), next[wave]);
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void zero_absent(const Args& a, int v, int col) {
  if (v >= a.V || col >= a.H) return;
  const int slot = ((v & ((1 << a.deal) - 1)) << a.range) + (v >> a.deal);
  if (a.start[slot] != a.start[slot + 1]) return;
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = 0.0f;
  Pack<T, V> z;
  z.set(x);
  z.store_past((T*)a.gweight + (int64_t)v * a.H + col);
}

// The unit of a wavefront of workgroups of four, in the grid of unit_grid().
__device__ __forceinline__ uint32_t unit_of(int wave) { return (blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave; }

template <typename T, int V>
__global__ __launch_bounds__(256) void k_runs(Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // a row's column tiles are neighbours; run and tile are scalar, so positions and tokens are scalar loads
  const uint32_t unit = unit_of(wave);
  const int run = (int)(unit / a.tiles), col = ((int)(unit % a.tiles) * 64 + lane) * V;
  if (run >= a.runs) return zero_absent<T, V>(a, run - a.runs, col);
  const int total = a.start[1 << (a.deal + a.range)];
  const int64_t b = (int64_t)run * a.run;
  if (b >= total) return;
  const int j0 = (int)b, j1 = j0 + a.run < total ? j0 + a.run : total;
  const bool in = col < a.H;
  const T* g = (const T*)a.gout + (in ? col : 0);
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.0f;
  constexpr int kAhead = 8;
  Pack<T, V> p[kAhead];
  auto fetch = [&](int j) {
    if (j + kAhead <= j1) {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) p[q].load(g + (int64_t)a.order[j + q] * a.H);
    } else {
#pragma unroll
      for (int q = 0; q < kAhead; ++q) p[q].load(g + (int64_t)a.order[j + q < j1 ? j + q : j1 - 1] * a.H);
    }
  };
  int t = a.sorted[j0];
  for (int j = j0; j < j1; j += kAhead) {
    fetch(j);
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      if (j + q >= j1) break;
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] += p[q].get(i);
      const int now = t;
      if (j + q + 1 < j1) {
        t = a.sorted[j + q + 1];
        if (t == now) continue;
      }
      const int s0 = a.start[now], s1 = a.start[now + 1];
      if (in) {
        if (s0 >= j0 && s1 <= j1) {
          Pack<T, V> o;
          float x[V];
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] = acc[i] * a.scale;
          o.set(x);
          o.store_past((T*)a.gweight + (int64_t)token_of(a, now) * a.H + col);
        } else {
          float* part = a.part + ((int64_t)run * 2 + (s0 < j0 ? 0 : 1)) * a.H + col;
#pragma unroll
          for (int i = 0; i < V; ++i) part[i] = acc[i];
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) acc[i] = 0.0f;
    }
  }
}

template <typename T, int V, typename Tok>
__global__ __launch_bounds__(256) void k_few(Args a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t unit = unit_of(wave);
  const int v = (int)(unit / a.tiles), col = ((int)(unit % a.tiles) * 64 + lane) * V;
  if (v >= a.V) return;
  const bool in = col < a.H;
  const T* g = (const T*)a.gout + (in ? col : 0);
  const Tok* tokens = (const Tok*)a.tokens;
  Tok t[kFewTokens / 64];
#pragma unroll
  for (int q = 0; q < kFewTokens / 64; ++q) t[q] = 64 * q + lane < (int)a.n ? tokens[64 * q + lane] : (Tok)-1;
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = 0.0f;
#pragma unroll
  for (int q = 0; q < kFewTokens / 64; ++q) {
    uint64_t left = __ballot((int64_t)t[q] == v && v != a.pad);
    while (left) {
      constexpr int kAhead = 8;
      Pack<T, V> p[kAhead];
      int n = 0;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {  // the next eight, as far as there are
        const int j = __ffsll((unsigned long long)left) - 1;
        if (k == 0 || left) {
          p[k].load(g + (int64_t)(64 * q + j) * a.H);
          left &= left - 1;
          ++n;
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (k < n)
#pragma unroll
          for (int i = 0; i < V; ++i) x[i] += p[k].get(i);
    }
  }
  if (!in) return;
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] *= a.scale;
  Pack<T, V> o;
  o.set(x);
  o.store_past((T*)a.gweight + (int64_t)v * a.H + col);
}

// One workgroup per run; only those whose last token starts in them and goes on work. A token of few partial rows: the
// wavefronts take a column tile each. One of many: they add a contiguous part of its rows each, one tile after another,
// and the first one joins them.
template <typename T, int V>
__global__ __launch_bounds__(64 * kJoinWaves) void k_join(Args a) {
  __shared__ float sums[kJoinWaves][64][V];
  const int total = a.start[1 << (a.deal + a.range)];
  const int64_t run = blockIdx.x;
  const int64_t b = run * a.run;
  if (b >= total) return;
  const int j0 = (int)b, j1 = j0 + a.run < total ? j0 + a.run : total;
  const int t = a.sorted[j1 - 1];
  const int s0 = a.start[t], s1 = a.start[t + 1];
  if (s0 < j0 || s1 <= j1) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, token = token_of(a, t);
  const int rows = (int)((s1 - 1) / a.run - run);  // partial rows of the runs after this one
  const float* own = a.part + (run * 2 + 1) * a.H;
  const float* next = a.part + (run + 1) * 2 * a.H;
  auto add = [&](float (&s)[V], int c0, int c1, int col) {
#pragma unroll 16
    for (int c = c0; c < c1; ++c) {
      Pack<float, V> x;
      x.load(next + (int64_t)c * 2 * a.H + col);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += x.get(i);
    }
  };
  auto finish = [&](const float (&s)[V], int col) {
#pragma unroll
    for (int i = 0; i < V; ++i) ((T*)a.gweight)[(int64_t)token * a.H + col + i] = narrow<T>(s[i] * a.scale);
  };
  if (rows <= kFewRows) {
    const int col = ((blockIdx.y * kJoinWaves + wave) * 64 + lane) * V;
    if (col >= a.H) return;
    float s[V];
    Pack<float, V> x;
    x.load(own + col);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = x.get(i);
    add(s, 0, rows, col);
    finish(s, col);
    return;
  }
  const int per = (rows + kJoinWaves - 1) / kJoinWaves;
  const int c0 = wave * per, c1 = c0 + per < rows ? c0 + per : rows;
  for (int tile = 0; tile < kJoinWaves; ++tile) {
    const int col = ((blockIdx.y * kJoinWaves + tile) * 64 + lane) * V;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.0f;
    if (col < a.H) {
      if (wave == 0) {
        Pack<float, V> x;
        x.load(own + col);
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = x.get(i);
      }
      add(s, c0, c1, col);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[wave][lane][i] = s[i];
    __syncthreads();
    if (wave == 0 && col < a.H) {
#pragma unroll
      for (int w = 1; w < kJoinWaves; ++w)
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] += sums[w][lane][i];
      finish(s, col);
    }
    __syncthreads();
  }
}

}  // namespace embed
}  // namespace ews

namespace {

using namespace ews::embed;

struct EPlan {
  int64_t runs;
  int deal, range, run;
  size_t order, sorted, start, part, total;
};

// Units of one wavefront each (a row or run by one column tile) that a launch has. A grid's x holds fewer than 2^32
// threads, so workgroups past 2^23 go to y; their number stays below 2^32 with the last y's that are over.
constexpr int64_t kMostUnits = ((int64_t)1 << 32) - (1 << 26);

dim3 unit_grid(int64_t units) {
  const int64_t blocks = (units + 3) / 4, x = blocks < 1 << 23 ? blocks : 1 << 23;
  return dim3((uint32_t)x, (uint32_t)((blocks + x - 1) / x));
}

size_t al256e(size_t x) { return (x + 255) & ~(size_t)255; }

int embed_plan(const ews_embed_desc* s, EPlan& p) {
  if (!s) return EWS_ERR_NULL;
  if (s->dtype != EWS_DTYPE_F32 && s->dtype != EWS_DTYPE_BF16) return EWS_ERR_OPTION;
  if (s->token_bytes != 4 && s->token_bytes != 8) return EWS_ERR_OPTION;
  // a launch has fewer than 2^32 threads along x and 2^16 workgroups along y
  if (s->count < 1 || s->count > 1 << 25 || s->width < 1 || s->vocab < 1) return EWS_ERR_SHAPE;
  if (s->width > 1 << 20 || s->vocab > 1 << 25 || s->weight_stride < s->width) return EWS_ERR_SHAPE;
  // one workgroup of k_sort per CU where the vocabulary allows it; each reads all the ids
  p.deal = 0;
  while (p.deal < 8 && (1 << p.deal) < s->vocab) ++p.deal;
  while (s->vocab > (int64_t)kMaxRange << p.deal) ++p.deal;
  p.range = 0;
  while (s->vocab > (int64_t)1 << (p.deal + p.range)) ++p.range;
  // long runs cut few tokens, but two thousand wavefronts keep the memory busy
  const int64_t tiles = (s->width + (s->dtype == EWS_DTYPE_F32 ? 255 : 511)) / (s->dtype == EWS_DTYPE_F32 ? 256 : 512);
  p.run = 32;
  while (p.run > 8 && s->count / p.run * tiles < 2048) p.run /= 2;
  p.runs = (s->count + p.run - 1) / p.run;
  // with the narrowest tiles, so that what is refused does not depend on addresses, nor on the direction
  if ((p.runs + s->vocab) * ((s->width + 63) / 64) > kMostUnits) return EWS_ERR_SHAPE;
  size_t off = 0;
  if (s->count <= kFewTokens) {
    p.total = 0;
    return EWS_OK;
  }
  p.order = off; off += al256e((size_t)s->count * 4);
  p.sorted = off; off += al256e((size_t)s->count * 4);
  p.start = off; off += al256e((((size_t)1 << (p.deal + p.range)) + 1) * 4);
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
int launch_few(const ews_embed_desc* s, Args a, hipStream_t st) {
  a.tiles = (a.H + 64 * V - 1) / (64 * V);
  const dim3 grid = unit_grid((int64_t)a.V * a.tiles);
  if (s->token_bytes == 8)
    hipLaunchKernelGGL((k_few<T, V, int64_t>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_few<T, V, int32_t>), grid, dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? EWS_OK : EWS_ERR_LAUNCH;
}

template <typename T, int V>
int launch_sums(const EPlan& p, Args a, hipStream_t st) {
  a.tiles = (a.H + 64 * V - 1) / (64 * V);
  hipLaunchKernelGGL((k_runs<T, V>), unit_grid((p.runs + a.V) * a.tiles), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  const int v = a.H % 4 == 0 ? 4 : 1;  // partial rows that start at multiples of 16 bytes
  const dim3 grid((uint32_t)p.runs, (a.H + 64 * v * kJoinWaves - 1) / (64 * v * kJoinWaves));
  if (v == 4)
    hipLaunchKernelGGL((k_join<T, 4>), grid, dim3(64 * kJoinWaves), 0, st, a);
  else
    hipLaunchKernelGGL((k_join<T, 1>), grid, dim3(64 * kJoinWaves), 0, st, a);
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
  if (!tokens || !grad_out || !grad_weight || (!workspace && desc->count > kFewTokens)) return EWS_ERR_NULL;
  Args a = embed_args(desc);
  char* w = (char*)workspace;
  a.tokens = tokens;
  a.gout = grad_out;
  a.gweight = grad_weight;
  a.deal = p.deal;
  a.range = p.range;
  a.run = p.run;
  a.runs = (int)p.runs;
  a.order = (int*)(w + p.order);
  a.sorted = (int*)(w + p.sorted);
  a.start = (int*)(w + p.start);
  a.part = (float*)(w + p.part);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = rows_aligned(desc, grad_out, grad_weight, desc->width);
  if (desc->count <= kFewTokens) {
    if (desc->dtype == EWS_DTYPE_F32)
      return wide ? launch_few<float, 4>(desc, a, st) : launch_few<float, 1>(desc, a, st);
    return wide ? launch_few<bf16, 8>(desc, a, st) : launch_few<bf16, 1>(desc, a, st);
  }
  if (desc->token_bytes == 8)
    hipLaunchKernelGGL((k_sort<int64_t>), dim3(1u << p.deal), dim3(kSortThreads), 0, st, a);
  else
    hipLaunchKernelGGL((k_sort<int32_t>), dim3(1u << p.deal), dim3(kSortThreads), 0, st, a);
  if (hipGetLastError() != hipSuccess) return EWS_ERR_LAUNCH;
  if (desc->dtype == EWS_DTYPE_F32)
    return wide ? launch_sums<float, 4>(p, a, st) : launch_sums<float, 1>(p, a, st);
  return wide ? launch_sums<bf16, 8>(p, a, st) : launch_sums<bf16, 1>(p, a, st);
}

}  // extern "C"
