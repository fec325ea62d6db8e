// rows_kernels.hip — rows of a table by index (the latent codes of a batch) and the gradient of the table:
//   y[n, :] = scale T[i_n, :]          dT[v, :] = scale sum over {n : i_n = v, v != padding} of g[n, :]
// Both move memory and nothing else.  An index outside [0, rows) reads nothing: its output row is NaN, and it adds nothing to the
// gradient.  The gradient adds the rows of one index in the order of their positions, in fp32, whatever the grid looks like: two
// runs give the same bits (no atomics).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "capi_common.h"
#include "train_ops_common.h"

namespace nphm {
namespace train_ops {

struct LookupArgs {
  const void* table;
  const void* idx;
  void* out;
  int64_t ld;          // elements between rows of the table
  int64_t count;       // indices
  int64_t rows;
  int dim;
  int idx64;
  float scale;
};

__device__ __forceinline__ int64_t load_index(const void* idx, int idx64, int64_t n) {
  return idx64 ? static_cast<const int64_t*>(idx)[n] : int64_t(static_cast<const int*>(idx)[n]);
}

// A group of LPR lanes takes one row (LPR * 16 bytes of it at a time); a wavefront 64 / LPR rows, so that narrow rows fill it too.  Few rows
// are cut along blockIdx.y.  Bound by memory: 16384 rows of 4096 bf16 out of 50000 take 44.8 us, 248 MB at 5.5 TB/s (a copy: 5.1).  IN, from rows
// and result together that fill the last cache: rows are not kept once read (54.6 us if they are; with a call behind it that reads the
// result 81 and 86; 8192 rows, which fit: 24.6 and 21.5; 65536, some of them named twice: 201 and 177).  OUT, from a result that fills
// it by itself: nor is that kept (65536 rows and a call that reads them: 345 us, 353 if it is).
template <class T, int LPR, bool IN, bool OUT>
__global__ __launch_bounds__(256) void lookup_kernel(LookupArgs p) {
  constexpr int V = Vec<T>::N, ROWS = 256 / LPR;
  typedef typename Vec<T>::type vec;
  const int sub = threadIdx.x % LPR;
  const int64_t n = int64_t(blockIdx.x) * ROWS + threadIdx.x / LPR;
  if (n >= p.count) return;
  const int64_t i = load_index(p.idx, p.idx64, n);
  const bool ok = i >= 0 && i < p.rows;
  const T* src = static_cast<const T*>(p.table) + (ok ? i : 0) * p.ld;
  T* dst = static_cast<T*>(p.out) + n * p.dim;
  const int full = p.dim / V * V;
  for (int c = (blockIdx.y * LPR + sub) * V; c < full; c += gridDim.y * LPR * V) {
    vec v;
    if (ok) v = load_vec<IN>(src + c);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = ok ? T(float(v[k]) * p.scale) : T(__builtin_nanf(""));
    store_vec<OUT>(dst + c, v);
  }
  if (blockIdx.y == 0) {
    const int c = full + sub;                       // V - 1 elements at most, LPR >= 8 lanes
    if (c < p.dim) dst[c] = ok ? T(float(src[c]) * p.scale) : T(__builtin_nanf(""));
  }
}

struct EntryArgs {
  const void* grad;    // [count, dim], rows ld apart
  const void* idx;
  int64_t* index;      // [count]
  void* values;        // [count, dim]
  int64_t ld, count, rows, padding;
  int dim, idx64;
  float scale;
};

// The gradient of the table with an entry for every index: the lookup's copy the other way round.  What must not count (padding, outside
// the table) becomes an entry of zeros for row 0, so that nobody has to know on the host how many there are.
template <class T, int LPR>
__global__ __launch_bounds__(256) void entries_kernel(EntryArgs p) {
  constexpr int V = Vec<T>::N, ROWS = 256 / LPR;
  typedef typename Vec<T>::type vec;
  const int sub = threadIdx.x % LPR;
  const int64_t n = int64_t(blockIdx.x) * ROWS + threadIdx.x / LPR;
  if (n >= p.count) return;
  const int64_t i = load_index(p.idx, p.idx64, n);
  const bool ok = i >= 0 && i < p.rows && i != p.padding;
  const T* src = static_cast<const T*>(p.grad) + n * p.ld;
  T* dst = static_cast<T*>(p.values) + n * p.dim;
  const int full = p.dim / V * V;
  for (int c = (blockIdx.y * LPR + sub) * V; c < full; c += gridDim.y * LPR * V) {
    vec v = *reinterpret_cast<const vec*>(src + c);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = ok ? T(float(v[k]) * p.scale) : T(0.f);
    *reinterpret_cast<vec*>(dst + c) = v;
  }
  if (blockIdx.y == 0) {
    const int c = full + sub;                       // V - 1 elements at most, LPR >= 8 lanes
    if (c < p.dim) dst[c] = ok ? T(float(src[c]) * p.scale) : T(0.f);
    if (sub == 0) p.index[n] = ok ? i : 0;
  }
}

struct GradArgs {
  const void* grad;    // [count, dim], rows ld apart
  const void* idx;
  void* out;           // [rows, dim]; merging: [count, dim]
  int64_t ld, count, rows;
  int dim, idx64;
  int64_t padding;     // -1: none
  float scale;
};

template <class T>
__device__ __forceinline__ void load_cols(float (&v)[Vec<T>::N], const T* row, int c, int dim) {
  constexpr int V = Vec<T>::N;
  if (c + V <= dim) {
    const typename Vec<T>::type x = *reinterpret_cast<const typename Vec<T>::type*>(row + c);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = float(x[k]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = c + k < dim ? float(row[c + k]) : 0.f;
  }
}
template <class T, bool STREAM = false>
__device__ __forceinline__ void store_cols(T* row, int c, int dim, const float (&v)[Vec<T>::N], float scale) {
  constexpr int V = Vec<T>::N;
  if (c + V <= dim) {
    typename Vec<T>::type x;
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = T(v[k] * scale);
    store_vec<STREAM>(row + c, x);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) if (c + k < dim) row[c + k] = T(v[k] * scale);
  }
}

// `count` elements from `to` on become zeros, by `threads` threads of which this is number `t`: whole 16-byte places but for the ends
template <bool STREAM, class T>
__device__ __forceinline__ void zero_run(T* to, int64_t count, int t, int threads) {
  constexpr int V = Vec<T>::N;
  const int head = int(min(count, int64_t((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15) / int64_t(sizeof(T))));
  const int64_t whole = (count - head) / V;
  for (int64_t i = t; i < whole; i += threads) store_vec<STREAM>(to + head + i * V, typename Vec<T>::type{});
  if (t < head) to[t] = T(0.f);
  const int64_t last = head + whole * V + t;
  if (last < count) to[last] = T(0.f);                               // (V - 1 elements at most on either end, at least 64 threads)
}

// ---- few indices: no sorting ----------------------------------------------------------------------------------------------------
// One launch.  A block owns `rows_each` rows of the table (one, if a row is longer than SPAN vectors: then blockIdx.y cuts it into pieces of
// them) and makes one run of zeros of them; one thread an index finds out which indices fall into them, and then each row that is named
// becomes the sum of its own, in the order of the indices.
constexpr int FEW = 256, SPAN = 1024;

template <class T, bool OUT>
__global__ __launch_bounds__(256) void grad_few_kernel(GradArgs p, int rows_each) {
  constexpr int V = Vec<T>::N;
  __shared__ uint64_t found[4], lead[4];
  __shared__ int64_t index[FEW];
  const int t = threadIdx.x;
  const int64_t v0 = int64_t(blockIdx.x) * rows_each, v1 = min(p.rows, v0 + rows_each);
  const int c0 = blockIdx.y * (SPAN * V), c1 = min(p.dim, c0 + SPAN * V);
  const int64_t i = t < p.count ? load_index(p.idx, p.idx64, t) : -1;
  index[t] = i;
  const bool in = i >= v0 && i < v1 && i != p.padding;
  const uint64_t hit = __ballot(in);
  if ((t & 63) == 0) found[t >> 6] = hit;
  T* out = static_cast<T*>(p.out);
  if (c0 == 0 && c1 == p.dim) zero_run<OUT>(out + v0 * p.dim, (v1 - v0) * p.dim, t, 256);
  else zero_run<OUT>(out + v0 * p.dim + c0, c1 - c0, t, 256);             // (one row)
  __syncthreads();
  if (!(found[0] | found[1] | found[2] | found[3])) return;
  bool leads = in;                                                   // the first index of its row
  for (int n = 0; leads && n < t; ++n) leads = index[n] != i;
  const uint64_t leader = __ballot(leads);
  if ((t & 63) == 0) lead[t >> 6] = leader;
  __syncthreads();                                                   // (orders the sums below behind the zeros, too)
  for (int u = 0; u < 4; ++u) {
    uint64_t rows = lead[u];
    while (rows) {
      const int first = u * 64 + __builtin_ctzll(rows);
      rows &= rows - 1;
      const int64_t v = index[first];
      for (int c = c0 + t * V; c < c1; c += 256 * V) {
        float acc[V] = {};
        for (int w = u; w < 4; ++w) {
          uint64_t mask = found[w];
          while (mask) {
            const int n = w * 64 + __builtin_ctzll(mask);
            mask &= mask - 1;
            if (index[n] != v) continue;
            float x[V];
            load_cols(x, static_cast<const T*>(p.grad) + n * p.ld, c, p.dim);
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += x[k];
          }
        }
        store_cols(out + v * p.dim, c, p.dim, acc, p.scale);
      }
    }
  }
}

// merging few: one wavefront a row and 64 vectors of its columns; all but the first row of an index become zeros
template <class T>
__global__ __launch_bounds__(256) void merge_few_kernel(GradArgs p) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & 63;
  const int64_t own = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (own >= p.count) return;
  const int64_t v = load_index(p.idx, p.idx64, own);
  const int c = (blockIdx.y * 64 + lane) * V;
  float acc[V] = {};
  for (int64_t n0 = 0; n0 < p.count; n0 += 64) {
    const int64_t n = n0 + lane;
    uint64_t hit = __ballot(n < p.count && load_index(p.idx, p.idx64, n < p.count ? n : 0) == v);
    if (hit && n0 + __builtin_ctzll(hit) < own) break;               // an earlier row owns the sum (nothing was added yet)
    while (hit) {
      const int b = __builtin_ctzll(hit);
      hit &= hit - 1;
      float x[V];
      load_cols(x, static_cast<const T*>(p.grad) + (n0 + b) * p.ld, c, p.dim);
#pragma unroll
      for (int k = 0; k < V; ++k) acc[k] += x[k];
    }
  }
  store_cols(static_cast<T*>(p.out) + own * p.dim, c, p.dim, acc, 1.f);
}

// ---- the indices, sorted ---------------------------------------------------------------------------------------------------------
// A stable sort of the keys with their positions; keys that must not count (padding, outside the table) become `rows`, behind all others.
__device__ __forceinline__ int key_of(const GradArgs& p, int64_t n) {
  const int64_t i = load_index(p.idx, p.idx64, n);
  return int(i < 0 || i >= p.rows || i == p.padding ? p.rows : i);
}

struct SortArgs {
  int *sorted, *perm;                  // [count]
  int *sorted2, *perm2;                // the other end of a radix pass
  int* hist;                           // [blocks][1 << digit bits]
  int shift, bits, per_block, blocks;
};

// The rows that no index names are zeros: the launches that sort, which leave most of the chip idle, clear the result with the blocks
// behind their own, a share each.  Either all of it, and the sums are written over it, or, where rows are long and enough of them are
// named, only the others: the first launch writes a place where it met a row to mark[row], and a row is named if the place that its
// mark holds names it (so marks are never cleared: whatever an untouched one holds, its place is looked up).  In units of 16 bits.
struct Zero {
  void* out;
  int64_t first, last;                 // with marks: rows
  int blocks;                          // the launch's own, in front
  const int* mark;                     // null: all is cleared
  int each;                            // rows a wavefront
  int64_t row;                         // units of one
};
constexpr int64_t ZERO_UNITS = 32768;                                // 64 KiB a block
template <bool OUT>
__device__ __forceinline__ bool cleared(const GradArgs& p, const Zero& z) {      // whether this was one of the blocks that clear
  if (int(blockIdx.x) < z.blocks) return false;
  if (z.mark) {
    const int lane = threadIdx.x & 63;
    const int64_t v0 = z.first + (int64_t(blockIdx.x - z.blocks) * (blockDim.x >> 6) + (threadIdx.x >> 6)) * z.each, v = v0 + lane;
    bool open = lane < z.each && v < z.last;
    if (open) {
      const int m = z.mark[v];
      open = m < 0 || m >= p.count || key_of(p, m) != v;
    }
    for (uint64_t rows = __ballot(open); rows; rows &= rows - 1)
      zero_run<OUT>(static_cast<bf16*>(z.out) + (v0 + __builtin_ctzll(rows)) * z.row, z.row, lane, 64);
    return true;
  }
  const int64_t at = z.first + int64_t(blockIdx.x - z.blocks) * ZERO_UNITS;
  zero_run<OUT>(static_cast<bf16*>(z.out) + at, min(ZERO_UNITS, z.last - at), threadIdx.x, blockDim.x);
  return true;
}

// Up to MIDDLE keys: a key's place is the number of keys before it.  A block places 16 keys: all keys are in LDS, its 64 rows of 16 lanes
// count over a 64th of them each (a read of four keys is the same for 16 lanes).  count^2 comparisons spread over the chip, one
// launch: 8.6 us for 4097 keys (14 with four wavefronts a block: one a SIMD waits for every read); a whole gradient of 8192 rows of
// 64 takes 21 us against 27 with the radix passes below, of 15000 rows 45 against 31.
constexpr int MIDDLE = 8192, PLACED = 16, RANGE = 64;               // keys a block places; ranges that all keys are cut into

__host__ __device__ inline int rank_room(int count) { return (count + 4 * RANGE - 1) / (4 * RANGE) * (4 * RANGE); }     // (whole reads a range)

template <bool OUT>
__global__ __launch_bounds__(PLACED * RANGE) void rank_kernel(GradArgs p, SortArgs s, Zero z) {
  extern __shared__ __attribute__((aligned(16))) int all[];
  __shared__ int part[RANGE][PLACED];
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  if (cleared<OUT>(p, z)) return;
  const int count = int(p.count), padded = rank_room(count), each = padded / RANGE;
#pragma unroll 8
  for (int n = threadIdx.x; n < padded; n += PLACED * RANGE) all[n] = n < count ? key_of(p, n) : 0x7ffffffe;
  __syncthreads();
  const int range = threadIdx.x / PLACED, own0 = blockIdx.x * PLACED, i = own0 + threadIdx.x % PLACED;
  const int own = all[i];
  const i32x4* k = reinterpret_cast<const i32x4*>(all + range * each);
  int before = 0;
  // an equal key in front counts: those before the block's own keys all do, those behind none, the block's own by their place.  Each range
  // starts one read further on than the one before it: the ranges of a wavefront then meet different banks.
  const int reads = each / 4;
  int u = range % reads;
#pragma unroll 8
  for (int step = 0; step < reads; ++step) {
    const i32x4 v = k[u];
    const int bound = range * each + 4 * u < own0 ? own + 1 : own;
#pragma unroll
    for (int e = 0; e < 4; ++e) before += v[e] < bound;
    u = u + 1 == reads ? 0 : u + 1;
  }
  if (range == 0)
#pragma unroll
    for (int e = 0; e < PLACED; ++e) before += own0 + e < i && all[own0 + e] == own;
  part[range][threadIdx.x % PLACED] = before;
  __syncthreads();
  if (threadIdx.x < PLACED && i < count) {
    int at = 0;
#pragma unroll
    for (int w = 0; w < RANGE; ++w) at += part[w][threadIdx.x];
    s.sorted[at] = own;
    s.perm[at] = i;
  }
}

// More: radix passes of up to 9 bits, least first.  hist: how often each block of keys has each digit.  The first pass takes its keys from
// the indices.
constexpr int MAX_DIGIT = 9;

template <bool FIRST, bool OUT>
__global__ __launch_bounds__(1024) void radix_hist_kernel(GradArgs p, const int* __restrict__ keys, SortArgs s, int* mark, Zero z) {
  __shared__ int bins[1 << MAX_DIGIT];
  if (cleared<OUT>(p, z)) return;
  const int digits = 1 << s.bits, t = threadIdx.x;
  for (int d = t; d < digits; d += 1024) bins[d] = 0;
  __syncthreads();
  const int64_t first = int64_t(blockIdx.x) * s.per_block;
  for (int u = t; u < s.per_block; u += 1024) {
    if (first + u >= p.count) break;
    const int key = FIRST ? key_of(p, first + u) : keys[first + u];
    atomicAdd(&bins[(key >> s.shift) & (digits - 1)], 1);
    if (FIRST && mark && key < p.rows) mark[key] = int(first + u);   // (any of them)
  }
  __syncthreads();
  for (int d = t; d < digits; d += 1024) s.hist[blockIdx.x * digits + d] = bins[d];
}

// Every block finds where its keys of each digit begin (the digits below it in all blocks, its own in the blocks before), then places its
// keys in order, 1024 at a time: in a wavefront the lanes of one digit find each other by ballots, wavefront follows wavefront.
template <bool FIRST, bool OUT>
__global__ __launch_bounds__(1024) void radix_place_kernel(GradArgs p, const int* __restrict__ keys, const int* __restrict__ perm, SortArgs s,
                                                           int* __restrict__ keys_out, int* __restrict__ perm_out, Zero z) {
  __shared__ int base[1 << MAX_DIGIT], scan[1 << MAX_DIGIT], seen[16][1 << MAX_DIGIT];
  if (cleared<OUT>(p, z)) return;
  const int digits = 1 << s.bits, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  {
    // 1024 / digits threads a digit, each over every so many blocks
    const int d = t & (digits - 1), side = 1024 >> s.bits, k = t >> s.bits;
    int total = 0, before = 0;
#pragma unroll 8
    for (int b = k; b < s.blocks; b += side) {
      const int h = s.hist[b * digits + d];
      total += h;
      before += b < int(blockIdx.x) ? h : 0;
    }
    int* totals = &seen[0][0];                                       // [1024] and [1024] of its 8192
    totals[t] = total;
    totals[1024 + t] = before;
    __syncthreads();
    if (t < digits) {
      total = before = 0;
      for (int q = 0; q < side; ++q) total += totals[(q << s.bits) + t], before += totals[1024 + (q << s.bits) + t];
      base[t] = before;
      scan[t] = total;
    }
    __syncthreads();
  }
  for (int o = 1; o < digits; o <<= 1) {
    const int v = t < digits && t >= o ? scan[t - o] : 0;
    __syncthreads();
    if (t < digits) scan[t] += v;
    __syncthreads();
  }
  if (t > 0 && t < digits) base[t] += scan[t - 1];
  const int64_t first = int64_t(blockIdx.x) * s.per_block;
  for (int u = 0; u < s.per_block; u += 1024) {
    const int64_t n = first + u + t;
    const bool in = n < p.count;
    const int key = !in ? 0 : FIRST ? key_of(p, n) : keys[n], d = (key >> s.shift) & (digits - 1);
    for (int q = t; q < 16 * digits; q += 1024) seen[q >> s.bits][q & (digits - 1)] = 0;
    __syncthreads();
    uint64_t mates = __ballot(in);
    for (int b = 0; b < s.bits; ++b) {
      const uint64_t ones = __ballot((d >> b) & 1);
      mates &= (d >> b) & 1 ? ones : ~ones;
    }
    const int ahead = __popcll(mates & ((uint64_t(1) << lane) - 1));
    if (in && ahead == 0) seen[wave][d] = __popcll(mates);
    __syncthreads();
    if (t < digits) {
      int at = base[t];
      for (int w = 0; w < 16; ++w) {
        const int h = seen[w][t];
        seen[w][t] = at;
        at += h;
      }
      base[t] = at;
    }
    __syncthreads();
    if (in) {
      const int at = seen[wave][d] + ahead;
      keys_out[at] = key;
      perm_out[at] = FIRST ? int(n) : perm[n];
    }
    __syncthreads();
  }
}

// ---- sums over runs of equal keys --------------------------------------------------------------------------------------------------
// A wavefront adds the rows of `chunk` consecutive places (64 vectors of columns): a run that lies inside goes out, one that the
// chunk's borders cut goes to partial[2 chunk + (begun before ? 0 : 1)] in fp32; join adds those in order, from the chunk where the run
// begins.  So a row that takes half of all indices costs no more than any other half.
// Bound by memory: 32768 rows of 2048 bf16 for 50000, 34 us (134 MB read once, named rows written once); sorting takes 36 with the clearing
// beside it and joining 8, most of it the way through six launches.  IN, where gradient and result do not fit into the last cache: rows
// are not kept once read (the whole: 96 us if they are, 83 so; 16384 rows of 1024, which fit: 44.3 and 46.6); OUT, nor is a result that does
// not fit by itself (32768 rows of 2048 into 100000 and a norm over it: 217 us if it is, 192 so).
struct SumArgs {
  const int *sorted, *perm;
  float* partial;
  int chunk, chunks, tiles;
  int64_t pitch;                       // floats a partial row
};

template <class T, bool STREAM>
__device__ __forceinline__ typename Vec<T>::type load_raw(const T* row, int c, int dim) {
  constexpr int V = Vec<T>::N;
  typename Vec<T>::type x;
  if (c + V <= dim) {
    x = load_vec<STREAM>(row + c);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) x[k] = c + k < dim ? row[c + k] : T(0.f);
  }
  return x;
}

template <class T, bool MERGE, bool IN, bool OUT>
__global__ __launch_bounds__(256) void sum_kernel(GradArgs p, SumArgs s) {
  constexpr int V = Vec<T>::N, AHEAD = 8;                            // rows on their way
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  T* out = static_cast<T*>(p.out);
  const T* grad = static_cast<const T*>(p.grad);
  const int64_t task = int64_t(blockIdx.x) * 4 + wave;
  if (task >= int64_t(s.chunks) * s.tiles) return;
  const int chunk = int(task / s.tiles), c = (int(task % s.tiles) * 64 + lane) * V;
  const int64_t p0 = int64_t(chunk) * s.chunk;
  const int n = int(min(p.count - p0, int64_t(s.chunk)));            // 64 at most: a lane holds a place's key and row
  const int keys = s.sorted[p0 + min(lane, n - 1)], rows = s.perm[p0 + min(lane, n - 1)];
  const int before = p0 > 0 ? s.sorted[p0 - 1] : -1, after = p0 + n < p.count ? s.sorted[p0 + n] : -1;
  const int live = __popcll(__ballot(lane < n && keys < p.rows));    // the places that count are in front
  if (!live) return;
  float acc[V] = {};
  int key = __builtin_amdgcn_readlane(keys, 0), head = __builtin_amdgcn_readlane(rows, 0);
  bool begun = before == key;
  auto flush = [&](bool goes_on) __attribute__((always_inline)) {
    if (!begun && !goes_on) {
      store_cols<T, OUT>(out + int64_t(MERGE ? head : key) * p.dim, c, p.dim, acc, p.scale);
    } else {
      float* to = s.partial + (2 * int64_t(chunk) + (begun ? 0 : 1)) * s.pitch + c;
      typedef float f32x4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int k = 0; k < V; k += 4) *reinterpret_cast<f32x4*>(to + k) = f32x4{acc[k], acc[k + 1], acc[k + 2], acc[k + 3]};
    }
  };
  typename Vec<T>::type x[AHEAD];
  for (int q = 0; q < live; q += AHEAD) {
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) x[a] = load_raw<T, IN>(grad + int64_t(__builtin_amdgcn_readlane(rows, min(q + a, live - 1))) * p.ld, c, p.dim);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
      if (q + a >= live) break;
      const int k = __builtin_amdgcn_readlane(keys, q + a);
      if (k != key) {
        flush(false);
        key = k;
        head = __builtin_amdgcn_readlane(rows, q + a);
        begun = false;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += float(x[a][e]);
    }
  }
  flush(live == n && after == key);
}

// A block a chunk, most of which have nothing to join (eight chunks a block: 10.2 us for the 4 of 4097 indices, one run waits for another).
constexpr int JOINERS = 8;             // wavefronts that join a run

template <class T, bool MERGE>
__global__ __launch_bounds__(64 * JOINERS) void join_kernel(GradArgs p, SumArgs s) {
  constexpr int V = Vec<T>::N;
  __shared__ float part[JOINERS - 1][64][V];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int chunk = blockIdx.x, c = (blockIdx.y * 64 + lane) * V;
  const int64_t p0 = int64_t(chunk) * s.chunk, p1 = min(p.count, p0 + s.chunk);
  const int key = s.sorted[p1 - 1];
  if (p1 >= p.count || key >= p.rows || s.sorted[p1] != key) return;             // its last run does not go on
  if (s.sorted[p0] == key && p0 > 0 && s.sorted[p0 - 1] == key) return;          // it began before this chunk
  int last = chunk;                                                              // the chunk where it ends
  for (;;) {
    const int64_t at = int64_t(last + 1 + lane) * s.chunk;
    const uint64_t on = __ballot(at < p.count && s.sorted[at < p.count ? at : 0] == key);
    const int run = on == ~uint64_t(0) ? 64 : __builtin_ctzll(~on);
    last += run;
    if (run < 64) break;
  }
  const int n = last - chunk, each = (n + JOINERS - 1) / JOINERS, from = chunk + 1 + wave * each, to = min(last + 1, from + each);
  float acc[V] = {};
  auto add = [&](int64_t row) __attribute__((always_inline)) {
    const float* q = s.partial + row * s.pitch + c;
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += q[k];
  };
  if (wave == 0) add(2 * int64_t(chunk) + 1);
#pragma unroll 8
  for (int k = from; k < to; ++k) add(2 * int64_t(k));
  if (wave) {
#pragma unroll
    for (int k = 0; k < V; ++k) part[wave - 1][lane][k] = acc[k];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < JOINERS - 1; ++w)
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] += part[w][lane][k];
  int64_t row = key;
  if constexpr (MERGE) {                                                         // the run's first place in this chunk (chunks have 64 at most)
    const uint64_t in = __ballot(p0 + lane < p1 && s.sorted[p0 + lane < p1 ? p0 + lane : p0] == key);
    row = s.perm[p0 + __builtin_ctzll(in)];
  }
  store_cols(static_cast<T*>(p.out) + row * p.dim, c, p.dim, acc, p.scale);
}

struct GradPlan {
  int passes, bits, blocks, per_block, chunk, chunks, tiles;
  bool marks;
  size_t sorted, perm, sorted2, perm2, hist, mark, partial, total;
};
inline GradPlan grad_plan(int64_t rows, int64_t dim, int64_t count, int element) {
  GradPlan g{};
  if (count <= FEW) return g;
  auto up = [](size_t v) { return (v + 255) / 256 * 256; };
  int bits = 1;
  while ((int64_t(1) << bits) <= rows) ++bits;
  g.passes = count <= MIDDLE ? 0 : (bits + MAX_DIGIT - 1) / MAX_DIGIT;
  g.bits = g.passes ? (bits + g.passes - 1) / g.passes : 0;
  g.per_block = int(((count + 255) / 256 + 1023) / 1024 * 1024);
  g.blocks = int((count + g.per_block - 1) / g.per_block);
  const int vec = 16 / element;
  g.tiles = int((dim + 64 * vec - 1) / (64 * vec));
  g.chunk = 8;
  // the longest chunks (fewer cut runs) that still make 4096 wavefronts: 32768 rows of 2048 bf16 take 99 us in chunks of 64 (2048
  // wavefronts), 71 in chunks of 32, 75 in chunks of 16
  while (g.chunk < 64 && count / (2 * g.chunk) * g.tiles >= 4096) g.chunk *= 2;
  g.chunks = int((count + g.chunk - 1) / g.chunk);
  const size_t ints = up(size_t(count) * 4), other = g.passes > 1 ? ints : 0;
  g.sorted = 0;
  g.perm = ints;
  g.sorted2 = 2 * ints;
  g.perm2 = g.sorted2 + other;
  g.hist = g.perm2 + other;
  // a look at each row for those that need not be cleared (50000 x 2048 bf16, 32768 skewed indices: 100.7 us without, 96.4 with)
  g.marks = g.passes && dim * element >= 1024 && count >= rows / 8;
  g.mark = g.hist + (g.passes ? up(size_t(g.blocks) * 4 << g.bits) : 0);
  g.partial = g.mark + (g.marks ? up(size_t(rows) * 4) : 0);
  g.total = g.partial + up(size_t(2) * g.chunks * g.tiles * 64 * vec * 4);
  return g;
}

template <class T, bool MERGE, bool OUT>
inline void grad_run(hipStream_t st, const GradArgs& a, const GradPlan& g, char* ws) {
  const unsigned tiles = unsigned((a.dim + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N));
  const int64_t out_rows = MERGE ? a.count : a.rows;
  if (a.count <= FEW) {
    if constexpr (MERGE) {
      hipLaunchKernelGGL((merge_few_kernel<T>), dim3(unsigned((out_rows + 3) / 4), tiles), dim3(256), 0, st, a);
    } else {
      // up to 64 KiB of rows a block, as long as there are 1024 blocks
      const int span = SPAN * Vec<T>::N;
      const int64_t fit = a.dim <= span ? 65536 / (int64_t(a.dim) * int64_t(sizeof(T))) : 1, each = std::max<int64_t>(1, std::min(a.rows / 1024, fit));
      hipLaunchKernelGGL((grad_few_kernel<T, OUT>), dim3(unsigned((a.rows + each - 1) / each), unsigned((a.dim + span - 1) / span)), dim3(256), 0, st, a,
                         int(each));
    }
    return;
  }
  SortArgs s{};
  s.sorted = reinterpret_cast<int*>(ws + g.sorted);
  s.perm = reinterpret_cast<int*>(ws + g.perm);
  s.sorted2 = reinterpret_cast<int*>(ws + g.sorted2);
  s.perm2 = reinterpret_cast<int*>(ws + g.perm2);
  s.hist = reinterpret_cast<int*>(ws + g.hist);
  s.bits = g.bits;
  s.per_block = g.per_block;
  s.blocks = g.blocks;
  // launch k of `launches` clears its share with the blocks behind its own
  const int launches = g.passes ? 2 * g.passes : 1;
  const int64_t units = out_rows * a.dim * int64_t(sizeof(T) / 2), share = (units / launches + ZERO_UNITS) / ZERO_UNITS * ZERO_UNITS;
  int* const marks = !MERGE && g.marks ? reinterpret_cast<int*>(ws + g.mark) : nullptr;
  auto zero = [&](int k, int blocks, unsigned& grid) {
    if (marks) {                                                     // (not in the first launch: it makes the marks)
      const int64_t each = std::max<int64_t>(1, std::min<int64_t>(64, 8192 / (a.dim * int64_t(sizeof(T))))), block = 16 * each;
      const int64_t part = (a.rows / (launches - 1) + block) / block * block;
      Zero z{a.out, k ? std::min(a.rows, (k - 1) * part) : 0, std::min(a.rows, k * part), blocks, marks, int(each), a.dim * int64_t(sizeof(T) / 2)};
      grid = unsigned(blocks + (z.last - z.first + block - 1) / block);
      return z;
    }
    Zero z{a.out, std::min(units, k * share), std::min(units, (k + 1) * share), blocks, nullptr, 0, 0};
    grid = unsigned(blocks + (z.last - z.first + ZERO_UNITS - 1) / ZERO_UNITS);
    return z;
  };
  unsigned grid = 0;
  if (!g.passes) {
    const Zero z = zero(0, int((a.count + PLACED - 1) / PLACED), grid);
    hipLaunchKernelGGL((rank_kernel<OUT>), dim3(grid), dim3(PLACED * RANGE), unsigned(rank_room(int(a.count)) * 4), st, a, s, z);
  }
  const int *kin = nullptr, *pin = nullptr;
  for (int pass = 0; pass < g.passes; ++pass) {                      // indices -> other -> ... -> sorted, whatever the number of passes
    const bool to_sorted = (g.passes - 1 - pass) % 2 == 0;
    int *kout = to_sorted ? s.sorted : s.sorted2, *pout = to_sorted ? s.perm : s.perm2;
    s.shift = pass * g.bits;
    Zero z = zero(2 * pass, g.blocks, grid);
    if (pass == 0) hipLaunchKernelGGL((radix_hist_kernel<true, OUT>), dim3(grid), dim3(1024), 0, st, a, kin, s, marks, z);
    else hipLaunchKernelGGL((radix_hist_kernel<false, OUT>), dim3(grid), dim3(1024), 0, st, a, kin, s, marks, z);
    z = zero(2 * pass + 1, g.blocks, grid);
    if (pass == 0) hipLaunchKernelGGL((radix_place_kernel<true, OUT>), dim3(grid), dim3(1024), 0, st, a, kin, pin, s, kout, pout, z);
    else hipLaunchKernelGGL((radix_place_kernel<false, OUT>), dim3(grid), dim3(1024), 0, st, a, kin, pin, s, kout, pout, z);
    kin = kout;
    pin = pout;
  }
  SumArgs u{};
  u.sorted = s.sorted;
  u.perm = s.perm;
  u.partial = reinterpret_cast<float*>(ws + g.partial);
  u.chunk = g.chunk;
  u.chunks = g.chunks;
  u.tiles = g.tiles;
  u.pitch = int64_t(g.tiles) * 64 * Vec<T>::N;
  const dim3 wide(unsigned((int64_t(g.chunks) * g.tiles + 3) / 4));
  if (OUT || (a.count + out_rows) * a.dim * int64_t(sizeof(T)) > CACHED) hipLaunchKernelGGL((sum_kernel<T, MERGE, true, OUT>), wide, dim3(256), 0, st, a, u);
  else hipLaunchKernelGGL((sum_kernel<T, MERGE, false, OUT>), wide, dim3(256), 0, st, a, u);
  hipLaunchKernelGGL((join_kernel<T, MERGE>), dim3(unsigned(g.chunks), tiles), dim3(64 * JOINERS), 0, st, a, u);
}

// max-norm: rows that an index names are flagged, then each flagged row is rescaled ONCE however often it is named
__global__ __launch_bounds__(256) void flags_clear_kernel(uint8_t* flags, int64_t rows) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows; i += int64_t(gridDim.x) * 256) flags[i] = 0;
}
__global__ __launch_bounds__(256) void flags_mark_kernel(const void* idx, int idx64, int64_t count, uint8_t* flags, int64_t rows) {
  const int64_t n = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (n >= count) return;
  const int64_t i = load_index(idx, idx64, n);
  if (i >= 0 && i < rows) flags[i] = 1;
}
template <class T>
__global__ __launch_bounds__(256) void renorm_kernel(T* table, int64_t ld, int64_t rows, int dim, const uint8_t* flags, float max_norm) {
  const int lane = threadIdx.x & 63;
  const int64_t v = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (v >= rows || !flags[v]) return;
  T* row = table + v * ld;
  double s = 0;
  for (int c = lane; c < dim; c += 64) { const double x = float(row[c]); s += x * x; }
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
  const double norm = sqrt(s);
  if (!(norm > double(max_norm))) return;
  const float f = float(double(max_norm) / (norm + 1e-7));
  for (int c = lane; c < dim; c += 64) row[c] = T(float(row[c]) * f);
}

constexpr int64_t MAX_ROWS = (int64_t(1) << 26) - 4;      // a wavefront a row: fewer than 2^32 threads in a launch

// f(lanes a row, grid) for `count` rows of `vecs` vectors
template <class F>
inline void for_rows(int64_t count, int64_t vecs, F&& f) {
  const int64_t blocks = (count + 3) / 4, cuts = std::max<int64_t>(1, std::min<int64_t>((vecs + 63) / 64, 1024 / blocks));
  if (vecs <= 8) f(std::integral_constant<int, 8>{}, dim3(unsigned((count + 31) / 32)));
  else if (vecs <= 16) f(std::integral_constant<int, 16>{}, dim3(unsigned((count + 15) / 16)));
  else f(std::integral_constant<int, 64>{}, dim3(unsigned(blocks), unsigned(cuts)));
}

inline int check_table(const char* what, const void* table, int64_t rows, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits,
                       int64_t count) {
  static thread_local char msg[160];
  const char* why = nullptr;
  if (!dtype_ok(dtype)) why = "dtype is 0 (fp32), 1 (bf16) or 2 (fp16)";
  else if (idx_bits != 32 && idx_bits != 64) why = "indices have 32 or 64 bits";
  else if (rows < 1 || dim < 1 || dim > (1 << 23) || rows > MAX_ROWS || count < 0 || count > MAX_ROWS) why = "sizes out of range";
  else if (ld < dim) why = "row stride below the width";
  else if (!table || (count && !idx)) why = "null pointer";
  if (!why) return 0;
  snprintf(msg, sizeof msg, "%s: %s", what, why);
  return nphm_fail_msg(msg);
}

}  // namespace train_ops
}  // namespace nphm

using namespace nphm::train_ops;

extern "C" {

int nphm_rows_lookup(const void* table, int64_t rows, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits, int64_t count,
                     float scale, void* out, void* stream) {
  if (int rc = check_table("nphm_rows_lookup", table, rows, dim, ld, dtype, idx, idx_bits, count)) return rc;
  if (count == 0) return 0;
  if (!out) return nphm_fail_msg("nphm_rows_lookup: null pointer");
  const int64_t bytes = count * dim * dtype_size(dtype);
  const bool in = 2 * bytes >= CACHED && count <= rows, to = bytes >= CACHED;
  const LookupArgs a{table, idx, out, ld, count, rows, int(dim), idx_bits == 64, scale};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    for_rows(count, (dim + Vec<T>::N - 1) / Vec<T>::N, [&](auto lanes, dim3 grid) {
      constexpr int L = decltype(lanes)::value;
      hipStream_t st = static_cast<hipStream_t>(stream);
      if (in && to) hipLaunchKernelGGL((lookup_kernel<T, L, true, true>), grid, dim3(256), 0, st, a);
      else if (in) hipLaunchKernelGGL((lookup_kernel<T, L, true, false>), grid, dim3(256), 0, st, a);
      else if (to) hipLaunchKernelGGL((lookup_kernel<T, L, false, true>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((lookup_kernel<T, L, false, false>), grid, dim3(256), 0, st, a);
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_lookup launch", e);
  return 0;
}

size_t nphm_rows_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t count, int dtype) {
  return dtype_ok(dtype) ? grad_plan(rows, dim, count, dtype_size(dtype)).total : 0;
}

int nphm_rows_grad(const void* grad, int64_t count, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits, int64_t rows,
                   int64_t padding, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_table("nphm_rows_grad", out, rows, dim, dim, dtype, idx, idx_bits, count)) return rc;
  if (count && (!grad || ld < dim)) return nphm_fail_msg("nphm_rows_grad: null gradient or row stride below the width");
  const GradPlan g = grad_plan(rows, dim, count, dtype_size(dtype));
  if (workspace_bytes < g.total || (g.total && !workspace)) return nphm_fail_msg("nphm_rows_grad: workspace too small");
  GradArgs a{grad, idx, out, ld, count, rows, int(dim), idx_bits == 64, padding, scale};
  with_dtype(dtype, [&](auto t) {
    if (rows * dim * dtype_size(dtype) > CACHED) grad_run<decltype(t), false, true>(static_cast<hipStream_t>(stream), a, g, static_cast<char*>(workspace));
    else grad_run<decltype(t), false, false>(static_cast<hipStream_t>(stream), a, g, static_cast<char*>(workspace));
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_grad launch", e);
  return 0;
}

int nphm_rows_entries(const void* grad, int64_t count, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits, int64_t rows,
                      int64_t padding, float scale, int64_t* index, void* values, void* stream) {
  if (count == 0) return 0;
  if (int rc = check_table("nphm_rows_entries", grad, rows, dim, ld, dtype, idx, idx_bits, count)) return rc;
  if (!index || !values) return nphm_fail_msg("nphm_rows_entries: null pointer");
  const EntryArgs a{grad, idx, index, values, ld, count, rows, padding, int(dim), idx_bits == 64, scale};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    for_rows(count, (dim + Vec<T>::N - 1) / Vec<T>::N, [&](auto lanes, dim3 grid) {
      hipLaunchKernelGGL((entries_kernel<T, decltype(lanes)::value>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
    });
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_entries launch", e);
  return 0;
}

int nphm_rows_merge(const void* grad, int64_t count, int64_t dim, int dtype, const void* idx, int idx_bits, int64_t rows, void* out,
                    void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_table("nphm_rows_merge", out, rows, dim, dim, dtype, idx, idx_bits, count)) return rc;
  if (count == 0) return 0;
  if (!grad || grad == out) return nphm_fail_msg("nphm_rows_merge: null pointer, or the result in place of the gradient");
  const GradPlan g = grad_plan(rows, dim, count, dtype_size(dtype));
  if (workspace_bytes < g.total || (g.total && !workspace)) return nphm_fail_msg("nphm_rows_merge: workspace too small");
  GradArgs a{grad, idx, out, dim, count, rows, int(dim), idx_bits == 64, -1, 1.f};
  with_dtype(dtype, [&](auto t) { grad_run<decltype(t), true, false>(static_cast<hipStream_t>(stream), a, g, static_cast<char*>(workspace)); });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_merge launch", e);
  return 0;
}

int nphm_rows_renorm(void* table, int64_t rows, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits, int64_t count,
                     float max_norm, void* flags, void* stream) {
  if (int rc = check_table("nphm_rows_renorm", table, rows, dim, ld, dtype, idx, idx_bits, count)) return rc;
  if (!(max_norm >= 0.f)) return nphm_fail_msg("nphm_rows_renorm: max_norm is negative or no number");
  if (count == 0) return 0;
  if (!flags) return nphm_fail_msg("nphm_rows_renorm: null pointer");
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint8_t* f = static_cast<uint8_t*>(flags);
  const int64_t want = (rows + 255) / 256;
  hipLaunchKernelGGL(flags_clear_kernel, dim3(unsigned(want < 2048 ? want : 2048)), dim3(256), 0, st, f, rows);
  hipLaunchKernelGGL(flags_mark_kernel, dim3(unsigned((count + 255) / 256)), dim3(256), 0, st, idx, idx_bits == 64, count, f, rows);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL((renorm_kernel<T>), dim3(unsigned((rows + 3) / 4)), dim3(256), 0, st, static_cast<T*>(table), ld, rows, int(dim), f,
                       max_norm);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_renorm launch", e);
  return 0;
}

}  // extern "C"
