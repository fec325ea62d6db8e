// clip_kernels.hip — the norm over many tensors, and their clipping by it:
//   n = sqrt(sum_t sum_i g_ti^2)  or  max |g_ti|,     c = min(1, limit / (n + 1e-6)),     out_t = c g_t
// Squares are added in fp64: no gradient of fp32, bf16 or fp16 overflows or vanishes in them, and the sum does not depend on how many
// there are.  Every block writes its own partial sum and they are added in block order: two runs give the same bits.
// Bound by memory: the gradients are read twice and written once.  290 bf16 tensors of 1 M elements (1.82 GB moved): 336 us, 5.4 TB/s; the
// tensors of a decoder (24 MB): 12.5 us, of which 5.0 for the norm and 6.3 for the scaling.  500 small tensors, 3 MB in all: 50 us for eight launches, 41 of
// them on the card: 4.95 each for the norm and 5.43 for the scaling, where an empty launch takes 2.6 (a chunk finds its tensor by
// eight reads of the arguments, each waiting for the one before).
// The tensors travel by value in the kernel's arguments, TABLE of them a launch (nothing is copied to the device, nothing has to
// outlive the call: a captured graph holds its own copy).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <vector>

#include "capi_common.h"
#include "train_ops_common.h"

namespace nphm {
namespace train_ops {

constexpr int TABLE = 150;               // tensors a launch: 150 x 25 bytes of the 4 KiB of arguments
constexpr int CHUNK = 16384;             // bytes a block takes at a time
constexpr int MAX_BLOCKS = 2048;

struct ClipTable {
  const void* in[TABLE];
  void* out[TABLE];
  uint32_t elements[TABLE];
  uint32_t first_chunk[TABLE + 1];
  uint8_t dtype[TABLE];
  int tensors;
};

// tensor of a chunk: the last one whose first chunk is not behind it
__device__ __forceinline__ int tensor_of(const ClipTable& t, uint32_t chunk) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first_chunk[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <class T>
__device__ __forceinline__ void take(double& acc, T x, int kind) {
  const double a = double(float(x));
  if (kind == 0) acc = fma(a, a, acc);
  else { const double b = fabs(a); acc = (b > acc || b != b) ? b : acc; }      // NaN stays
}
__device__ __forceinline__ double join(double a, double b, int kind) {
  if (kind == 0) return a + b;
  return (b > a || b != b) ? b : a;
}

// the block's values -> one, the same on every thread, in a fixed order
template <int THREADS>
__device__ __forceinline__ double block_join(double v, int kind) {
  __shared__ double part[THREADS / 64];
#pragma unroll
  for (int o = 32; o; o >>= 1) v = join(v, __shfl_xor(v, o), kind);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  v = part[0];
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w) v = join(v, part[w], kind);
  return v;
}

template <class T>
__device__ __forceinline__ void norm_chunk(const ClipTable& t, int i, uint32_t chunk, int kind, double& acc) {
  constexpr int V = Vec<T>::N, PER = CHUNK / sizeof(T);
  const T* g = static_cast<const T*>(t.in[i]);
  const uint32_t n = t.elements[i], begin = (chunk - t.first_chunk[i]) * PER, end = min(n, begin + PER);
  const uint32_t full = begin + (end - begin) / V * V;
  for (uint32_t c = begin + threadIdx.x * V; c < full; c += 256 * V) {
    const typename Vec<T>::type v = *reinterpret_cast<const typename Vec<T>::type*>(g + c);
#pragma unroll
    for (int k = 0; k < V; ++k) take(acc, v[k], kind);
  }
  if (full + threadIdx.x < end) take(acc, g[full + threadIdx.x], kind);
}

__global__ __launch_bounds__(256) void norm_kernel(ClipTable t, uint32_t chunks, int kind, double* partial) {
  double acc = 0;
  for (uint32_t c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int i = tensor_of(t, c);
    if (t.dtype[i] == DT_F32) norm_chunk<float>(t, i, c, kind, acc);
    else if (t.dtype[i] == DT_BF16) norm_chunk<bf16>(t, i, c, kind, acc);
    else norm_chunk<fp16>(t, i, c, kind, acc);
  }
  acc = block_join<256>(acc, kind);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// partial sums -> norm (fp32) and the factor
template <int THREADS>
__device__ __forceinline__ void finish(const double* partial, int n, int kind, double limit, float& norm, float& factor) {
  double acc = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) acc = join(acc, partial[i], kind);
  acc = block_join<THREADS>(acc, kind);
  if (kind == 0) acc = sqrt(acc);
  const double f = limit / (acc + 1e-6);
  norm = float(acc);
  factor = f > 1.0 ? 1.f : float(f);
}

__global__ __launch_bounds__(1024) void finish_kernel(const double* partial, int n, int kind, double limit, float* norm, float* factor) {
  float a, f;
  finish<1024>(partial, n, kind, limit, a, f);
  if (threadIdx.x == 0) {
    *norm = a;
    if (factor) *factor = f;
  }
}

template <class T, bool STREAM>
__device__ __forceinline__ void scale_chunk(const ClipTable& t, int i, uint32_t chunk, float f) {
  constexpr int V = Vec<T>::N, PER = CHUNK / sizeof(T);
  const T* g = static_cast<const T*>(t.in[i]);
  T* o = static_cast<T*>(t.out[i]);
  const uint32_t n = t.elements[i], begin = (chunk - t.first_chunk[i]) * PER, end = min(n, begin + PER);
  const uint32_t full = begin + (end - begin) / V * V;
  for (uint32_t c = begin + threadIdx.x * V; c < full; c += 256 * V) {
    typename Vec<T>::type v = load_vec<STREAM>(g + c);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = T(float(v[k]) * f);
    store_vec<true>(o + c, v);
  }
  if (full + threadIdx.x < end) o[full + threadIdx.x] = T(float(g[full + threadIdx.x]) * f);
}

// Up to FOLD partial sums every block adds up by itself (8 KiB from L2, no launch for them); more have their factor ready.
constexpr int FOLD = 1024;

struct Factor {
  const double* partial;
  int n, kind;
  double limit;
  float* norm;               // written by the first block where the partial sums are folded here
  const float* ready;        // null: fold
  bool stream;
};

// What is scaled is not read again: where all do not fit into the last cache its lines are not kept, to the good of what the norm has left there (290
// bf16 tensors, 606 MB: 361 us, 336 so; 8 MB: 12.4, 14.7 so).  What is written never is (378, 361 so).

template <bool STREAM>
__device__ __forceinline__ void scale_any(const ClipTable& t, int i, uint32_t c, float f) {
  if (t.dtype[i] == DT_F32) scale_chunk<float, STREAM>(t, i, c, f);
  else if (t.dtype[i] == DT_BF16) scale_chunk<bf16, STREAM>(t, i, c, f);
  else scale_chunk<fp16, STREAM>(t, i, c, f);
}

__global__ __launch_bounds__(256) void scale_kernel(ClipTable t, uint32_t chunks, Factor s) {
  float f;
  if (s.ready) {
    f = *s.ready;
  } else {
    float norm;
    finish<256>(s.partial, s.n, s.kind, s.limit, norm, f);
    if (blockIdx.x == 0 && threadIdx.x == 0 && s.norm) *s.norm = norm;
  }
  for (uint32_t b = blockIdx.x; b < chunks; b += gridDim.x) {
    const uint32_t c = chunks - 1 - b;                               // the other way round: what was read last is still in the cache
    const int i = tensor_of(t, c);
    if (f == 1.f && t.in[i] == t.out[i]) continue;                 // nothing to change in place
    if (s.stream) scale_any<true>(t, i, c, f);
    else scale_any<false>(t, i, c, f);
  }
}

// cuts the list into tables, from its end where `back`: f(table, chunks)
template <class F>
inline void for_tables(const void* const* in, void* const* out, const int64_t* counts, const int* dtypes, int n, bool back, F&& f) {
  ClipTable t;
  t.tensors = 0;
  uint32_t chunks = 0;
  auto flush = [&] {
    if (!t.tensors) return;
    t.first_chunk[t.tensors] = chunks;
    f(t, chunks);
    t.tensors = 0;
    chunks = 0;
  };
  constexpr int64_t PIECE = int64_t(1) << 30;                      // a tensor of more elements takes several entries
  for (int u = 0; u < n; ++u) {
    const int i = back ? n - 1 - u : u, e = dtype_size(dtypes[i]);
    for (int64_t at = 0; at < counts[i]; at += PIECE) {
      const int64_t m = std::min(PIECE, counts[i] - at);
      const int k = t.tensors++;
      t.in[k] = static_cast<const char*>(in[i]) + at * e;
      t.out[k] = out ? static_cast<char*>(out[i]) + at * e : nullptr;
      t.elements[k] = uint32_t(m);
      t.dtype[k] = uint8_t(dtypes[i]);
      t.first_chunk[k] = chunks;
      chunks += uint32_t((m * e + CHUNK - 1) / CHUNK);
      if (t.tensors == TABLE) flush();
    }
  }
  flush();
}

inline int table_count(const int64_t* counts, int n) {
  int64_t entries = 0;
  for (int i = 0; i < n; ++i) entries += (counts[i] + (int64_t(1) << 30) - 1) >> 30;
  return int((entries + TABLE - 1) / TABLE);
}

struct Range { uintptr_t begin, end; };
inline bool before(const Range& x, const Range& y) { return x.begin < y.begin; }
// whether two written ranges meet, or a read one meets a written one (a tensor clipped in place is among the written ones only)
inline bool meet(std::vector<Range>& written, std::vector<Range>& read) {
  if (!std::is_sorted(written.begin(), written.end(), before)) std::sort(written.begin(), written.end(), before);
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].begin < written[i - 1].end) return true;
  for (const Range& r : read) {
    auto at = std::lower_bound(written.begin(), written.end(), r, before);
    if (at != written.end() && at->begin < r.end) return true;
    if (at != written.begin() && (at - 1)->end > r.begin) return true;
  }
  return false;
}

}  // namespace train_ops
}  // namespace nphm

using namespace nphm::train_ops;

extern "C" {

size_t nphm_clip_workspace_bytes(const int64_t* counts, int n) {
  if (!counts || n < 1) return 0;
  return (size_t(table_count(counts, n)) * MAX_BLOCKS + 1) * sizeof(double);
}

int nphm_clip_grads(const void* const* in, void* const* out, const int64_t* counts, const int* dtypes, int n, int kind, double limit,
                    float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  if (n < 1 || !in || !counts || !dtypes || !norm || !workspace) return nphm_fail_msg("nphm_clip_grads: null pointer or no tensors");
  if (kind != 0 && kind != 1) return nphm_fail_msg("nphm_clip_grads: kind is 0 (2-norm) or 1 (largest magnitude)");
  if (out && !(limit >= 0)) return nphm_fail_msg("nphm_clip_grads: the limit is negative or no number");
  try {
    std::vector<Range> written, read;
    if (out) written.reserve(n), read.reserve(n);
    for (int i = 0; i < n; ++i) {
      if (!dtype_ok(dtypes[i])) return nphm_fail_msg("nphm_clip_grads: dtype is 0 (fp32), 1 (bf16) or 2 (fp16)");
      if (counts[i] < 0 || counts[i] > (int64_t(1) << 36)) return nphm_fail_msg("nphm_clip_grads: element count out of range");
      if (counts[i] && (!in[i] || (out && !out[i]))) return nphm_fail_msg("nphm_clip_grads: null pointer");
      if (out && counts[i]) {
        const uintptr_t bytes = uintptr_t(counts[i]) * dtype_size(dtypes[i]), o = reinterpret_cast<uintptr_t>(out[i]), p = reinterpret_cast<uintptr_t>(in[i]);
        written.push_back({o, o + bytes});
        if (p != o) read.push_back({p, p + bytes});
      }
    }
    if (meet(written, read)) return nphm_fail_msg("nphm_clip_grads: two of the tensors share memory");
    if (workspace_bytes < nphm_clip_workspace_bytes(counts, n)) return nphm_fail_msg("nphm_clip_grads: workspace too small");
  } catch (...) {
    return nphm_fail_msg("nphm_clip_grads: out of host memory");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  float* factor = reinterpret_cast<float*>(partial + size_t(table_count(counts, n)) * MAX_BLOCKS);
  int parts = 0;
  for_tables(in, out, counts, dtypes, n, false, [&](const ClipTable& t, uint32_t chunks) {
    const uint32_t blocks = std::min<uint32_t>(chunks, MAX_BLOCKS);
    hipLaunchKernelGGL(norm_kernel, dim3(blocks), dim3(256), 0, st, t, chunks, kind, partial + parts);
    parts += int(blocks);
  });
  const bool fold = out && parts && parts <= FOLD;
  if (!fold) hipLaunchKernelGGL(finish_kernel, dim3(1), dim3(1024), 0, st, partial, parts, kind, limit, norm, out ? factor : nullptr);
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += counts[i] * dtype_size(dtypes[i]);
  Factor s{partial, parts, kind, limit, norm, fold ? nullptr : factor, bytes > CACHED};
  if (out)
    for_tables(in, out, counts, dtypes, n, true, [&](const ClipTable& t, uint32_t chunks) {
      hipLaunchKernelGGL(scale_kernel, dim3(std::min<uint32_t>(chunks, MAX_BLOCKS)), dim3(256), 0, st, t, chunks, s);
      s.norm = nullptr;
    });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_clip_grads launch", e);
  return 0;
}

}  // extern "C"
