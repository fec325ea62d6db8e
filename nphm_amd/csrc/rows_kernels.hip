// rows_kernels.hip — rows of a table by index (the latent codes of a batch) and the gradient of the table:
//   y[n, :] = scale T[i_n, :]          dT[v, :] = scale sum over {n : i_n = v, v != padding} of g[n, :]
// Both move memory and nothing else.  An index outside [0, rows) reads nothing: its output row is NaN, and it adds nothing to the
// gradient.  The gradient adds the rows of one index in the order of their positions, in fp32, whatever the grid looks like: two
// runs give the same bits (no atomics).
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// A group of LPR lanes takes one row (LPR * 16 bytes of it at a time); a wavefront 64 / LPR rows, so that narrow rows fill it too.
template <class T, int LPR>
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
    if (ok) v = *reinterpret_cast<const vec*>(src + c);
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = ok ? T(float(v[k]) * p.scale) : T(__builtin_nanf(""));
    *reinterpret_cast<vec*>(dst + c) = v;
  }
  if (blockIdx.y == 0) {
    const int c = full + sub;                       // V - 1 elements at most, LPR >= 8 lanes
    if (c < p.dim) dst[c] = ok ? T(float(src[c]) * p.scale) : T(__builtin_nanf(""));
  }
}

struct GradArgs {
  const void* grad;    // [count, dim], rows ld apart
  const void* idx;
  void* out;           // [rows, dim]
  int64_t ld, count, rows;
  int dim, idx64;
  int64_t padding;     // -1: none
  float scale;
};

// One wavefront a row of the table and 64 vectors of its columns: it looks through all indices, 64 at a time, and adds the rows
// that name its own.
template <class T>
__global__ __launch_bounds__(256) void grad_owner_kernel(GradArgs p) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & 63;
  const int64_t v = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (v >= p.rows) return;
  const int c = (blockIdx.y * 64 + lane) * V;
  float acc[V] = {};
  if (v != p.padding) {
    for (int64_t n0 = 0; n0 < p.count; n0 += 64) {
      const int64_t n = n0 + lane;
      uint64_t hit = __ballot(n < p.count && load_index(p.idx, p.idx64, n < p.count ? n : 0) == v);
      while (hit) {
        const int b = __builtin_ctzll(hit);
        hit &= hit - 1;
        const T* g = static_cast<const T*>(p.grad) + (n0 + b) * p.ld;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c + k < p.dim) acc[k] += float(g[c + k]);
      }
    }
  }
  T* dst = static_cast<T*>(p.out) + v * p.dim;
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (c + k < p.dim) dst[c + k] = T(acc[k] * p.scale);
}

// out[n] = the sum of the rows that name the same index as row n, if n is the first of them, else zeros: duplicates of a row gradient
// [count, dim] folded into one entry each, its shape unchanged
template <class T>
__global__ __launch_bounds__(256) void merge_kernel(GradArgs p) {
  constexpr int V = Vec<T>::N;
  const int lane = threadIdx.x & 63;
  const int64_t own = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (own >= p.count) return;
  const int c = (blockIdx.y * 64 + lane) * V;
  const int64_t v = load_index(p.idx, p.idx64, own);
  float acc[V] = {};
  for (int64_t n0 = 0; n0 < p.count; n0 += 64) {
    const int64_t n = n0 + lane;
    uint64_t hit = __ballot(n < p.count && load_index(p.idx, p.idx64, n < p.count ? n : 0) == v);
    if (hit && n0 + __builtin_ctzll(hit) < own) break;             // an earlier row owns the sum (nothing was added yet)
    while (hit) {
      const int b = __builtin_ctzll(hit);
      hit &= hit - 1;
      const T* g = static_cast<const T*>(p.grad) + (n0 + b) * p.ld;
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (c + k < p.dim) acc[k] += float(g[c + k]);
    }
  }
  T* dst = static_cast<T*>(p.out) + own * p.dim;
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (c + k < p.dim) dst[c + k] = T(acc[k]);
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
  LookupArgs a{table, idx, out, ld, count, rows, int(dim), idx_bits == 64, scale};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const int64_t vecs = (dim + Vec<T>::N - 1) / Vec<T>::N;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (vecs <= 8) hipLaunchKernelGGL((lookup_kernel<T, 8>), dim3((count + 31) / 32), dim3(256), 0, st, a);
    else if (vecs <= 16) hipLaunchKernelGGL((lookup_kernel<T, 16>), dim3((count + 15) / 16), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((lookup_kernel<T, 64>), dim3((count + 3) / 4), dim3(256), 0, st, a);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_lookup launch", e);
  return 0;
}

size_t nphm_rows_grad_workspace_bytes(int64_t rows, int64_t dim, int64_t count) { return 0; }

int nphm_rows_grad(const void* grad, int64_t count, int64_t dim, int64_t ld, int dtype, const void* idx, int idx_bits, int64_t rows,
                   int64_t padding, float scale, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_table("nphm_rows_grad", out, rows, dim, dim, dtype, idx, idx_bits, count)) return rc;
  if (count && (!grad || ld < dim)) return nphm_fail_msg("nphm_rows_grad: null gradient or row stride below the width");
  if (workspace_bytes < nphm_rows_grad_workspace_bytes(rows, dim, count)) return nphm_fail_msg("nphm_rows_grad: workspace too small");
  GradArgs a{grad, idx, out, ld, count, rows, int(dim), idx_bits == 64, padding, scale};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned tiles = unsigned((dim + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N));
    hipLaunchKernelGGL((grad_owner_kernel<T>), dim3(unsigned((rows + 3) / 4), tiles), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_rows_grad launch", e);
  return 0;
}

int nphm_rows_merge(const void* grad, int64_t count, int64_t dim, int dtype, const void* idx, int idx_bits, void* out, void* stream) {
  if (int rc = check_table("nphm_rows_merge", out, 1, dim, dim, dtype, idx, idx_bits, count)) return rc;
  if (count == 0) return 0;
  if (!grad) return nphm_fail_msg("nphm_rows_merge: null pointer");
  GradArgs a{grad, idx, out, dim, count, 0, int(dim), idx_bits == 64, -1, 1.f};
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned tiles = unsigned((dim + 64 * Vec<T>::N - 1) / (64 * Vec<T>::N));
    hipLaunchKernelGGL((merge_kernel<T>), dim3(unsigned((count + 3) / 4), tiles), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  });
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
