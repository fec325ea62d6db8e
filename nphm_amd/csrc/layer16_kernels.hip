// layer16_kernels.hip — one dense layer in 16-bit storage (bf16 or fp16), fp32 accumulation:
//   z = x W^T + b,   y = a(z) + r            and its gradients   gz = g a'(z),  dx = gz W,  dW = gz^T x,  db = sum_m gz
// One kernel computes all three products, C[i, j] = sum_k A(i, k) B(j, k), from strided operands.
// Roundings to 16 bits: the outputs, z as it is kept for the backward pass (a' moves by at most z 2^-9 a''(z), which is below the
// rounding of the gradients themselves for every activation here), and gz before the two products that read it (the matrix
// instructions take 16-bit operands).  Sums over k, over m and over splits are in fp32, in a fixed order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "capi_common.h"
#include "train_ops_common.h"

namespace nphm {
namespace train_ops {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16 fp16x8 __attribute__((ext_vector_type(8)));
template <class T> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<fp16> { typedef fp16x8 type; };
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(fp16x8 a, fp16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_SOFTPLUS = 4 };

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

__device__ __forceinline__ float act_value(float z, int act, float beta) {
  switch (act) {
    case ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case ACT_SILU: return z * sigmoid(z);
    case ACT_GELU: return 0.5f * z * (1.f + erff(z * 0.70710678f));
    case ACT_SOFTPLUS: {
      const float t = beta * z;
      return t > 20.f ? z : log1pf(__expf(t)) / beta;
    }
    default: return z;
  }
}
__device__ __forceinline__ float act_slope(float z, int act, float beta) {
  switch (act) {
    case ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case ACT_SILU: { const float s = sigmoid(z); return s + z * s * (1.f - s); }
    case ACT_GELU: return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * __expf(-0.5f * z * z);
    case ACT_SOFTPLUS: return sigmoid(beta * z);
    default: return 1.f;
  }
}

struct GemmArgs {
  const void* A; int64_t a_i, a_k;       // element strides
  const void* B; int64_t b_j, b_k;
  int I, J, K;
  int splits, k_per_split;               // > 1: partial products to `parts`
  float* parts;                          // [splits][I][J]
  void* C;                               // [I, J]
  // forward epilogue
  const void* bias;                      // [J] or null
  const void* residual;                  // [I, J] or null
  void* z;                               // [I, J] or null: the value before the activation
  int act;
  float beta;
};

// z as it is kept: finite where z is (a' of an infinity is no number for some activations)
template <class T>
__device__ __forceinline__ T keep(float v) {
  constexpr float MOST = std::is_same<T, fp16>::value ? 65504.f : 3.38953139e38f;
  return T(v != v ? v : fminf(fmaxf(v, -MOST), MOST));
}

constexpr int GT = 64, GK = 32, GP = GK + 8;

template <class T>
__global__ __launch_bounds__(256) void gemm_simple_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(16))) T sa[GT * GP], sb[GT * GP];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int i0 = blockIdx.y * GT, j0 = blockIdx.x * GT;
  const int kb = blockIdx.z * p.k_per_split, ke = min(p.K, kb + p.k_per_split);
  const T* A = static_cast<const T*>(p.A);
  const T* B = static_cast<const T*>(p.B);
  f32x16 acc = {};
  for (int k0 = kb; k0 < ke; k0 += GK) {
    for (int u = t; u < GT * GK; u += 256) {
      const int r = u / GK, k = u % GK;
      sa[r * GP + k] = (i0 + r < p.I && k0 + k < ke) ? A[int64_t(i0 + r) * p.a_i + int64_t(k0 + k) * p.a_k] : T(0.f);
      sb[r * GP + k] = (j0 + r < p.J && k0 + k < ke) ? B[int64_t(j0 + r) * p.b_j + int64_t(k0 + k) * p.b_k] : T(0.f);
    }
    __syncthreads();
    typedef typename Frag<T>::type frag;
#pragma unroll
    for (int s = 0; s < GK; s += 16) {
      const frag a = *reinterpret_cast<const frag*>(sa + ((wave >> 1) * 32 + (lane & 31)) * GP + s + 8 * (lane >> 5));
      const frag b = *reinterpret_cast<const frag*>(sb + ((wave & 1) * 32 + (lane & 31)) * GP + s + 8 * (lane >> 5));
      acc = mfma(a, b, acc);
    }
    __syncthreads();
  }
  const int j = j0 + (wave & 1) * 32 + (lane & 31);
  if (j >= p.J) return;
  const float bias = p.bias ? float(static_cast<const T*>(p.bias)[j]) : 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int i = i0 + (wave >> 1) * 32 + 8 * (q >> 2) + 4 * (lane >> 5) + (q & 3);
    if (i >= p.I) continue;
    const int64_t at = int64_t(i) * p.J + j;
    if (p.splits > 1) { p.parts[int64_t(blockIdx.z) * p.I * p.J + at] = acc[q]; continue; }
    float v = acc[q] + bias;
    if (p.z) static_cast<T*>(p.z)[at] = keep<T>(v);
    v = act_value(v, p.act, p.beta);
    if (p.residual) v += float(static_cast<const T*>(p.residual)[at]);
    static_cast<T*>(p.C)[at] = T(v);
  }
}

template <class T>
__global__ __launch_bounds__(256) void join_splits_kernel(const float* parts, int splits, int64_t count, T* out) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t(gridDim.x) * 256) {
    float s = 0.f;
    for (int z = 0; z < splits; ++z) s += parts[int64_t(z) * count + i];
    out[i] = T(s);
  }
}

// gz = g a'(z) and the column sums of every 64-row tile of it (before it is rounded)
template <class T>
__global__ __launch_bounds__(256) void gz_kernel(const T* g, const T* z, T* gz, float* sums, int M, int N, int act, float beta) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  const int m0 = blockIdx.y * 64, m1 = min(M, m0 + 64);
  float s = 0.f;
  for (int m = m0; m < m1; ++m) {
    const int64_t at = int64_t(m) * N + n;
    float v = float(g[at]);
    if (z) { v *= act_slope(float(z[at]), act, beta); gz[at] = T(v); }
    s += v;
  }
  if (sums) sums[int64_t(blockIdx.y) * N + n] = s;
}

template <class T>
__global__ __launch_bounds__(256) void column_sums16_kernel(const float* sums, int tiles, int N, T* out) {
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float s = 0.f;
  for (int t = 0; t < tiles; ++t) s += sums[int64_t(t) * N + n];
  out[n] = T(s);
}

struct Plan {
  size_t gz = 0, sums = 0, parts = 0, total = 0;    // byte offsets
  int w_splits = 1;
};
inline size_t up(size_t v) { return (v + 255) / 256 * 256; }
inline Plan backward_plan(int64_t M, int64_t N, int64_t K, int act) {
  Plan p;
  const int64_t tiles = ((N + GT - 1) / GT) * ((K + GT - 1) / GT);
  int64_t s = tiles >= 512 ? 1 : 512 / tiles;
  if (s > (M + 255) / 256) s = (M + 255) / 256;
  p.w_splits = int(s < 1 ? 1 : s);
  p.gz = 0;
  p.sums = p.gz + (act != ACT_NONE ? up(size_t(M) * N * 2) : 0);
  p.parts = p.sums + up(size_t((M + 63) / 64) * N * 4);
  p.total = p.parts + (p.w_splits > 1 ? up(size_t(p.w_splits) * N * K * 4) : 0);
  return p;
}

template <class T>
inline void gemm(hipStream_t st, GemmArgs a) {
  a.k_per_split = ((a.K + a.splits - 1) / a.splits + GK - 1) / GK * GK;
  hipLaunchKernelGGL((gemm_simple_kernel<T>), dim3((a.J + GT - 1) / GT, (a.I + GT - 1) / GT, a.splits), dim3(256), 0, st, a);
  if (a.splits > 1) {
    const int64_t count = int64_t(a.I) * a.J, want = (count + 255) / 256;
    hipLaunchKernelGGL((join_splits_kernel<T>), dim3(unsigned(want < 4096 ? want : 4096)), dim3(256), 0, st, a.parts, a.splits, count,
                       static_cast<T*>(a.C));
  }
}

inline int check_layer(const char* what, int64_t M, int64_t N, int64_t K, int dtype, int act, float beta) {
  static thread_local char msg[160];
  const char* why = nullptr;
  if (dtype != DT_BF16 && dtype != DT_F16) why = "dtype is 1 (bf16) or 2 (fp16)";
  else if (M < 1 || N < 1 || K < 1 || M > (1 << 22) || N > (1 << 20) || K > (1 << 20)) why = "sizes out of range (M up to 2^22, N and K up to 2^20)";
  else if (act < ACT_NONE || act > ACT_SOFTPLUS) why = "unknown activation";
  else if (act == ACT_SOFTPLUS && !(beta > 0.f && beta < 1e30f)) why = "Softplus takes a positive beta";
  if (!why) return 0;
  snprintf(msg, sizeof msg, "%s: %s", what, why);
  return nphm_fail_msg(msg);
}

}  // namespace train_ops
}  // namespace nphm

using namespace nphm::train_ops;

extern "C" {

size_t nphm_layer16_forward_workspace_bytes(int64_t M, int64_t N, int64_t K) { return 0; }

int nphm_layer16_forward(const void* x, const void* weight, const void* bias, const void* residual, void* y, void* z, int64_t M, int64_t N,
                         int64_t K, int dtype, int act, float beta, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_layer("nphm_layer16_forward", M, N, K, dtype, act, beta)) return rc;
  if (!x || !weight || !y) return nphm_fail_msg("nphm_layer16_forward: null pointer");
  GemmArgs a{};
  a.A = x; a.a_i = K; a.a_k = 1;
  a.B = weight; a.b_j = K; a.b_k = 1;
  a.I = int(M); a.J = int(N); a.K = int(K);
  a.splits = 1;
  a.C = y; a.bias = bias; a.residual = residual; a.z = z; a.act = act; a.beta = beta;
  with_dtype(dtype, [&](auto t) {
    if constexpr (sizeof(t) == 2) gemm<decltype(t)>(static_cast<hipStream_t>(stream), a);
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_layer16_forward launch", e);
  return 0;
}

size_t nphm_layer16_backward_workspace_bytes(int64_t M, int64_t N, int64_t K, int act) { return backward_plan(M, N, K, act).total; }

int nphm_layer16_backward(const void* g, const void* x, const void* weight, const void* z, void* dx, void* dweight, void* dbias, int64_t M,
                          int64_t N, int64_t K, int dtype, int act, float beta, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_layer("nphm_layer16_backward", M, N, K, dtype, act, beta)) return rc;
  if (!g || (act != ACT_NONE && !z) || (dx && !weight) || (dweight && !x) || !workspace) return nphm_fail_msg("nphm_layer16_backward: null pointer");
  const Plan plan = backward_plan(M, N, K, act);
  if (workspace_bytes < plan.total) return nphm_fail_msg("nphm_layer16_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  with_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if constexpr (sizeof(T) == 2) {
      T* gz = act == ACT_NONE ? const_cast<T*>(static_cast<const T*>(g)) : reinterpret_cast<T*>(ws + plan.gz);
      float* sums = reinterpret_cast<float*>(ws + plan.sums);
      const unsigned tiles = unsigned((M + 63) / 64);
      if (act != ACT_NONE || dbias)
        hipLaunchKernelGGL((gz_kernel<T>), dim3(unsigned((N + 255) / 256), tiles), dim3(256), 0, st, static_cast<const T*>(g),
                           act == ACT_NONE ? nullptr : static_cast<const T*>(z), gz, dbias ? sums : nullptr, int(M), int(N), act, beta);
      if (dbias)
        hipLaunchKernelGGL((column_sums16_kernel<T>), dim3(unsigned((N + 255) / 256)), dim3(256), 0, st, sums, int(tiles), int(N),
                           static_cast<T*>(dbias));
      if (dx) {
        GemmArgs a{};
        a.A = gz; a.a_i = N; a.a_k = 1;
        a.B = weight; a.b_j = 1; a.b_k = K;
        a.I = int(M); a.J = int(K); a.K = int(N);
        a.splits = 1; a.C = dx;
        gemm<T>(st, a);
      }
      if (dweight) {
        GemmArgs a{};
        a.A = gz; a.a_i = 1; a.a_k = N;
        a.B = x; a.b_j = 1; a.b_k = K;
        a.I = int(N); a.J = int(K); a.K = int(M);
        a.splits = plan.w_splits; a.parts = reinterpret_cast<float*>(ws + plan.parts); a.C = dweight;
        gemm<T>(st, a);
      }
    }
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_layer16_backward launch", e);
  return 0;
}

}  // extern "C"
