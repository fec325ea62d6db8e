// layer16_kernels.hip — one dense layer in 16-bit storage (bf16 or fp16), fp32 accumulation:
//   z = x W^T + b,   y = a(z) + r            and its gradients   gz = g a'(z),  dx = gz W,  dW = gz^T x,  db = sum_m gz
// All three products are C[i, j] = sum_k A(i, k) B(j, k) with either operand as it lies in memory, k beside k or row beside row (nothing is
// transposed on the way).  Bound by the matrix cores: M = 8192, N = K = 4096 in bf16 take 190 us a product on random numbers, 1.45
// PFLOP/s (library: 174 us); the matrix pipe is busy in 68 to 70 % of the cycles (78 %), the rest is the step's barrier and the loads in
// front of it.  M = 16384, N = K = 1024 with Softplus: forward 41 us, dx 33, dW 43 and 5 to join its quarters, gz and db 23; one tile a
// CU, so that what a tile stores (67 MB, 13 us at the copy's rate) hides behind nothing.  Rows that do not start on 16 bytes are copied to
// such first (4095 x 515 and 1024 x 515: 7 us).
// Roundings to 16 bits, each half a step h of the type (bf16 2^-8, fp16 2^-11) of the value that is rounded: the outputs; z as it is kept for the
// backward pass; gz before the two products that read it (the matrix instructions take 16-bit operands).  z's moves a'(z) by at most
// max |z a''(z)| h = 0.34 h (Softplus 0.23, SiLU 0.31, GELU 0.34), so gz by 0.34 h |g|: that is a part of |g|, not of gz.  Where a' is small
// it is much of it (Softplus at beta z = -10: ten half steps, 4 % in bf16), where a' crosses zero all of it; ReLU's is exact unless z is
// below fp16's smallest number.  Error of dx and dW against 64 bits, as a part of their 2-norm, M = 2048, N = K = 512 in bf16: 1.66e-3 if gz stays
// in fp32 (the results' own rounding), 1.70e-3 here with Softplus (beta 100), 2.4e-3 with SiLU and GELU; db 1.69e-3 and 1.78e-3 (SiLU).
// Sums over k, over m and over splits are in fp32, in a fixed order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>

#include "capi_common.h"
#include "train_ops_common.h"

namespace nphm {
namespace train_ops {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef fp16 fp16x8 __attribute__((ext_vector_type(8)));
template <class T> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<fp16> { typedef fp16x8 type; };
// 16 x 16 x 32: on random numbers the chip's power lets it sustain 1990 TFLOP/s of these from registers, 1780 of the 32 x 32 x 16 ones, whose
// accumulators move twice as often
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(fp16x8 a, fp16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_SOFTPLUS = 4 };

// exp and log in base 2 and the reciprocal are the hardware's (1 ulp): far below a 16-bit rounding
__device__ __forceinline__ float exp_(float v) { return __builtin_amdgcn_exp2f(1.44269504f * v); }
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_(-z)); }
// normal distribution, P(X < z): erfc by Abramowitz & Stegun 7.1.26 (off by 1.5e-7 at most), e = exp(-z^2 / 2).  e is a factor of the small
// side, so that its relative error stays small where 1 + erf has no bits left: 5e-4 at z = -4, 2e-3 at -5, 4e-3 at -6, 2e-2 at -10.
__device__ __forceinline__ float normal_cdf(float z, float e) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678f * fabsf(z));
  const float half = 0.5f * e * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z > 0.f ? 1.f - half : half;
}

__device__ __forceinline__ float act_value(float z, int act, float beta) {
  switch (act) {
    case ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case ACT_SILU: return z * sigmoid(z);
    case ACT_GELU: return z * normal_cdf(z, exp_(-0.5f * z * z));
    case ACT_SOFTPLUS: {                                             // max(z, 0) + log(1 + exp(-|beta z|)) / beta
      const float t = exp_(-fabsf(beta * z));
      const float l = t < 1e-3f ? t - 0.5f * t * t : 0.693147181f * __builtin_amdgcn_logf(1.f + t);
      return fmaxf(z, 0.f) + l * __builtin_amdgcn_rcpf(beta);
    }
    default: return z;
  }
}
__device__ __forceinline__ float act_slope(float z, int act, float beta) {
  switch (act) {
    case ACT_RELU: return z > 0.f ? 1.f : (z != z ? z : 0.f);
    case ACT_SILU: { const float s = sigmoid(z); return s + z * s * (1.f - s); }
    case ACT_GELU: { const float e = exp_(-0.5f * z * z); return normal_cdf(z, e) + z * 0.39894228f * e; }
    case ACT_SOFTPLUS: return sigmoid(beta * z);
    default: return 1.f;
  }
}

struct GemmArgs {
  const void* A; int64_t lda;            // [I, K] rows lda elements apart, or (transposed) [K, I]
  const void* B; int64_t ldb;            // [J, K], or (transposed) [K, J]
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
  bool stream_z, stream_c;               // not kept in the caches
};

// z is read again in the backward pass, after all that follows in this one: from 32 MiB on it is not kept, and neither are it and g when they
// are read for gz (six layers of 16384 x 1024 x 1024 with SiLU, forward and backward: 860 us if they are, 823 so; eight of 4096 x 512 x 512:
// 242 and 250).  y is for the next layer: it is kept unless it fills the last cache by itself (16384 x 16384: 1644 us if it is, 1625
// so; the six layers' forward pass 211 us, 215 if y never is).
constexpr int64_t Z_KEPT = CACHED / 8;

// z as it is kept: finite where z is (a' of an infinity is no number for some activations)
template <class T>
__device__ __forceinline__ T keep(float v) {
  constexpr float MOST = std::is_same<T, fp16>::value ? 65504.f : 3.38953139e38f;
  return T(v != v ? v : fminf(fmaxf(v, -MOST), MOST));
}

constexpr int BK = 64;                   // k a step: 128 bytes of a row
constexpr int SLOTS = 5;                 // tiles of one operand in LDS or on their way: two steps and a half

// One operand's tile of ROWS rows (its i or j) x 64 k, on its way from memory to LDS and from there into fragments.
// Not transposed: memory holds k beside k.  LDS row r: 128 bytes, its eight 16-byte pieces c at place c ^ (r / 2 % 8), so that the lanes of a
//   fragment read (16 rows, the same k) meet every bank.  A fragment's 8 k are one ds_read_b128.
// Transposed: memory holds row beside row.  LDS row k: 2 ROWS bytes, piece c at c ^ 2 turn(k).  A fragment's 8 k are two ds_read_b64_tr: 16 lanes
//   read 4 k x 16 rows and get them turned round; 32 lanes read k, k + 1, k + 2, k + 3 and the four 8 on, in different banks by turn.
// Both are written by LDS-DMA (the destination is linear in the lane: the lanes load permuted pieces instead), 1 KiB an instruction.
// Pieces behind the operand's end have an offset behind the buffer's: they arrive as zeros.
template <int ROWS>
__device__ __forceinline__ int turn(int k) { return ROWS >= 128 ? (k & 3) | ((k >> 3) & 1) << 2 : ((k >> 1) & 1) | ((k >> 3) & 1) << 1; }

template <class T, int ROWS, int WAVES, bool TR>
struct Operand {
  static constexpr int BYTES = ROWS * BK * 2, DMA = BYTES / 1024 / WAVES, CPR = TR ? ROWS / 8 : BK / 8;
  static_assert(BYTES % (1024 * WAVES) == 0, "whole DMA instructions a wavefront");
  static constexpr unsigned NOWHERE = 0x80000000u;                   // behind every buffer (each is below 2^31 bytes)
  const char* base;
  int64_t ld;
  int rows, K;                                                       // valid rows from the tile's first
  unsigned voff[DMA];
  unsigned lds0;                                                     // this wavefront's first KiB of a slot
  v4i rsrc;
  unsigned soff;

  // the piece of a row (not transposed) or the piece and row (transposed) that lane `lane` takes in instruction d
  __device__ __forceinline__ static int row_of(int d, int wave, int lane) { return ((d * WAVES + wave) * 64 + lane) / CPR; }
  __device__ __forceinline__ static int piece_of(int d, int wave, int lane) {
    const int row = row_of(d, wave, lane), at = lane % CPR;
    return TR ? at ^ (turn<ROWS>(row) << 1) : at ^ ((row >> 1) & 7);
  }
  __device__ __forceinline__ void init(const void* P, int64_t ld_, int r0, int I, int K_, int wave, int lane, unsigned lds_first) {
    ld = ld_;
    K = K_;
    rows = min(ROWS, I - r0);
    base = static_cast<const char*>(P) + (TR ? int64_t(r0) * 2 : int64_t(r0) * ld * 2);
    lds0 = __builtin_amdgcn_readfirstlane(lds_first + wave * 1024);
#pragma unroll
    for (int d = 0; d < DMA; ++d) {
      const int c = piece_of(d, wave, lane);
      voff[d] = TR && c * 8 >= rows ? NOWHERE : unsigned(row_of(d, wave, lane) * int(ld) * 2 + c * 16);
    }
  }
  // The 64 k from k0 (behind K: zeros, nothing is read), in ascending order of k0: aim() once, then issue(d) for every instruction d, into the
  // slot `shift` bytes behind the first.
  __device__ __forceinline__ void aim(int k0, int lane, int wave) {
    const char* p = TR ? base + int64_t(k0) * ld * 2 : base;
    const unsigned bytes = k0 >= K ? 0u : (TR ? unsigned(min(BK, K - k0)) : unsigned(rows)) * unsigned(ld * 2);
    rsrc[0] = __builtin_amdgcn_readfirstlane(int(uint32_t(uintptr_t(p))));
    rsrc[1] = __builtin_amdgcn_readfirstlane(int(uint32_t(uintptr_t(p) >> 32) & 0xffff));
    rsrc[2] = __builtin_amdgcn_readfirstlane(int(bytes));
    rsrc[3] = 0x00020000;
    soff = __builtin_amdgcn_readfirstlane(TR ? 0 : k0 * 2);
    if (!TR && k0 < K && k0 + BK > K) {                              // the last, cut step: pieces behind K are nowhere from here on
#pragma unroll
      for (int d = 0; d < DMA; ++d) if (k0 + piece_of(d, wave, lane) * 8 >= K) voff[d] = NOWHERE;
    }
  }
  template <int D>
  __device__ __forceinline__ void issue(unsigned shift) const {
    const unsigned to = __builtin_amdgcn_readfirstlane(lds0 + shift);
    asm volatile("s_add_u32 m0, %2, %4\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds" ::"v"(voff[D]), "s"(rsrc), "s"(to), "s"(soff),
                 "n"(D * WAVES * 1024)
                 : "memory", "m0", "scc");
  }
};

template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (N > 0) {
    each<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

template <bool TR, int ROWS>
struct Reader {
  // lane -> its place in a fragment's rows; fragment (t, ks): rows w0 + 16 t .. + 15, k 32 ks .. + 31
  unsigned at;
  __device__ __forceinline__ void init(int w0, int lane) {
    const int kg = lane >> 4;
    if constexpr (TR) {
      const int k = kg * 8 + ((lane & 15) >> 2), q = lane & 3, c = w0 / 8 + (q >> 1);
      at = unsigned(k * ROWS * 2 + ((c ^ (turn<ROWS>(k) << 1)) * 16) + (q & 1) * 8);
    } else {
      const int row = w0 + (lane & 15);
      at = unsigned(row * 128 + ((kg ^ ((row >> 1) & 7)) * 16));
    }
  }
  template <class F>
  __device__ __forceinline__ F read(const char* tile, int t, int ks) const {
    if constexpr (TR) {
      const char* p = tile + (at ^ (t << 5)) + ks * (32 * ROWS * 2);
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef short s8 __attribute__((ext_vector_type(8)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p));
      const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * ROWS * 2));
      const s8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(F, v);
    } else {
      return *reinterpret_cast<const F*>(tile + (at ^ (ks << 6)) + t * (16 * 128));
    }
  }
};

// eight values beside each other, `width` of them there (more than eight: all); a row may start anywhere
template <class T>
__device__ __forceinline__ typename Vec<T>::type round8(const float (&v)[8]) {
  typename Vec<T>::type o;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = T(v[e]);
  return o;
}
template <class T>
__device__ __forceinline__ void put8(T* to, const float (&v)[8], int width) {
  const typename Vec<T>::type o = round8<T>(v);
  if (width >= 8) { store_vec<false>(to, o); return; }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < width) to[e] = o[e];
}
__device__ __forceinline__ void put8(float* to, const float (&v)[8], int width) {
  if (width >= 8) {
    *reinterpret_cast<f32x4_u*>(to) = f32x4_u{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4_u*>(to + 4) = f32x4_u{v[4], v[5], v[6], v[7]};
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < width) to[e] = v[e];
}
template <class T>
__device__ __forceinline__ void get8(float (&v)[8], const T* from, int width) {
  if (width >= 8) {
    const typename Vec<T>::type x = *reinterpret_cast<const typename Vec<T>::type*>(from);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = float(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < width ? float(from[e]) : 0.f;
  }
}
// (the choice once for eight values: it is the same for the whole launch)
__device__ __forceinline__ void act_values(float (&v)[8], int act, float beta) {
  if (act == ACT_NONE) return;
#define NPHM_EACH(A) case A: _Pragma("unroll") for (int e = 0; e < 8; ++e) v[e] = act_value(v[e], A, beta); break
  switch (act) { NPHM_EACH(ACT_RELU); NPHM_EACH(ACT_SILU); NPHM_EACH(ACT_GELU); NPHM_EACH(ACT_SOFTPLUS); }
#undef NPHM_EACH
}

// what follows a product of the forward pass, for eight values with their bias: z as it is kept, then y
template <class T>
__device__ __forceinline__ void layer_out(float (&v)[8], const GemmArgs& p, int64_t at, int width) {
  if (p.z) {
    float k[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = float(keep<T>(v[e]));
    put8(static_cast<T*>(p.z) + at, k, width);
  }
  float r[8] = {};
  if (p.residual) get8(r, static_cast<const T*>(p.residual) + at, width);
  act_values(v, p.act, p.beta);
  if (p.residual) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  }
  put8(static_cast<T*>(p.C) + at, v, width);
}

// U rows `row` elements apart, all there.  (The empty asm keeps the compiler from making one store, without the hint, of the two.)
template <class T, int U>
__device__ __forceinline__ void put_rows(T* to, const typename Vec<T>::type (&o)[U], int64_t row, bool stream) {
  if (stream) {
    asm volatile("");
#pragma unroll
    for (int u = 0; u < U; ++u) store_vec<true>(to + u * row, o[u]);
    asm volatile("");
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) store_vec<false>(to + u * row, o[u]);
  }
}

// the same for U rows: what is asked once for them stands between them, not in front of each
template <class T, int ACT, int U>
__device__ __forceinline__ void layer_rows(float (&v)[U][8], const GemmArgs& p, int64_t at, int64_t row) {
  typename Vec<T>::type r[U];
  if (p.z) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) r[u][e] = keep<T>(v[u][e]);
    put_rows<T, U>(static_cast<T*>(p.z) + at, r, row, p.stream_z);
  }
  if (p.residual) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = *reinterpret_cast<const typename Vec<T>::type*>(static_cast<const T*>(p.residual) + at + u * row);
  }
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[u][e] = act_value(v[u][e], ACT, p.beta);
  if (p.residual) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] += float(r[u][e]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) r[u] = round8<T>(v[u]);
  put_rows<T, U>(static_cast<T*>(p.C) + at, r, row, p.stream_c);
}

enum { OUT_LAYER = 0, OUT_PLAIN = 1, OUT_PARTS = 2, OUT_EITHER = 3 };       // EITHER: PARTS where the k range is split, else PLAIN

// One tile BM x BN of C[i, j] = sum_k A(i, k) B(j, k), by WM x WN wavefronts.  256 x 256 by eight: a wavefront's 128 x 64 is 128 accumulators a
// lane, and its fragments take 12 KiB of LDS reads for 32 k.  Tried with 32 x 32 x 16 instructions (8192 x 4096 x 4096: 206 us): four
// wavefronts of 128 x 128 read less, but nothing stands in for one that waits (218); blocks that stay and fetch the next tile's first steps
// while the last one's results leave (209: loads wait behind a wavefront's stores); slots of 32 k, a barrier twice as often, slower.
template <class T, int BM, int BN, int WM, int WN, bool TA, bool TB, int OUT>
__device__ __forceinline__ void gemm_tile(const GemmArgs& p, int block) {
  constexpr int WAVES = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  typedef Operand<T, BM, WAVES, TA> OpA;
  typedef Operand<T, BN, WAVES, TB> OpB;
  constexpr unsigned SLOT = OpA::BYTES;
  static_assert(OpA::BYTES == OpB::BYTES, "slots take tiles of either operand");
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Blocks go round the 8 XCDs: each XCD gets a run of consecutive tiles, 8 tiles of i to one of j, so that the 32 that it works on
  // at a time share 8 + 4 panels in its L2.
  const int mt = (p.I + BM - 1) / BM, nt = (p.J + BN - 1) / BN, tiles = mt * nt * p.splits, per = (tiles + 7) / 8;
  const int tile = (block & 7) * per + (block >> 3);
  if ((block >> 3) >= per || tile >= tiles) return;
  const int split = tile / (mt * nt), rest = tile % (mt * nt);
  const int group = rest / (8 * nt), m_first = group * 8, m_count = min(8, mt - m_first), in = rest - group * 8 * nt;
  const int i0 = (m_first + in % m_count) * BM, j0 = in / m_count * BN;
  const int kb = split * p.k_per_split, ke = min(p.K, kb + p.k_per_split);
  const unsigned lds0 = unsigned(size_t((__attribute__((address_space(3))) char*)lds));

  OpA a;
  OpB b;
  a.init(p.A, p.lda, i0, p.I, ke, wave, lane, lds0);
  b.init(p.B, p.ldb, j0, p.J, ke, wave, lane, lds0);
  Reader<TA, BM> ra;
  Reader<TB, BN> rb;
  ra.init((wave / WN) * TM * 16, lane);
  rb.init((wave % WN) * TN * 16, lane);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int x = 0; x < TM; ++x)
#pragma unroll
    for (int y = 0; y < TN; ++y) acc[x][y] = f32x4{};
  typedef typename Frag<T>::type frag;

  // Fragments come from LDS while products run that do not need them, one or two reads behind a product: B's for the next 32 k beside those
  // in use, an A fragment's successor into its own registers as soon as its last product is issued.  The step's barrier stands LEAD
  // fragments of A into its last 32 k: the last read of this step is then old enough not to be waited for, and behind it the first
  // fragments of the next step are read and the loads of the one after it start, each behind a product too (a wavefront issues in
  // order: a burst of either would leave the matrix pipe idle).  16384 x 16384 x 4096: 1609 us with LEAD 2, 1556 with 4; where A lies row beside
  // row 2 is a little better.
  constexpr int NMUL = TM * TN, NREAD = TM + TN, LEAD = TM < 8 ? 1 : TA ? 2 : 4, EARLY = NMUL + LEAD * TN, LATE = NMUL - LEAD * TN;
  frag fa[TM], fb[2][TN];
  auto read_one = [&](int set, const char* at, const char* bt, int ks, int n) __attribute__((always_inline)) {
    if (n < TN) fb[set][n] = rb.template read<frag>(bt, n, ks);
    else fa[n - TN] = ra.template read<frag>(at, n - TN, ks);
  };
  // behind product `m` of 32 k: those of the NREAD reads whose turn it is, spread over the products from `from` on; an A fragment's not before
  // its last product
  auto reads = [&](int set, const char* at, const char* bt, int ks, int m, int from) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NREAD; ++n) {
      const int even = from + n * (NMUL - from) / NREAD, last = n < TN ? 0 : (n - TN + 1) * TN - 1;
      if (m == (even > last ? even : last)) read_one(set, at, bt, ks, n);
    }
  };
  // products [from, to) of 32 k
  auto multiply = [&](int set, int from, int to, auto&& behind) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < NMUL; ++m) {
      if (m < from || m >= to) continue;
      acc[m / TN][m % TN] = mfma(fb[set][m % TN], fa[m / TN], acc[m / TN][m % TN]);
      __builtin_amdgcn_sched_barrier(0);
      behind(m);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // LDS holds five tiles, A and B in turn: A of step t in slot 2 t, B in slot 2 t + 1 (modulo 5).  Step t loads A of step t + 2 into the slot
  // that B of step t - 1 has left, spread over what is in front of its barrier, and behind it B of step t + 2 into A's own slot:
  // the loads' rate is two thirds of what the path takes, in bursts it would hold up the products.
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (u & 1) {
      b.aim(kb + u / 2 * BK, lane, wave);
      each<OpB::DMA>([&](auto d) __attribute__((always_inline)) { b.template issue<decltype(d)::value>(u * SLOT); });
    } else {
      a.aim(kb + u / 2 * BK, lane, wave);
      each<OpA::DMA>([&](auto d) __attribute__((always_inline)) { a.template issue<decltype(d)::value>(u * SLOT); });
    }
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(OpA::DMA + OpB::DMA) : "memory");
  unsigned sa = 0, sb = SLOT, sfree = 4 * SLOT;
  auto two_on = [](unsigned slot) { const unsigned v = slot + 2 * SLOT; return v >= SLOTS * SLOT ? v - SLOTS * SLOT : v; };
#pragma unroll
  for (int n = 0; n < NREAD; ++n) read_one(0, lds + sa, lds + sb, 0, n);
  for (int k0 = kb; k0 < ke; k0 += BK) {
    a.aim(k0 + 2 * BK, lane, wave);
    auto load_a = [&](int m) __attribute__((always_inline)) {
      each<OpA::DMA>([&](auto d) __attribute__((always_inline)) {
        if (decltype(d)::value * EARLY / OpA::DMA == m) a.template issue<decltype(d)::value>(sfree);
      });
    };
    multiply(0, 0, NMUL, [&](int m) __attribute__((always_inline)) {
      reads(1, lds + sa, lds + sb, 1, m, 0);
      load_a(m);
    });
    multiply(1, 0, LEAD * TN, [&](int m) __attribute__((always_inline)) { load_a(NMUL + m); });
    // the next step's tiles have landed (the A behind them may still be on its way), every wavefront has read this step's out
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(OpA::DMA) : "memory");
    const unsigned na = two_on(sa), nb = two_on(sb);
    b.aim(k0 + 2 * BK, lane, wave);
    multiply(1, LEAD * TN, NMUL, [&](int m) __attribute__((always_inline)) {
      reads(0, lds + na, lds + nb, 0, m, LEAD * TN);                    // (behind the last step: nothing that is used)
      each<OpB::DMA>([&](auto d) __attribute__((always_inline)) {
        if (LEAD * TN + decltype(d)::value * LATE / OpB::DMA == m) b.template issue<decltype(d)::value>(sa);
      });
    });
    sfree = sb;
    sa = na;
    sb = nb;
  }

  // Register q of a lane: i = lane % 16, j = 4 (lane / 16) + q of its 16 x 16 tile.  Through LDS (every wavefront its own part of the tiles'
  // room, AT rows at a time) to eight j beside each other a lane: whole 128-byte pieces of C, z and the residual.
  constexpr int COLS = TN * 16, PITCH = COLS + 4, LPR = COLS / 8, RPI = 64 / LPR, AT = TM * 16 < 64 ? TM * 16 : 64, U = AT / RPI < 4 ? AT / RPI : 4;
  static_assert(WAVES * AT * PITCH * 4 <= SLOTS * SLOT, "the epilogue's rows fit the tiles' room");
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");      // every wavefront has left the tiles, no load is on its way
  float* out = reinterpret_cast<float*>(lds) + wave * AT * PITCH;
  const int j = j0 + (wave % WN) * COLS + (lane % LPR) * 8, width = min(8, p.J - j);
  const bool inside = i0 + BM <= p.I && j0 + BN <= p.J;
  const bool parts = OUT == OUT_PARTS || (OUT == OUT_EITHER && p.splits > 1);
  float* const to_parts = p.parts + int64_t(split) * p.I * p.J;
  float bias[8] = {};
  if (OUT == OUT_LAYER && p.bias && width > 0) get8(bias, static_cast<const T*>(p.bias) + j, width);
#pragma nounroll
  for (int x0 = 0; x0 < TM; x0 += AT / 16) {
    each<TM * 16 / AT>([&](auto part) __attribute__((always_inline)) {
      if (decltype(part)::value * (AT / 16) != x0) return;
#pragma unroll
      for (int x = 0; x < AT / 16; ++x)
#pragma unroll
        for (int y = 0; y < TN; ++y)
          *reinterpret_cast<f32x4*>(out + (x * 16 + (lane & 15)) * PITCH + y * 16 + 4 * (lane >> 4)) = acc[decltype(part)::value * (AT / 16) + x][y];
    });
    const int i = i0 + (wave / WN) * TM * 16 + x0 * 16 + lane / LPR;
    const float* from = out + lane / LPR * PITCH + (lane % LPR) * 8;
    auto take = [&](float (&v)[8], int r) __attribute__((always_inline)) {
      *reinterpret_cast<f32x4*>(v) = *reinterpret_cast<const f32x4*>(from + r * PITCH);
      *reinterpret_cast<f32x4*>(v + 4) = *reinterpret_cast<const f32x4*>(from + r * PITCH + 4);
      if constexpr (OUT == OUT_LAYER) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
      }
    };
    if (inside) {                                                      // U rows at a time, without a look at the ends
      auto rows = [&](auto act) __attribute__((always_inline)) {
#pragma nounroll
        for (int r = 0; r < AT; r += U * RPI) {
          float v[U][8];
          const int64_t at = int64_t(i + r) * p.J + j, row = int64_t(RPI) * p.J;
#pragma unroll
          for (int u = 0; u < U; ++u) take(v[u], r + u * RPI);
          if constexpr (OUT == OUT_LAYER) {
            layer_rows<T, decltype(act)::value, U>(v, p, at, row);
          } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
              if (parts) put8(to_parts + at + u * row, v[u], 8);
              else put8(static_cast<T*>(p.C) + at + u * row, v[u], 8);
            }
          }
        }
      };
      if constexpr (OUT == OUT_LAYER) {
#define NPHM_EACH(A) case A: rows(std::integral_constant<int, A>{}); break
        switch (p.act) { NPHM_EACH(ACT_NONE); NPHM_EACH(ACT_RELU); NPHM_EACH(ACT_SILU); NPHM_EACH(ACT_GELU); NPHM_EACH(ACT_SOFTPLUS); }
#undef NPHM_EACH
      } else {
        rows(std::integral_constant<int, ACT_NONE>{});
      }
    } else {
#pragma nounroll
      for (int r = 0; r < AT; r += RPI) {
        if (i + r >= p.I || width <= 0) continue;
        float v[8];
        take(v, r);
        const int64_t at = int64_t(i + r) * p.J + j;
        if (parts) put8(to_parts + at, v, width);
        else if constexpr (OUT == OUT_LAYER) layer_out<T>(v, p, at, width);
        else put8(static_cast<T*>(p.C) + at, v, width);
      }
    }
  }
}

// wavefronts a SIMD that LDS has room for: told to the compiler, which would put fragments into accumulator registers and back for more
// (1024 x 1024 x 16384 in tiles of 128: 62 us so, 44 told)
constexpr int waves_of(int size) { return size == 64 ? 4 : 2; }

template <class T, int B, int WM, int WN, bool TA, bool TB, int OUT>
__global__ __launch_bounds__(64 * WM * WN) __attribute__((amdgpu_waves_per_eu(waves_of(B), waves_of(B)))) void gemm_kernel(GemmArgs p) {
  gemm_tile<T, B, B, WM, WN, TA, TB, OUT>(p, blockIdx.x);
}

// rows of `cols` elements -> rows of `ld` elements (whole 16-byte pieces), zeros behind them; 16 lanes a row; one or two operands
struct Pack {
  const void* src;
  void* dst;
  int64_t rows;
};

template <class T>
__device__ __forceinline__ void pack_rows(Pack p, const Pack& q, unsigned blocks, unsigned block, int cols, int ld) {
  typedef typename Vec<T>::type vec;
  if (block >= blocks) p = q, block -= blocks;
  const int64_t r = int64_t(block) * 16 + threadIdx.x / 16;
  if (r >= p.rows) return;
  const T* s = static_cast<const T*>(p.src) + r * cols;
  T* d = static_cast<T*>(p.dst) + r * ld;
  const int whole = cols / 8 * 8, c0 = (threadIdx.x % 16) * 8;
#pragma unroll 4
  for (int c = c0; c < whole; c += 128) *reinterpret_cast<vec*>(d + c) = *reinterpret_cast<const vec*>(s + c);
  if (whole < ld && c0 == whole % 128) {
    vec v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = whole + e < cols ? s[whole + e] : T(0.f);
    *reinterpret_cast<vec*>(d + whole) = v;
  }
}
template <class T>
__global__ __launch_bounds__(256) void pack_kernel(Pack p, Pack q, unsigned blocks, int cols, int ld) {
  pack_rows<T>(p, q, blocks, blockIdx.x, cols, ld);
}

// the partial products of all k ranges, added in order, and what the tiles' epilogue does otherwise; a thread takes eight elements beside
// each other, across the ends of rows.  From SLICED ranges on (small results, then) eight threads share them, every eighth range each.
constexpr int SLICED = 16, SLICES = 8;

template <class T, int OUT>
__device__ __forceinline__ void join_splits(const GemmArgs& p, int block, int blocks) {
  __shared__ float part[SLICES - 1][256 / SLICES][9];
  const int64_t count = int64_t(p.I) * p.J;
  const bool sliced = p.splits >= SLICED;
  const int step = sliced ? SLICES : 1, per = 256 / step, slice = sliced ? threadIdx.x / per : 0, piece = threadIdx.x % per;
  for (int64_t base = int64_t(block) * per * 8; base < count; base += int64_t(blocks) * per * 8) {
    const int64_t at = base + piece * 8;
    const int width = int(min(count - at, int64_t(8)));
    float v[8] = {};
    if (width == 8) {
#pragma unroll 4
      for (int s = slice; s < p.splits; s += step) {
        const float* q = p.parts + int64_t(s) * count + at;
        const f32x4_u lo = *reinterpret_cast<const f32x4_u*>(q), hi = *reinterpret_cast<const f32x4_u*>(q + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
      }
    } else {
      for (int s = slice; s < p.splits; s += step)
#pragma unroll
        for (int e = 0; e < 8; ++e) if (e < width) v[e] += p.parts[int64_t(s) * count + at + e];
    }
    if (sliced) {
      if (slice)
#pragma unroll
        for (int e = 0; e < 8; ++e) part[slice - 1][piece][e] = v[e];
      __syncthreads();
      if (!slice)
#pragma unroll
        for (int w = 0; w < SLICES - 1; ++w)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += part[w][piece][e];
      __syncthreads();
    }
    if (slice || width <= 0) continue;
    if constexpr (OUT == OUT_LAYER) {
      if (p.bias) {
        int j = int(at % p.J);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] += float(static_cast<const T*>(p.bias)[j]);
          j = j + 1 == p.J ? 0 : j + 1;
        }
      }
      layer_out<T>(v, p, at, width);
    } else {
      put8(static_cast<T*>(p.C) + at, v, width);
    }
  }
}

// both products' partial products: blocks below `first` take p, the others q
template <class T>
__global__ __launch_bounds__(256) void join_pair_kernel(GemmArgs p, GemmArgs q, int first) {
  const int b = blockIdx.x;
  if (b < first) join_splits<T, OUT_PLAIN>(p, b, first);
  else join_splits<T, OUT_PLAIN>(q, b - first, int(gridDim.x) - first);
}

// gz = g a'(z) (rows `ld` elements apart, zeros behind them) and the column sums of every tile of rows of it (before it is rounded).  A
// thread takes eight columns of ROWS rows; LPR threads a row, 256 / LPR rows side by side.  Bound by memory: 16384 x 1024 with Softplus,
// 101 MB in 18 to 23 us (4.4 TB/s and more, as much as is still in the last cache).
// The blocks behind its own pack the operands of the products that follow (a launch less: 4095 x 515 -> 1024, 4 us).
struct Packs {
  Pack p, q;
  unsigned blocks;                       // of p
  int cols, ld;
};

template <class T, int LPR, int ROWS, bool STREAM>
__global__ __launch_bounds__(256) void gz_kernel(const T* g, const T* z, T* gz, float* sums, T* dbias, int M, int N, int ld, int act, float beta,
                                                 int tiles, unsigned own, Packs packs) {
  constexpr int SIDE = 256 / LPR;
  typedef typename Vec<T>::type vec;
  __shared__ float part[256][9];
  if (blockIdx.x >= own) return pack_rows<T>(packs.p, packs.q, packs.blocks, blockIdx.x - own, packs.cols, packs.ld);
  const int tile = int(blockIdx.x % unsigned(tiles)), side = int(blockIdx.x / unsigned(tiles));
  const int c = (side * LPR + threadIdx.x % LPR) * 8, m0 = tile * (SIDE * ROWS) + threadIdx.x / LPR;
  float s[8] = {};
  if (c < ld) {
#pragma unroll 4
    for (int r = 0; r < ROWS; ++r) {
      const int m = m0 + r * SIDE;
      if (m >= M) continue;
      const int64_t at = int64_t(m) * N + c;
      float v[8] = {}, zz[8] = {};
      if (c + 8 <= N) {
        const vec x = load_vec<STREAM>(g + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = float(x[e]);
        if (z) {
          const vec y = load_vec<STREAM>(z + at);
#pragma unroll
          for (int e = 0; e < 8; ++e) zz[e] = float(y[e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) if (c + e < N) { v[e] = float(g[at + e]); if (z) zz[e] = float(z[at + e]); }
      }
      if (z) {
#define NPHM_EACH(A) case A: _Pragma("unroll") for (int e = 0; e < 8; ++e) v[e] *= act_slope(zz[e], A, beta); break
        switch (act) { NPHM_EACH(ACT_RELU); NPHM_EACH(ACT_SILU); NPHM_EACH(ACT_GELU); NPHM_EACH(ACT_SOFTPLUS); }
#undef NPHM_EACH
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += c + e < N ? v[e] : 0.f;
      if (gz) {
        vec o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = c + e < N ? T(v[e]) : T(0.f);
        *reinterpret_cast<vec*>(gz + int64_t(m) * ld + c) = o;
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) part[threadIdx.x][e] = s[e];
  __syncthreads();
  for (int u = threadIdx.x; u < LPR * 8; u += 256) {
    const int n = side * LPR * 8 + u;
    if (n >= N) continue;
    float o = 0.f;
#pragma unroll
    for (int k = 0; k < SIDE; ++k) o += part[k * LPR + u / 8][u % 8];
    if (tiles == 1) dbias[n] = T(o);
    else sums[int64_t(tile) * N + n] = o;
  }
}

// the tiles' sums, added up: 32 columns a block, eight threads a column (part: [8][32])
struct Columns {
  const float* sums;
  void* out;
  int tiles, N;
};
template <class T>
__device__ __forceinline__ void column_sums(const Columns& c, int block, float (*part)[32]) {
  const float* sums = c.sums;
  T* out = static_cast<T*>(c.out);
  const int tiles = c.tiles, N = c.N;
  const int col = threadIdx.x & 31, k = threadIdx.x >> 5, n = block * 32 + col;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (int t = k; t < tiles; t += 8) s += sums[int64_t(t) * N + n];
  }
  part[k][col] = s;
  __syncthreads();
  if (k || n >= N) return;
#pragma unroll
  for (int q = 1; q < 8; ++q) s += part[q][col];
  out[n] = T(s);
}
template <class T>
__global__ __launch_bounds__(256) void column_sums16_kernel(Columns c) {
  __shared__ float part[8][32];
  column_sums<T>(c, blockIdx.x, part);
}

// blocks below `own` join p, the others add up columns
template <class T, int OUT>
__global__ __launch_bounds__(256) void join_splits_kernel(GemmArgs p, int own, Columns c) {
  __shared__ float part[8][32];
  if (int(blockIdx.x) < own) join_splits<T, OUT>(p, blockIdx.x, own);
  else column_sums<T>(c, blockIdx.x - own, part);
}

// dx, dW and the last sums of db side by side in one launch, where none of them fills the chip: blocks [0, bx) make dx in tiles of BX,
// [bx, bw) dW in tiles of BW, the others db (4095 x 515 -> 1024: 25 us, 33 + 4 one after the other).
template <class T, int BX, int BW>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(waves_of(BX > BW ? BX : BW), waves_of(BX > BW ? BX : BW)))) void gradients_kernel(GemmArgs x, GemmArgs w, Columns c, int bx, int bw) {
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int b = blockIdx.x;
  if (b < bx) gemm_tile<T, BX, BX, 2, 2, false, true, OUT_EITHER>(x, b);
  else if (b < bw) gemm_tile<T, BW, BW, 2, 2, true, true, OUT_EITHER>(w, b - bx);
  else column_sums<T>(c, b - bw, reinterpret_cast<float(*)[32]>(lds));
}

inline unsigned pack_blocks(const Pack& p) { return unsigned((p.rows + 15) / 16); }
inline size_t up(size_t v) { return (v + 255) / 256 * 256; }
inline int gz_lanes(int64_t ldn) { return ldn <= 64 ? 8 : ldn <= 128 ? 16 : ldn <= 256 ? 32 : 64; }
// rows a thread: 16 where that leaves 512 blocks, for fewer sums to add up (16384 x 1024: 30 us, 32 with 4), else 4 (4095 x 1024: 11 us, 13 with 8)
inline int gz_rows(int64_t M, int64_t ldn) {
  const int64_t lanes = gz_lanes(ldn), rows = 256 / lanes * 16;
  return (M + rows - 1) / rows * ((ldn + lanes * 8 - 1) / (lanes * 8)) >= 512 ? 16 : 4;
}
inline int64_t gz_tiles(int64_t M, int64_t ldn) { const int64_t rows = 256 / gz_lanes(ldn) * gz_rows(M, ldn); return (M + rows - 1) / rows; }

// -> what is left to add up for dbias (tiles 0: nothing)
template <class T>
inline Columns make_gz(hipStream_t st, const T* g, const T* z, T* gz, float* sums, T* dbias, int M, int N, int ld, int act, float beta, const Packs& packs) {
  const int lanes = gz_lanes(ld), tiles = int(gz_tiles(M, ld));
  const unsigned own = unsigned(tiles) * unsigned((ld + lanes * 8 - 1) / (lanes * 8)), grid = own + packs.blocks + pack_blocks(packs.q);
  float* s = dbias ? sums : nullptr;
  const bool many = gz_rows(M, ld) == 16;
  auto go = [&](auto lanes_c) {
    constexpr int L = decltype(lanes_c)::value;
    if (many && gz && int64_t(M) * N * 2 >= Z_KEPT)
      hipLaunchKernelGGL((gz_kernel<T, L, 16, true>), dim3(grid), dim3(256), 0, st, g, z, gz, s, dbias, M, N, ld, act, beta, tiles, own, packs);
    else if (many) hipLaunchKernelGGL((gz_kernel<T, L, 16, false>), dim3(grid), dim3(256), 0, st, g, z, gz, s, dbias, M, N, ld, act, beta, tiles, own, packs);
    else hipLaunchKernelGGL((gz_kernel<T, L, 4, false>), dim3(grid), dim3(256), 0, st, g, z, gz, s, dbias, M, N, ld, act, beta, tiles, own, packs);
  };
  if (lanes == 8) go(std::integral_constant<int, 8>{});
  else if (lanes == 16) go(std::integral_constant<int, 16>{});
  else if (lanes == 32) go(std::integral_constant<int, 32>{});
  else go(std::integral_constant<int, 64>{});
  return Columns{sums, dbias, dbias && tiles > 1 ? tiles : 0, N};
}

inline int64_t whole8(int64_t v) { return (v + 7) / 8 * 8; }

struct Tiling { int size, splits; };               // size: 256, 128 or 64
// Among the tiles that fill the 256 CUs the size whose fullest CU is done first: a tile takes its steps of 64 k, times what an element of it
// costs against one of a 256-tile (LDS is read more often for a smaller one), and as many steps again for its first loads and its
// epilogue, of which small tiles hide more behind each other.  Fitted to 16384 x 1024 x 1024 (36, 43, 67 us in tiles of 256, 128, 64),
// 5000 x 1000 x 5000 (-, 86, 120), 200000 x 64 x 64 (83, 42, 26), 5000 x 5000 x 64 (46, 42, 38); 35200 x 512 x 512: 33 us, 39 in tiles of 256,
// of which the second round has 20.  Where none fills them, or 128-tiles do with the k range in pieces of 1024 and more, pieces, added by a
// second launch: with tiles of 128 (1024 x 1024 x 16384: 46 us in four, 56 whole in tiles of 64; 1024 x 512 x 32768: 48 in eight, 104 in
// two with tiles of 64), else of 64 (1 x 4096 x 4096: 9.6 us in eight, 32 whole; 128 x 128 x 100000: 18 us in 64, 46 in 16; 1024 x 1024 x
// 1024: 8.5 us whole, 14 in two).
inline Tiling tiling(int64_t I, int64_t J, int64_t K) {
  auto tiles = [&](int64_t b) { return ((I + b - 1) / b) * ((J + b - 1) / b); };
  const int64_t t128 = tiles(128), t64 = tiles(64);
  const double steps = double((K + BK - 1) / BK);
  Tiling best{64, 1};
  double least = 0;
  auto offer = [&](int size, double element, double ends) {
    if (tiles(size) < 192) return;
    const double cost = double((tiles(size) + 255) / 256) * size * size * (element * steps + ends);
    if (least == 0 || cost < least) best.size = size, least = cost;
  };
  offer(256, 1.0, 8.0);
  offer(128, 1.4, 7.0);
  offer(64, 2.8, 4.7);
  const int64_t s128 = (256 + t128 - 1) / t128;
  if (t128 < 192 && I > 64 && J > 64 && K >= 4096 && s128 * 1024 <= K) return {128, int(s128)};
  if (least > 0 || K <= 1024) return best;
  const int64_t fill = I <= 64 ? 512 : 256, s = std::min<int64_t>((fill + t64 - 1) / t64, K / 512);
  return {64, int(std::max<int64_t>(s, 1))};
}
inline size_t parts_bytes(const Tiling& t, int64_t I, int64_t J) { return t.splits > 1 ? up(size_t(t.splits) * I * J * 4) : 0; }

// tells the device once of a kernel that takes more LDS than it would give unasked (a refusal shows at the launch)
template <auto KERNEL>
inline void allow_lds(unsigned bytes) {
  if (bytes <= 65536) return;
  static std::atomic<uint64_t> told{0};                              // devices that know, by their numbers
  int dev = 0;
  (void)hipGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (told.load(std::memory_order_relaxed) & bit) return;
  (void)hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
  told.fetch_or(bit, std::memory_order_relaxed);
}
constexpr unsigned lds_of(int size) { return SLOTS * size * BK * 2; }
static_assert(lds_of(256) <= 160 * 1024, "the slots fit");
// blocks of a product in tiles of `size`, whole rounds of the XCDs
inline int64_t blocks_of(const GemmArgs& a, int size) {
  return (((a.I + size - 1) / size) * int64_t((a.J + size - 1) / size) * a.splits + 7) / 8 * 8;
}

template <class T, int B, int WM, int WN, bool TA, bool TB, int OUT>
inline void launch_gemm(hipStream_t st, const GemmArgs& a) {
  allow_lds<&gemm_kernel<T, B, WM, WN, TA, TB, OUT>>(lds_of(B));
  hipLaunchKernelGGL((gemm_kernel<T, B, WM, WN, TA, TB, OUT>), dim3(unsigned(blocks_of(a, B))), dim3(64 * WM * WN), lds_of(B), st, a);
}

inline void split(GemmArgs& a, int splits) {
  a.k_per_split = ((a.K + splits - 1) / splits + BK - 1) / BK * BK;
  a.splits = (a.K + a.k_per_split - 1) / a.k_per_split;
}
inline int64_t join_blocks(const GemmArgs& a) {
  const int64_t each = a.splits >= SLICED ? 2048 / SLICES : 2048, want = (int64_t(a.I) * a.J + each - 1) / each;
  return want < 8192 ? want : 8192;
}

inline unsigned column_blocks(const Columns& c) { return c.tiles ? unsigned(c.N + 31) / 32 : 0; }
template <class T>
inline void sum_columns(hipStream_t st, const Columns& c) {
  if (c.tiles) hipLaunchKernelGGL((column_sums16_kernel<T>), dim3(column_blocks(c)), dim3(256), 0, st, c);
}

// the product, with its k range in t.splits pieces where that is more than one: `a.parts` has room for parts_bytes; and db's last sums
template <class T, bool TA, bool TB, int OUT>
inline void gemm(hipStream_t st, GemmArgs a, Tiling t, const Columns& columns = {}) {
  split(a, t.splits);
  auto launch = [&](auto out) {
    constexpr int O = decltype(out)::value;
    if constexpr (O != OUT_PARTS)                                    // (tiling() cuts k ranges for tiles of 128 and 64 alone)
      if (t.size == 256) return launch_gemm<T, 256, 2, 4, TA, TB, O>(st, a);
    if (t.size == 128) launch_gemm<T, 128, 2, 2, TA, TB, O>(st, a);
    else launch_gemm<T, 64, 2, 2, TA, TB, O>(st, a);
  };
  if (a.splits == 1) {
    sum_columns<T>(st, columns);
    return launch(std::integral_constant<int, OUT>{});
  }
  launch(std::integral_constant<int, OUT_PARTS>{});
  const int own = int(join_blocks(a));
  hipLaunchKernelGGL((join_splits_kernel<T, OUT>), dim3(own + column_blocks(columns)), dim3(256), 0, st, a, own, columns);
}

// dx, dW and db together (x, w: their own tilings of 64 or 128, rooms of their own for partial products)
template <class T, int BX, int BW>
inline void launch_gradients(hipStream_t st, GemmArgs x, GemmArgs w, const Columns& c) {
  constexpr unsigned LDS = lds_of(BX > BW ? BX : BW);
  allow_lds<&gradients_kernel<T, BX, BW>>(LDS);
  const int64_t bx = blocks_of(x, BX), bw = bx + blocks_of(w, BW), all = bw + column_blocks(c);
  hipLaunchKernelGGL((gradients_kernel<T, BX, BW>), dim3(unsigned(all)), dim3(256), LDS, st, x, w, c, int(bx), int(bw));
  const int64_t jx = x.splits > 1 ? join_blocks(x) : 0, jw = w.splits > 1 ? join_blocks(w) : 0;
  if (jx + jw == 0) return;
  hipLaunchKernelGGL((join_pair_kernel<T>), dim3(unsigned(jx + jw)), dim3(256), 0, st, x, w, int(jx));
}

// p, q or both (rows 0: not) in a launch of their own
template <class T>
inline void pack(hipStream_t st, const Packs& k) {
  const unsigned blocks = k.blocks + pack_blocks(k.q);
  if (blocks) hipLaunchKernelGGL((pack_kernel<T>), dim3(blocks), dim3(256), 0, st, k.p, k.q, k.blocks, k.cols, k.ld);
}
inline Packs packs_of(const Pack& p, const Pack& q, int64_t cols) { return Packs{p, q, pack_blocks(p), int(cols), int(whole8(cols))}; }

inline bool aligned(const void* p, unsigned to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

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

inline bool packed(const void* p, int64_t cols) { return cols % 8 || !aligned(p, 16); }     // rows that the tile loads do not take as they are

struct Forward {
  Tiling t;
  size_t x, weight, parts, total;
};
inline Forward forward_plan(const void* x, const void* weight, int64_t M, int64_t N, int64_t K) {
  Forward p;
  p.t = tiling(M, N, K);
  p.x = 0;
  p.weight = p.x + (packed(x, K) ? up(size_t(M) * whole8(K) * 2) : 0);
  p.parts = p.weight + (packed(weight, K) ? up(size_t(N) * whole8(K) * 2) : 0);
  p.total = p.parts + parts_bytes(p.t, M, N);
  return p;
}

struct Backward {
  Tiling x_t, w_t;
  bool same;                                        // g as it stands is gz
  size_t gz, sums, x, weight, parts_x, parts_w, total;      // byte offsets
};
inline Backward backward_plan(const void* g, const void* x, const void* weight, int64_t M, int64_t N, int64_t K, int act) {
  Backward p;
  p.x_t = tiling(M, K, N);
  p.w_t = tiling(N, K, M);
  p.same = act == ACT_NONE && !packed(g, N);
  p.gz = 0;
  p.sums = p.gz + (p.same || !(x || weight) ? 0 : up(size_t(M) * whole8(N) * 2));      // (db alone: nobody reads gz)
  p.x = p.sums + up(size_t(gz_tiles(M, whole8(N))) * N * 4);
  p.weight = p.x + (x && packed(x, K) ? up(size_t(M) * whole8(K) * 2) : 0);
  p.parts_x = p.weight + (weight && packed(weight, K) ? up(size_t(N) * whole8(K) * 2) : 0);
  p.parts_w = p.parts_x + (weight ? parts_bytes(p.x_t, M, K) : 0);
  p.total = p.parts_w + (x ? parts_bytes(p.w_t, N, K) : 0);
  return p;
}

}  // namespace train_ops
}  // namespace nphm

using namespace nphm::train_ops;

extern "C" {

size_t nphm_layer16_forward_workspace_bytes(const void* x, const void* weight, int64_t M, int64_t N, int64_t K) {
  return forward_plan(x, weight, M, N, K).total;
}

int nphm_layer16_forward(const void* x, const void* weight, const void* bias, const void* residual, void* y, void* z, int64_t M, int64_t N,
                         int64_t K, int dtype, int act, float beta, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_layer("nphm_layer16_forward", M, N, K, dtype, act, beta)) return rc;
  if (!x || !weight || !y) return nphm_fail_msg("nphm_layer16_forward: null pointer");
  const Forward plan = forward_plan(x, weight, M, N, K);
  if (workspace_bytes < plan.total || (plan.total && !workspace)) return nphm_fail_msg("nphm_layer16_forward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  with_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if constexpr (sizeof(T) == 2) {
      GemmArgs a{};
      a.A = x; a.lda = K;
      a.B = weight; a.ldb = K;
      const bool px = packed(x, K), pw = packed(weight, K);
      pack<T>(st, packs_of(Pack{x, ws + plan.x, px ? M : 0}, Pack{weight, ws + plan.weight, pw ? N : 0}, K));
      if (px) { a.A = ws + plan.x; a.lda = whole8(K); }
      if (pw) { a.B = ws + plan.weight; a.ldb = whole8(K); }
      a.I = int(M); a.J = int(N); a.K = int(K);
      a.C = y; a.bias = bias; a.residual = residual; a.z = z; a.act = act; a.beta = beta;
      a.stream_z = M * N * 2 >= Z_KEPT;
      a.stream_c = M * N * 2 >= CACHED;
      a.parts = reinterpret_cast<float*>(ws + plan.parts);
      gemm<T, false, false, OUT_LAYER>(st, a, plan.t);
    }
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_layer16_forward launch", e);
  return 0;
}

size_t nphm_layer16_backward_workspace_bytes(const void* g, const void* x, const void* weight, int64_t M, int64_t N, int64_t K, int act) {
  return backward_plan(g, x, weight, M, N, K, act).total;
}

int nphm_layer16_backward(const void* g, const void* x, const void* weight, const void* z, void* dx, void* dweight, void* dbias, int64_t M,
                          int64_t N, int64_t K, int dtype, int act, float beta, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_layer("nphm_layer16_backward", M, N, K, dtype, act, beta)) return rc;
  if (!g || (act != ACT_NONE && !z) || (dx && !weight) || (dweight && !x) || !workspace) return nphm_fail_msg("nphm_layer16_backward: null pointer");
  const Backward plan = backward_plan(g, x, weight, M, N, K, act);
  if (workspace_bytes < plan.total) return nphm_fail_msg("nphm_layer16_backward: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  with_dtype(dtype, [&](auto t) {
    typedef decltype(t) T;
    if constexpr (sizeof(T) == 2) {
      const int64_t ldn = whole8(N), ldk = whole8(K);
      T* gz = plan.same ? const_cast<T*>(static_cast<const T*>(g)) : reinterpret_cast<T*>(ws + plan.gz);
      const bool px = dweight && packed(x, K), pw = dx && packed(weight, K);
      const Packs packs = packs_of(Pack{x, ws + plan.x, px ? M : 0}, Pack{weight, ws + plan.weight, pw ? N : 0}, K);
      Columns columns{};
      if (!plan.same || dbias)
        columns = make_gz<T>(st, static_cast<const T*>(g), act == ACT_NONE ? nullptr : static_cast<const T*>(z), plan.same || !(dx || dweight) ? nullptr : gz,
                             reinterpret_cast<float*>(ws + plan.sums), static_cast<T*>(dbias), int(M), int(N), int(ldn), act, beta, packs);
      else
        pack<T>(st, packs);
      GemmArgs ax{}, aw{};
      ax.A = aw.A = gz;
      ax.lda = aw.lda = ldn;
      ax.B = pw ? ws + plan.weight : weight;
      ax.ldb = pw ? ldk : K;
      aw.B = px ? ws + plan.x : x;
      aw.ldb = px ? ldk : K;
      ax.I = int(M); ax.J = int(K); ax.K = int(N);
      aw.I = int(N); aw.J = int(K); aw.K = int(M);
      ax.C = dx;
      aw.C = dweight;
      ax.parts = reinterpret_cast<float*>(ws + plan.parts_x);
      aw.parts = reinterpret_cast<float*>(ws + plan.parts_w);
      if (dx && dweight && plan.x_t.size <= 128 && plan.w_t.size <= 128) {
        split(ax, plan.x_t.splits);
        split(aw, plan.w_t.splits);
        if (plan.x_t.size == 128 && plan.w_t.size == 128) launch_gradients<T, 128, 128>(st, ax, aw, columns);
        else if (plan.x_t.size == 128) launch_gradients<T, 128, 64>(st, ax, aw, columns);
        else if (plan.w_t.size == 128) launch_gradients<T, 64, 128>(st, ax, aw, columns);
        else launch_gradients<T, 64, 64>(st, ax, aw, columns);
      } else {
        if (dx) gemm<T, false, true, OUT_PLAIN>(st, ax, plan.x_t);
        if (dweight) gemm<T, true, true, OUT_PLAIN>(st, aw, plan.w_t, columns);
        else sum_columns<T>(st, columns);
      }
    }
  });
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return nphm_fail("nphm_layer16_backward launch", e);
  return 0;
}

}  // extern "C"
