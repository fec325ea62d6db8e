// train_ops_common.h — element types, unaligned vectors and reductions shared by the training operators (rows_kernels.hip,
// clip_kernels.hip, layer16_kernels.hip)
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nphm {
namespace train_ops {

typedef _Float16 fp16;
typedef __bf16 bf16;

// 16 bytes of a row.  Aligned to ONE element only: rows of odd width and views that start anywhere take the same wide loads (the
// global memory path of gfx950 accepts any byte address)
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
typedef bf16 bf16x8_u __attribute__((ext_vector_type(8), aligned(2)));
typedef fp16 fp16x8_u __attribute__((ext_vector_type(8), aligned(2)));

template <class T> struct Vec;
template <> struct Vec<float> { typedef f32x4_u type; static constexpr int N = 4; };
template <> struct Vec<bf16> { typedef bf16x8_u type; static constexpr int N = 8; };
template <> struct Vec<fp16> { typedef fp16x8_u type; static constexpr int N = 8; };

// the last cache, bytes.  Work that does not fit into it says so: what it reads for the last time, or writes without a chance to be read from
// there, is not kept
constexpr int64_t CACHED = int64_t(256) << 20;
// (the choice is made at compile time: of two accesses that differ in nothing else the compiler makes one, without the hint)
template <bool STREAM, class T>
__device__ __forceinline__ typename Vec<T>::type load_vec(const T* p) {
  const auto* from = reinterpret_cast<const typename Vec<T>::type*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(from);
  else return *from;
}
template <bool STREAM, class T>
__device__ __forceinline__ void store_vec(T* p, const typename Vec<T>::type& v) {
  auto* to = reinterpret_cast<typename Vec<T>::type*>(p);
  if constexpr (STREAM) __builtin_nontemporal_store(v, to);
  else *to = v;
}

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
inline bool dtype_ok(int d) { return d >= DT_F32 && d <= DT_F16; }
inline int dtype_size(int d) { return d == DT_F32 ? 4 : 2; }

// f(T{}) for the element type of code d
template <class F>
inline void with_dtype(int d, F&& f) {
  if (d == DT_F32) f(float{});
  else if (d == DT_BF16) f(bf16{});
  else f(fp16{});
}

}  // namespace train_ops
}  // namespace nphm
