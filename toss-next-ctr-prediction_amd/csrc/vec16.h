// Element types of the 16-bit / fp32 operators (ln.hip, diffattn.hip, newton_schulz.hip): codes of the C ABI, and
// 8-element vector access at any alignment of the element (global dwordx4 accesses need none on gfx950).
#pragma once
#include "common.h"

namespace ctr {

enum { TY_F32 = 0, TY_BF16 = 1, TY_F16 = 2 };

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Vec;
template <> struct Vec<__bf16> { typedef bf16x8 v8; typedef bf16x4 v4; };
template <> struct Vec<_Float16> { typedef f16x8 v8; typedef f16x4 v4; };
template <> struct Vec<float> { typedef f32x8 v8; typedef f32x4 v4; };

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 ld8(const T* p) {
  typename Vec<T>::v8 v;
  __builtin_memcpy(&v, p, sizeof(v));
  return v;
}
template <typename T>
__device__ __forceinline__ void st8(T* p, typename Vec<T>::v8 v) { __builtin_memcpy(p, &v, sizeof(v)); }

// the 8 elements from p of which n are there (the others read 0 / are not written)
template <typename T>
__device__ __forceinline__ f32x8 ld8f(const T* p, int n) {
  if (n >= 8) return __builtin_convertvector(ld8(p), f32x8);
  f32x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = i < n ? (float)p[i] : 0.f;
  return o;
}
template <typename T>
__device__ __forceinline__ void st8f(T* p, f32x8 v, int n) {
  typename Vec<T>::v8 o = __builtin_convertvector(v, typename Vec<T>::v8);
  if (n >= 8) { st8(p, o); return; }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = o[i];
}

}  // namespace ctr
