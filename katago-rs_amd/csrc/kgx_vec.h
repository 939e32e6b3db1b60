// Vectors of 16 bytes of a row at its elements' alignment, as floats; `left`: the row's elements from there on.
#pragma once
#include "kgx_device.h"

namespace kgx {

typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x8_any __attribute__((ext_vector_type(8), aligned(2)));
template <typename T> inline constexpr int kVec = 16 / sizeof(T);
template <typename T> struct RowVec { typedef u16x8_any type; };
template <> struct RowVec<float> { typedef f32x4_any type; };

template <typename T>
__device__ __forceinline__ float widen1(const typename RowVec<T>::type& v, int j) {
  if constexpr (std::is_same<T, float>::value) return v[j];
  else if constexpr (std::is_same<T, bf16>::value) return __uint_as_float((unsigned)v[j] << 16);
  else return (float)__builtin_bit_cast(f16, (unsigned short)v[j]);
}
template <typename T>
__device__ __forceinline__ void load_vec(const T* p, int left, float (&f)[kVec<T>]) {
  if (left >= kVec<T>) {
    const typename RowVec<T>::type v = *(const typename RowVec<T>::type*)p;
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) f[j] = widen1<T>(v, j);
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++) f[j] = j < left ? (float)p[j] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, int left, const float (&f)[kVec<T>]) {
  T t[kVec<T>];
#pragma unroll
  for (int j = 0; j < kVec<T>; j++) t[j] = to_t<T>(f[j]);
  if (left >= kVec<T>) {
    *(typename RowVec<T>::type*)p = __builtin_bit_cast(typename RowVec<T>::type, t);
  } else {
#pragma unroll
    for (int j = 0; j < kVec<T>; j++)
      if (j < left) p[j] = t[j];
  }
}
// A whole vector past the caches.
template <typename T>
__device__ __forceinline__ void store_past(T* p, const float (&f)[kVec<T>]) {
  T t[kVec<T>];
#pragma unroll
  for (int j = 0; j < kVec<T>; j++) t[j] = to_t<T>(f[j]);
  asm volatile("");  // (or this and a plain store in another branch become one, a plain one)
  __builtin_nontemporal_store(__builtin_bit_cast(typename RowVec<T>::type, t), (typename RowVec<T>::type*)p);
  asm volatile("");
}

}  // namespace kgx
