// Element types of the operators that take more than fp32: loads widen to fp32, stores round once (to nearest, ties to
// even), VEC elements at a time.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef _Float16 dg_f16;
struct dg_bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float dg_widen(float v) { return v; }
__device__ __forceinline__ float dg_widen(dg_f16 v) { return (float)v; }
__device__ __forceinline__ float dg_widen(dg_bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

template <typename T>
__device__ __forceinline__ T dg_round(float v);
template <>
__device__ __forceinline__ float dg_round<float>(float v) { return v; }
template <>
__device__ __forceinline__ dg_f16 dg_round<dg_f16>(float v) { return (dg_f16)v; }
template <>
__device__ __forceinline__ dg_bf16 dg_round<dg_bf16>(float v) {
  return {__builtin_bit_cast(uint16_t, (__bf16)v)};
}

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) dg_vec {
  T v[VEC];
};

template <int VEC, typename T>
__device__ __forceinline__ void dg_load(const T *p, float (&f)[VEC]) {
  const dg_vec<T, VEC> w = *reinterpret_cast<const dg_vec<T, VEC> *>(p);
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = dg_widen(w.v[e]);
}

template <int VEC, typename T>
__device__ __forceinline__ void dg_store(T *p, const float (&f)[VEC]) {
  dg_vec<T, VEC> w;
#pragma unroll
  for (int e = 0; e < VEC; ++e) w.v[e] = dg_round<T>(f[e]);
  *reinterpret_cast<dg_vec<T, VEC> *>(p) = w;
}

// The same for rows that start anywhere: the hardware takes vector accesses at any address of an element (a few more
// cache lines touched), so only the ends of a row go element by element.
template <int BYTES>
struct dg_words {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(2)));
};

template <int VEC, typename T>
__device__ __forceinline__ void dg_load_unaligned(const T *p, float (&f)[VEC]) {
  const typename dg_words<sizeof(T) * VEC>::type q = *reinterpret_cast<const typename dg_words<sizeof(T) * VEC>::type *>(p);
  T w[VEC];
  __builtin_memcpy(w, &q, sizeof(w));
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = dg_widen(w[e]);
}

template <int VEC, typename T>
__device__ __forceinline__ void dg_store_unaligned(T *p, const float (&f)[VEC]) {
  T w[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) w[e] = dg_round<T>(f[e]);
  typename dg_words<sizeof(T) * VEC>::type q;
  __builtin_memcpy(&q, w, sizeof(w));
  *reinterpret_cast<typename dg_words<sizeof(T) * VEC>::type *>(p) = q;
}
