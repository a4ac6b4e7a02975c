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

template <int BYTES, int ALIGN>
struct dg_words {
  typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN)));
};

// VEC elements as they lie in memory.
template <typename T, int VEC>
struct dg_vec {
  T v[VEC];
};

// (through a vector of words: element-wise stores of a struct end up as such)
template <int VEC, int ALIGN, typename T>
__device__ __forceinline__ dg_vec<T, VEC> dg_load_raw(const T *p) {
  dg_vec<T, VEC> w;
  if constexpr (VEC == 1) {
    w.v[0] = *p;
  } else {
    typedef typename dg_words<sizeof(T) * VEC, ALIGN>::type words;
    const words q = *reinterpret_cast<const words *>(p);
    __builtin_memcpy(&w, &q, sizeof(w));
  }
  return w;
}

template <int VEC, int ALIGN, typename T>
__device__ __forceinline__ void dg_store_raw(T *p, const dg_vec<T, VEC> &w) {
  if constexpr (VEC == 1) {
    *p = w.v[0];
  } else {
    typedef typename dg_words<sizeof(T) * VEC, ALIGN>::type words;
    words q;
    __builtin_memcpy(&q, &w, sizeof(w));
    *reinterpret_cast<words *>(p) = q;
  }
}

template <int VEC, int ALIGN, typename T>
__device__ __forceinline__ void dg_load_at(const T *p, float (&f)[VEC]) {
  const dg_vec<T, VEC> w = dg_load_raw<VEC, ALIGN>(p);
#pragma unroll
  for (int e = 0; e < VEC; ++e) f[e] = dg_widen(w.v[e]);
}

template <int VEC, int ALIGN, typename T>
__device__ __forceinline__ void dg_store_at(T *p, const float (&f)[VEC]) {
  dg_vec<T, VEC> w;
#pragma unroll
  for (int e = 0; e < VEC; ++e) w.v[e] = dg_round<T>(f[e]);
  dg_store_raw<VEC, ALIGN>(p, w);
}

// Rows that start on 16 bytes.
template <int VEC, typename T>
__device__ __forceinline__ void dg_load(const T *p, float (&f)[VEC]) { dg_load_at<VEC, 16>(p, f); }
template <int VEC, typename T>
__device__ __forceinline__ void dg_store(T *p, const float (&f)[VEC]) { dg_store_at<VEC, 16>(p, f); }

// Rows that start anywhere: the hardware takes vector accesses at any address of an element (a few more cache lines
// touched), so only the ends of a row go element by element.
template <int VEC, typename T>
__device__ __forceinline__ void dg_load_unaligned(const T *p, float (&f)[VEC]) { dg_load_at<VEC, 2>(p, f); }
template <int VEC, typename T>
__device__ __forceinline__ void dg_store_unaligned(T *p, const float (&f)[VEC]) { dg_store_at<VEC, 2>(p, f); }
