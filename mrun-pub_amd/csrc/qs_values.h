// Values of an activation type in fp32 registers: loads, stores, conversions.
#pragma once

#include "qs_common.h"

namespace qs {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return static_cast<float>(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v) {  // round to nearest even
  return static_cast<T>(v);
}

// N consecutive values, N * sizeof(T) = 4, 8, 16 or a multiple of 16 bytes, aligned to
// that (to 16 for more).
template <class T, int N>
struct Pack {
  static constexpr int kBytes = N * sizeof(T);
  typedef T type __attribute__((ext_vector_type(kBytes >= 16 ? 16 / (int)sizeof(T) : N)));
  static constexpr int kEach = kBytes >= 16 ? 16 / (int)sizeof(T) : N;
};

template <class T, int N>
__device__ __forceinline__ void load_values(const T* p, float (&v)[N]) {
  using P = Pack<T, N>;
#pragma unroll
  for (int i = 0; i < N / P::kEach; ++i) {
    const typename P::type w = reinterpret_cast<const typename P::type*>(p)[i];
#pragma unroll
    for (int e = 0; e < P::kEach; ++e) v[i * P::kEach + e] = to_f32(w[e]);
  }
}

template <class T, int N>
__device__ __forceinline__ void store_values(T* p, const float (&v)[N]) {
  using P = Pack<T, N>;
#pragma unroll
  for (int i = 0; i < N / P::kEach; ++i) {
    typename P::type w;
#pragma unroll
    for (int e = 0; e < P::kEach; ++e) w[e] = from_f32<T>(v[i * P::kEach + e]);
    reinterpret_cast<typename P::type*>(p)[i] = w;
  }
}

}  // namespace qs
