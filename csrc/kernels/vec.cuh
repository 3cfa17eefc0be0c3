// Vectors of N values of an activation type (bf16, fp16 or fp32) and their exact widening to fp32.
#pragma once

#include "common.cuh"

namespace mtorus {

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void widen(const Vec<T, N>& a, float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = to_f<T>(a.v[i]);
}

// One rounding to nearest of each value.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> narrow(const float* f) {
  Vec<T, N> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.v[i] = from_f<T>(f[i]);
  return a;
}

// Streaming (read once) load and store: the line is the first to leave L1 and L2.
template <typename V>
__device__ __forceinline__ V load_stream(const V* p) {
  V r;
  if constexpr (sizeof(V) == 16) {
    *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else if constexpr (sizeof(V) == 8) {
    *reinterpret_cast<uint2*>(&r) = __ldcs(reinterpret_cast<const uint2*>(p));
  } else if constexpr (sizeof(V) == 4) {
    *reinterpret_cast<uint32_t*>(&r) = __ldcs(reinterpret_cast<const uint32_t*>(p));
  } else {
    static_assert(sizeof(V) == 2, "vectors of 2, 4, 8 or 16 bytes");
    *reinterpret_cast<uint16_t*>(&r) = __ldcs(reinterpret_cast<const uint16_t*>(p));
  }
  return r;
}

template <typename V>
__device__ __forceinline__ void store_stream(V* p, const V& a) {
  if constexpr (sizeof(V) == 16) {
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&a));
  } else if constexpr (sizeof(V) == 8) {
    __stcs(reinterpret_cast<uint2*>(p), *reinterpret_cast<const uint2*>(&a));
  } else if constexpr (sizeof(V) == 4) {
    __stcs(reinterpret_cast<uint32_t*>(p), *reinterpret_cast<const uint32_t*>(&a));
  } else {
    static_assert(sizeof(V) == 2, "vectors of 2, 4, 8 or 16 bytes");
    __stcs(reinterpret_cast<uint16_t*>(p), *reinterpret_cast<const uint16_t*>(&a));
  }
}

// f(T{}) with the activation type of a checked tensor.
template <typename F>
inline void dispatch_act(at::ScalarType t, F&& f) {
  switch (t) {
    case at::kBFloat16: f(bf16{}); break;
    case at::kHalf: f(__half{}); break;
    case at::kFloat: f(float{}); break;
    default: TORCH_CHECK_TYPE(false, "activations are bf16, fp16 or fp32, not ", t);
  }
}

}  // namespace mtorus
