// Vectors of N values of an activation type (bf16, fp16 or fp32) and their exact widening to fp32.
#pragma once

#include "common.cuh"

namespace mtorus {

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// A pair of 16-bit values in one 32-bit word, lower half first.
template <typename T>
__device__ __forceinline__ float2 widen_pair(uint32_t w);
template <>
__device__ __forceinline__ float2 widen_pair<bf16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 widen_pair<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T>
__device__ __forceinline__ uint32_t narrow_pair(float2 f);
template <>
__device__ __forceinline__ uint32_t narrow_pair<bf16>(float2 f) {
  const bf162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t narrow_pair<__half>(float2 f) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int N>
__device__ __forceinline__ void widen(const Vec<T, N>& a, float* f) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&a);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 t = widen_pair<T>(w[i]);
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f<T>(a.v[i]);
  }
}

// One rounding to nearest of each value.
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> narrow(const float* f) {
  Vec<T, N> a;
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&a);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = narrow_pair<T>(make_float2(f[2 * i], f[2 * i + 1]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = from_f<T>(f[i]);
  }
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

// Packed fp32 pairs: one instruction for two values (sm_100 f32x2), each rounded as on its own.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// 16-byte asynchronous copy global -> shared (address d); reads the first `bytes` bytes only, zeros take the others' place.
__device__ __forceinline__ void copy_async16(uint32_t d, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `pending` (0 .. 3) of this thread's youngest groups are in flight.
__device__ __forceinline__ void copy_async_wait(int pending) {
  if (pending >= 3)
    asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending == 2)
    asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (pending == 1)
    asm volatile("cp.async.wait_group 1;" ::: "memory");
  else
    asm volatile("cp.async.wait_group 0;" ::: "memory");
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
