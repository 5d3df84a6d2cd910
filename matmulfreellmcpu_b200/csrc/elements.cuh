// elements.cuh -- fp32, bf16 and fp16 rows read and written as fp32 registers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>
#include <type_traits>

namespace mmfree_cuda {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V consecutive elements as they lie in memory, at most 16 bytes per access.
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T v[V];
};

// V elements as whole words, for values that stay in flight: a load into single 16-bit elements is taken apart, and so
// waited for, where it is issued.
template <typename T, int V>
struct Words {
  static constexpr int kBytes = sizeof(T) * V;
  using Type = std::conditional_t<kBytes == 2, uint16_t, std::conditional_t<kBytes == 4, uint32_t, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 16, uint4, Pack<uint4, 2>>>>>;
  Type w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const Type*>(p); }
  __device__ __forceinline__ float operator[](int i) const {
    Pack<T, V> k;
    memcpy(&k, &w, kBytes);
    return to_f32(k.v[i]);
  }
};

// V elements from a 16-byte aligned address (kVec), or the first n of them one by one.
template <bool kVec, typename T, int V>
__device__ __forceinline__ void load_row(const T* p, int n, float (&r)[V]) {
  if constexpr (kVec) {
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = to_f32(k.v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = i < n ? to_f32(p[i]) : 0.0f;
  }
}

template <bool kVec, typename T, int V>
__device__ __forceinline__ void store_row(T* p, int n, const float (&r)[V]) {
  if constexpr (kVec) {
    Pack<T, V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) k.v[i] = from_f32<T>(r[i]);
    *reinterpret_cast<Pack<T, V>*>(p) = k;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = from_f32<T>(r[i]);
  }
}

// Two values rounded to T: as they lie in memory, and as fp32 again.
__device__ __forceinline__ uint32_t round2(float& lo, float& hi, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &p, 4);
  lo = __uint_as_float(w << 16);
  hi = __uint_as_float(w & 0xFFFF0000u);
  return w;
}
__device__ __forceinline__ uint32_t round2(float& lo, float& hi, __half) {
  const __half2 p = __floats2half2_rn(lo, hi);
  uint32_t w;
  memcpy(&w, &p, 4);
  const float2 f = __half22float2(p);
  lo = f.x;
  hi = f.y;
  return w;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr float kLog2E = 1.44269504088896341f;

// 2^v and 1 / v by the special-function unit (relative errors of at most 2^-22 and 2^-23; below 2^-126 both are 0).
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float silu_f32(float v) { return v * rcp(1.0f + ex2(-v * kLog2E)); }

}  // namespace mmfree_cuda
