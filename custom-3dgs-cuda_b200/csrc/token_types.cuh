// Element types of the token operators (rotary positions, norms, attention): 32-bit floats, half
// and bfloat16 in memory, 32-bit arithmetic, one rounding when a result is written.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gs3d_b200.h"

namespace gs {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N elements of T moved as one aligned access (N * sizeof(T) is 2, 4, 8 or 16 bytes, or 32 bytes
// as two accesses of 16).
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[N]) {
  const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_f32<T>(a.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[N]) {
  Pack<T, N> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.v[i] = from_f32<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = a;
}

// The larger of two, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

inline size_t element_size(int dtype) { return dtype == GS_FP32 ? 4 : 2; }
inline bool known_type(int dtype) {
  return dtype == GS_FP32 || dtype == GS_FP16 || dtype == GS_BF16;
}

}  // namespace gs
