// Rows of 16- and 32-bit floats in registers: loads and stores of W values
// (W = 8: 16-byte accesses, the address 16-byte aligned; W = 1: any address).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace kb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int W>
__device__ __forceinline__ void load_row(const float* p, float (&v)[W]) {
  if constexpr (W == 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) v[u] = p[u];
  }
}

// 8 values of a 16-byte register.
__device__ __forceinline__ void unpack(const __half*, const uint4& r, float (&v)[8]) {
  const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 f = __half22float2(h[u]);
    v[2 * u] = f.x, v[2 * u + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const __nv_bfloat16*, const uint4& r, float (&v)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const float2 f = __bfloat1622float2(h[u]);
    v[2 * u] = f.x, v[2 * u + 1] = f.y;
  }
}

template <int W, typename T>
__device__ __forceinline__ void load_row(const T* p, float (&v)[W]) {
  if constexpr (W == 8) {
    unpack(p, *reinterpret_cast<const uint4*>(p), v);
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) v[u] = to_float(p[u]);
  }
}

template <int W, typename T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[W]) {
  if constexpr (W == 8) {
    alignas(16) T h[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) h[u] = from_float<T>(v[u]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) p[u] = from_float<T>(v[u]);
  }
}

}  // namespace kb
