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
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(h)[i];
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) p[u] = from_float<T>(v[u]);
  }
}

// W values of a row as they are stored (W = 8 of F32: two registers of 16 bytes).
template <typename T, int W>
struct Run {
  static constexpr int N = W == 8 ? (int)sizeof(T) / 2 : 1;
  uint4 raw[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (W == 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      raw[0].x = __float_as_uint(to_float(*p));
    }
  }
  __device__ __forceinline__ void values(float (&v)[W]) const {
    if constexpr (W == 8 && sizeof(T) == 2) {
      unpack((const T*)nullptr, raw[0], v);
    } else if constexpr (W == 8) {
      const uint32_t b[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[N - 1].x, raw[N - 1].y, raw[N - 1].z, raw[N - 1].w};
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = __uint_as_float(b[u]);
    } else {
      v[0] = __uint_as_float(raw[0].x);
    }
  }
  // The values, rounded to T.
  __device__ __forceinline__ void set(const float (&v)[W]) {
    if constexpr (W == 8) {
      alignas(16) T h[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) h[u] = from_float<T>(v[u]);
#pragma unroll
      for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(h)[i];
    } else {
      raw[0].x = __float_as_uint(to_float(from_float<T>(v[0])));
    }
  }
};

}  // namespace kb
