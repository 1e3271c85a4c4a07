// Row quantisation to 8-bit integers: what the quantising kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vec.cuh"

namespace kb {

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
  float scale, inv;
};

// From the bit pattern of the row's largest magnitude. Under 1e-30 the row is
// taken as zeros: 127 / amax would overflow. An infinite or NaN amax gives
// inv = 0 or NaN, codes of 0 (a NaN converts to 0) and that scale.
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float amax = __uint_as_float(top);
  if (amax < 1e-30f) return {0.f, 0.f};
  return {amax / 127.f, 127.f / amax};
}

// |v * inv| rounds to at most 127 since |v| <= amax.
__device__ __forceinline__ int code_of(float v, float inv) { return __float2int_rn(v * inv); }

template <int W>
__device__ __forceinline__ void store_codes(int8_t* out, const float (&v)[W], float inv) {
  if constexpr (W == 8) {
    uint32_t w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) w[h] |= (uint32_t)(code_of(v[h * 4 + u], inv) & 0xff) << (8 * u);
    }
    *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) out[u] = (int8_t)code_of(v[u], inv);
  }
}

}  // namespace kb
