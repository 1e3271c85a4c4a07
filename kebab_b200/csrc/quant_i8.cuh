// Row quantisation to 8-bit integers: what the quantising kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "vec.cuh"

namespace kb {

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

struct RowScale {
  float scale, inv;  // inv 0: the row's codes are 0
};

// From the bit pattern of the row's largest magnitude. Under 1e-30 the row is
// taken as zeros: 127 / amax would overflow. A row with an infinity or a NaN
// keeps that as its scale.
__device__ __forceinline__ RowScale row_scale(uint32_t top) {
  const float amax = __uint_as_float(top);
  if (amax < 1e-30f) return {0.f, 0.f};
  return {amax / 127.f, top < 0x7f800000u ? 127.f / amax : 0.f};
}

// rint(v * inv), at most 127 since |v| <= amax, as the low byte: added to
// 1.5 * 2^23 a value is rounded to an integer, ties to even, in the low bits of
// the sum. (The product is rounded on its own first; a conversion instruction
// takes several times an addition's issue slots.)
__device__ __forceinline__ uint32_t code_bits(float v, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.f));
}

// The low bytes of four.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int W>
__device__ __forceinline__ void store_codes(int8_t* out, const float (&v)[W], float inv) {
  if constexpr (W == 8) {
    uint32_t c[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) c[u] = inv == 0.f ? 0u : code_bits(v[u], inv);
    *reinterpret_cast<uint2*>(out) = make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
  } else {
#pragma unroll
    for (int u = 0; u < W; ++u) out[u] = inv == 0.f ? 0 : (int8_t)(code_bits(v[u], inv) & 0xffu);
  }
}

}  // namespace kb
