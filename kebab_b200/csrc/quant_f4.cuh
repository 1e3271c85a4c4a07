// Codes and scales of blocks of 32 values in microscaled 4-bit floating point, of
// four lanes a block (quant_f4.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "quant_i8.cuh"

namespace kb {
namespace {

// Codes of eight values, the first in the lowest nibble. Nearest, ties to even.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Bits of the largest magnitude of the 32 values of four neighbouring lanes.
// Values of 16 bits are compared in pairs, as they are stored (their magnitudes
// order as integers, a NaN above everything).
template <typename T>
__device__ __forceinline__ uint32_t block_top(const Run<T, 8>& run) {
  if constexpr (sizeof(T) == 2) {
    constexpr uint32_t M = 0x7fff7fffu;
    const uint4 r = run.raw[0];
    uint32_t m = __vmaxu2(__vmaxu2(r.x & M, r.y & M), __vmaxu2(r.z & M, r.w & M));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint16_t h = (uint16_t)max(m >> 16, m & 0xffffu);
    return __float_as_uint(to_float(*reinterpret_cast<const T*>(&h)));
  } else {
    float v[8];
    run.values(v);
    uint32_t top = largest<8>(v, 0u);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    return max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  }
}

// The scale's byte and 2^-e.
struct BlockScale {
  uint32_t byte;
  float inv;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t top) {
  if (top >= 0x7f800000u) return {255u, 0.f};
  const int byte = max((int)((top + 0x3fffffu) >> 23) - 2, 0);
  return {(uint32_t)byte, __uint_as_float((uint32_t)(254 - byte) << 23)};
}

// Eight values' codes, and in 16 lanes' word the scales of their four blocks.
struct EightCodes {
  uint32_t codes, scales;
};
template <typename T>
__device__ __forceinline__ EightCodes eight_codes(const Run<T, 8>& run, int lane) {
  const BlockScale s = block_scale(block_top(run));
  float v[8];
  run.values(v);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= s.inv;
  EightCodes r;
  r.codes = s.byte == 255u ? 0u : codes8(v);  // 0: an infinity or NaN in the block
  r.scales = s.byte << (lane / 4 % 4 * 8);
  r.scales |= __shfl_xor_sync(0xffffffffu, r.scales, 4);
  r.scales |= __shfl_xor_sync(0xffffffffu, r.scales, 8);
  return r;
}
}  // namespace
}  // namespace kb
