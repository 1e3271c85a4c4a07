// Quantisation to microscaled 4-bit floating point, and back.
//
// Four lanes take a block of 32 values, 8 each, so that a warp reads 512
// contiguous bytes of a row (16-bit types): the largest magnitude by two
// shuffles, the scale's exponent from its bits (adding 0x3fffff carries into
// the exponent if the mantissa is above 1.5, so that the result is the least
// power of two of which amax is at most 6), the codes by the conversion
// instruction after an exact multiplication by a power of two. Four blocks'
// scales make a word. Bound by memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>

#include "f4.h"
#include "kebab/f4.h"
#include "quant_i8.cuh"

namespace kb {
namespace {
constexpr int THREADS = 256, WARPS = THREADS / 32;

// Codes of two values: `lo` in the low nibble. Nearest, ties to even, at most 6.
__device__ __forceinline__ uint32_t codes2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 c, z;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n\t"
      "mov.b32 %0, {c, 0, 0, 0};\n\t}"
      : "=r"(r)
      : "f"(lo), "f"(hi));
  return r;
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

struct QuantArgs {
  const void* X;
  int64_t ldx, x_stride;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows;     // of a matrix
  int K, tiles;     // tiles: runs of 128 values
  int64_t entries;  // tokens: R + F4_SLACK
};

// A warp takes 256 values (two runs of 128) of a row; blockIdx.y is the matrix.
// TOKENS picks the layout of the scales.
template <typename T, bool VEC, bool TOKENS>
__global__ void __launch_bounds__(THREADS) quantize_f4_kernel(const QuantArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int spans = (g.tiles + 1) / 2;  // of 256 values
  const int64_t at = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int64_t padded = TOKENS ? g.rows : (g.rows + 127) / 128 * 128;
  if (at >= padded * spans) return;
  const int64_t row = at / spans;
  const int k = (int)(at - row * spans) * 256 + lane * 8;
  float v[8];
  const bool real = row < g.rows;
  const T* x = static_cast<const T*>(g.X) + blockIdx.y * g.x_stride + row * g.ldx;
  if (VEC && real && k + 8 <= g.K) {
    load_row<8>(x + k, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = real && k + i < g.K ? to_float(x[k + i]) : 0.f;
  }
  uint32_t top = largest<8>(v, 0u);
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const BlockScale s = block_scale(top);
  uint32_t word = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = s.byte == 255u ? 0.f : v[2 * i] * s.inv, hi = s.byte == 255u ? 0.f : v[2 * i + 1] * s.inv;
    word |= codes2(lo, hi) << (8 * i);
  }
  const int pitch = (int)f4_pitch(g.K);
  if (real && k / 2 < pitch)
    *reinterpret_cast<uint32_t*>(g.codes + (blockIdx.y * g.rows + row) * (int64_t)pitch + k / 2) = word;
  // Of 16 lanes, the scales of blocks 0 .. 3.
  uint32_t scales = s.byte << (lane / 4 % 4 * 8);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 4);
  scales |= __shfl_xor_sync(0xffffffffu, scales, 8);
  const int tile = k / 128, part = lane % 16;
  if (tile >= g.tiles) return;
  if (TOKENS) {
    const int64_t entry = row - 32 * part;
    if (part < 4 && entry >= 0)
      reinterpret_cast<uint32_t*>(g.scales)[(tile * g.entries + entry) * 4 + part] = scales;
  } else if (part == 0) {
    uint8_t* to = g.scales + ((blockIdx.y * (padded / 128) + row / 128) * g.tiles + tile) * 512;
    *reinterpret_cast<uint32_t*>(to + row % 32 * 16 + row % 128 / 32 * 4) = scales;
  }
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* W;
  int64_t rows;
  int K, tiles;
};

// The value of a code's low nibble: 2^e times its magnitude, by a table of halves.
__device__ __forceinline__ float value_of(uint32_t code, float scale) {
  const float m = (float)(0xC8643210u >> (code & 7u) * 4 & 15u) * 0.5f;
  return (code & 8u ? -m : m) * scale;
}

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255u ? 0x7fffffffu : byte << 23);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) dequantize_f4_kernel(const DequantArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int runs = (g.K + 7) / 8;
  const int64_t at = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (at >= g.rows * runs) return;
  const int64_t row = at / runs;
  const int k = (int)(at - row * runs) * 8;
  const uint32_t word =
      *reinterpret_cast<const uint32_t*>(g.codes + (blockIdx.y * g.rows + row) * f4_pitch(g.K) + k / 2);
  const uint8_t* tile = g.scales + ((blockIdx.y * ((g.rows + 127) / 128) + row / 128) * g.tiles + k / 128) * 512;
  const float scale = scale_of(tile[row % 32 * 16 + row % 128 / 32 * 4 + k / 32 % 4]);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = value_of(word >> (4 * i), scale);
  T* w = static_cast<T*>(g.W) + (blockIdx.y * g.rows + row) * (int64_t)g.K + k;
  if (VEC) {
    store_row<8>(w, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < g.K) w[i] = from_float<T>(v[i]);
  }
}

constexpr int64_t kMaxDim = int64_t(1) << 30;

template <typename T, bool TOKENS>
int quantize(const QuantArgs& g, int64_t E, cudaStream_t stream) {
  const int64_t rows = TOKENS ? g.rows : (g.rows + 127) / 128 * 128;
  const int64_t blocks = (rows * ((g.tiles + 1) / 2) + WARPS - 1) / WARPS;
  if (blocks > INT32_MAX) return fail(KEBAB_EINVAL, "quantize_f4: too many values");
  const bool vec = (reinterpret_cast<uintptr_t>(g.X) & 15u) == 0 && (g.ldx * sizeof(T)) % 16 == 0 &&
                   (E == 1 || (g.x_stride * sizeof(T)) % 16 == 0);
  PdlLaunch l(dim3((unsigned)blocks, (unsigned)E), dim3(THREADS), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(
      &l.cfg, vec ? quantize_f4_kernel<T, true, TOKENS> : quantize_f4_kernel<T, false, TOKENS>, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "quantize_f4 launch");
}

template <bool TOKENS>
int quantize_any(int dtype, const QuantArgs& g, int64_t E, cudaStream_t s) {
  return dtype == KEBAB_F16    ? quantize<__half, TOKENS>(g, E, s)
         : dtype == KEBAB_BF16 ? quantize<__nv_bfloat16, TOKENS>(g, E, s)
                               : quantize<float, TOKENS>(g, E, s);
}

template <typename T>
int dequantize(const DequantArgs& g, int64_t E, cudaStream_t stream) {
  const int64_t blocks = (g.rows * ((g.K + 7) / 8) + THREADS - 1) / THREADS;
  if (blocks > INT32_MAX) return fail(KEBAB_EINVAL, "dequantize_f4: too many values");
  const bool vec = (reinterpret_cast<uintptr_t>(g.W) & 15u) == 0 && g.K % 8 == 0;
  PdlLaunch l(dim3((unsigned)blocks, (unsigned)E), dim3(THREADS), 0, stream);
  const cudaError_t e =
      cudaLaunchKernelEx(&l.cfg, vec ? dequantize_f4_kernel<T, true> : dequantize_f4_kernel<T, false>, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "dequantize_f4 launch");
}

int check_any(const char* what, int dtype, int64_t E, int64_t rows, int64_t K, bool empty_ok) {
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16 && dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16, BF16 and F32 are implemented");
  if (E < 1 || E > kMaxExperts)
    return fail(KEBAB_EINVAL, std::string(what) + ": number of matrices " + std::to_string(E) + " is not in 1.." +
                                  std::to_string(kMaxExperts));
  if (rows < (empty_ok ? 0 : 1) || K <= 0 || rows > kMaxDim || K > kMaxDim)
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions rows=" + std::to_string(rows) +
                                  " K=" + std::to_string(K));
  return KEBAB_OK;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int64_t kebab_f4_code_bytes(int64_t rows, int64_t K) {
  if (rows < 0 || K <= 0 || rows > kMaxDim || K > kMaxDim) return -KEBAB_EINVAL;
  return rows * f4_pitch(K);
}

int64_t kebab_f4_weight_scale_bytes(int64_t N, int64_t K) {
  if (N <= 0 || K <= 0 || N > kMaxDim || K > kMaxDim) return -KEBAB_EINVAL;
  return (N + 127) / 128 * ((K + 127) / 128) * 512;
}

int64_t kebab_f4_token_scale_bytes(int64_t R, int64_t K) {
  if (R < 0 || K <= 0 || R > F4_MAX_ROWS || K > kMaxDim) return -KEBAB_EINVAL;
  return (K + 127) / 128 * (R + F4_SLACK) * 16;
}

int kebab_quantize_f4(kebab_dtype dtype, const void* W, int64_t ldw, int64_t w_stride, uint8_t* codes, uint8_t* scales,
                      int64_t E, int64_t N, int64_t K, kebab_stream_t stream) {
  return guarded([&] {
    const int rc = check_any("quantize_f4", dtype, E, N, K, false);
    if (rc) return rc;
    if (ldw < K) return fail(KEBAB_EINVAL, "quantize_f4: the row pitch is below the row length");
    if (!W || !codes || !scales) return fail(KEBAB_EINVAL, "quantize_f4: null pointer");
    if (!on16(codes) || !on16(scales))
      return fail(KEBAB_EINVAL, "quantize_f4: codes and scales must be 16-byte aligned");
    const QuantArgs g = {W, ldw, w_stride, codes, scales, N, (int)K, (int)((K + 127) / 128), 0};
    return quantize_any<false>(dtype, g, E, reinterpret_cast<cudaStream_t>(stream));
  });
}

int kebab_quantize_f4_tokens(kebab_dtype dtype, const void* X, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t R,
                             int64_t K, kebab_stream_t stream) {
  return guarded([&] {
    const int rc = check_any("quantize_f4_tokens", dtype, 1, R, K, true);
    if (rc) return rc;
    if (R > F4_MAX_ROWS) return fail(KEBAB_EINVAL, "quantize_f4_tokens: more than 2^27 rows");
    if (ldx < K) return fail(KEBAB_EINVAL, "quantize_f4_tokens: the row pitch is below the row length");
    if (R == 0) return KEBAB_OK;
    if (!X || !codes || !scales) return fail(KEBAB_EINVAL, "quantize_f4_tokens: null pointer");
    if (!on16(codes) || !on16(scales))
      return fail(KEBAB_EINVAL, "quantize_f4_tokens: codes and scales must be 16-byte aligned");
    const QuantArgs g = {X, ldx, 0, codes, scales, R, (int)K, (int)((K + 127) / 128), R + F4_SLACK};
    return quantize_any<true>(dtype, g, 1, reinterpret_cast<cudaStream_t>(stream));
  });
}

int kebab_dequantize_f4(kebab_dtype dtype, const uint8_t* codes, const uint8_t* scales, void* W, int64_t E, int64_t N,
                        int64_t K, kebab_stream_t stream) {
  return guarded([&] {
    const int rc = check_any("dequantize_f4", dtype, E, N, K, false);
    if (rc) return rc;
    if (!W || !codes || !scales) return fail(KEBAB_EINVAL, "dequantize_f4: null pointer");
    if (!on16(codes) || !on16(scales))
      return fail(KEBAB_EINVAL, "dequantize_f4: codes and scales must be 16-byte aligned");
    const DequantArgs g = {codes, scales, W, N, (int)K, (int)((K + 127) / 128)};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == KEBAB_F16 ? dequantize<__half>(g, E, s) : dtype == KEBAB_BF16 ? dequantize<__nv_bfloat16>(g, E, s) : dequantize<float>(g, E, s);
  });
}

}  // extern "C"
