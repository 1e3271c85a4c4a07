// Quantisation to microscaled 4-bit floating point, and back.
//
// Four lanes take a block of 32 values, 8 each, so that a warp reads 512
// contiguous bytes of a row (16-bit types): the largest magnitude by two
// shuffles, the scale's exponent from its bits (adding 0x3fffff carries into
// the exponent if the mantissa is above 1.5, so that the result is the least
// power of two of which amax is at most 6), the codes by the conversion
// instruction after an exact multiplication by a power of two. Four blocks'
// scales make a word. Bound by memory, and near it by the ALU (16-bit types: 83
// instructions of a warp for 256 values): 8192 x 8192 BF16 in 29 us, 5.8 TB/s,
// and back in 35; FP32 45 and 72. Rows that start anywhere are loaded value by
// value (8192 x 8191 BF16 47 us).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "f4.h"
#include "kebab/f4.h"
#include "quant_f4.cuh"

namespace kb {
namespace {
constexpr int THREADS = 256, WARPS = THREADS / 32;

struct QuantArgs {
  const void* X;
  int64_t ldx, x_stride;
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows;  // of a matrix
  int K, tiles;  // tiles: runs of 128 values
  int spans;     // runs of 256 values that a warp takes
  int64_t entries;  // tokens: R + F4_SLACK
};

// A warp takes spans of 256 values (two runs of 128) of a row, four of them in
// flight; blockIdx.y is the part of the row, blockIdx.z the matrix. TOKENS picks
// the layout of the scales.
template <typename T, bool VEC, bool TOKENS>
__global__ void __launch_bounds__(THREADS) quantize_f4_kernel(const QuantArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, part = lane % 16;
  const int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  const bool real = row < g.rows;
  const int64_t row_tiles = (g.rows + 127) / 128;
  if (TOKENS ? !real : row >= row_tiles * 128) return;
  const T* x = static_cast<const T*>(g.X) + blockIdx.z * g.x_stride + row * g.ldx;
  const int pitch = (int)f4_pitch(g.K);
  uint8_t* codes = g.codes + (blockIdx.z * g.rows + row) * (int64_t)pitch;
  const int64_t entry = row - 32 * part;
  // Where this lane's words of scales go: the place of tile 0, and the next tile's.
  uint32_t* to = reinterpret_cast<uint32_t*>(g.scales);
  if (TOKENS) to += entry * 4 + part;
  else to += (blockIdx.z * row_tiles + row / 128) * g.tiles * 128 + row % 32 * 4 + row % 128 / 32;
  const int64_t step = TOKENS ? g.entries * 4 : 128;
  const bool writes = TOKENS ? part < 4 && entry >= 0 : part == 0;
  const int begin = (int)blockIdx.y * g.spans * 256, end = min(begin + g.spans * 256, g.tiles * 128);
  // The codes and scales of 8 values a lane from k on; INSIDE: all of the span is within the row.
  auto span = [&](auto inside, Run<T, 8>& run, int k) {
    constexpr bool INSIDE = decltype(inside)::value;
    const EightCodes r = eight_codes(run, lane);
    if (INSIDE || (real && k / 2 < pitch)) *reinterpret_cast<uint32_t*>(codes + k / 2) = r.codes;
    const int tile = k / 128;
    if (writes && (INSIDE || tile < g.tiles)) to[tile * step] = r.scales;
  };
  constexpr int UNROLL = 4;
  int k0 = begin;
  if (VEC && real) {
    const T* from = x + lane * 8;
    for (; k0 + UNROLL * 256 <= min(end, g.K); k0 += UNROLL * 256) {
      Run<T, 8> run[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) run[u].load(from + k0 + u * 256);
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) span(std::true_type(), run[u], k0 + u * 256 + lane * 8);
    }
  }
  for (; k0 < end; k0 += 256) {
    const int k = k0 + lane * 8;
    Run<T, 8> run;
    if (VEC && real && k + 8 <= g.K) {
      run.load(x + k);
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = real && k + i < g.K ? to_float(x[k + i]) : 0.f;
      run.set(v);
    }
    span(std::false_type(), run, k);
  }
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* W;
  int64_t rows;
  int K, tiles, spans;
};

// The values of a byte's two codes, the low nibble's first.
__device__ __forceinline__ float2 values2(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 c, x, y, z;\n\t"
      "mov.b32 {c, x, y, z}, %1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, c;\n\t}"
      : "=r"(h)
      : "r"(byte));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255u ? 0x7fffffffu : byte << 23);
}

// A warp takes spans of 256 values of a row, four in flight; 8 values a lane, of
// a 16-byte granule of W (SHIFT: rows that start `off` values into their first
// granule; then the codes of the eight are cut from two words, and they may lie
// in two blocks).
template <typename T, bool SHIFT>
__global__ void __launch_bounds__(THREADS) dequantize_f4_kernel(const DequantArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (row >= g.rows) return;
  const int pitch = (int)f4_pitch(g.K);
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(g.codes + (blockIdx.z * g.rows + row) * (int64_t)pitch);
  const uint8_t* scales = g.scales + (blockIdx.z * ((g.rows + 127) / 128) + row / 128) * g.tiles * 512 + row % 32 * 16 +
                          row % 128 / 32 * 4;
  T* w = static_cast<T*>(g.W) + (blockIdx.z * g.rows + row) * (int64_t)g.K;
  const int off = SHIFT ? (int)((reinterpret_cast<uintptr_t>(w) & 15u) / sizeof(T)) : 0;
  const int begin = (int)blockIdx.y * g.spans * 256, end = min(begin + g.spans * 256, g.K + off);
  auto scale_at = [&](int k) { return scale_of(scales[k / 128 * 512 + k / 32 % 4]); };
  constexpr int UNROLL = 4;
  for (int k0 = begin + lane * 8 - off; k0 < end - off; k0 += UNROLL * 256) {
    uint32_t word[UNROLL], next[UNROLL];
    float first[UNROLL], second[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int k = k0 + u * 256;
      if (k < end - off) {
        word[u] = k >= 0 ? codes[k >> 3] : 0u;
        first[u] = k >= 0 ? scale_at(k) : 0.f;
        if (SHIFT) {
          const int last = min(k + 7, g.K - 1);
          next[u] = codes[last >> 3];
          second[u] = scale_at(last);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int k = k0 + u * 256;
      if (k >= end - off) break;
      const uint32_t eight = SHIFT ? __funnelshift_r(word[u], next[u], (k & 7) * 4) : word[u];
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 two = values2(eight >> (8 * i));
        v[2 * i] = two.x, v[2 * i + 1] = two.y;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= SHIFT && ((k + i) >> 5) != (k >> 5) ? second[u] : first[u];
      if (!SHIFT || (k >= 0 && k + 8 <= g.K)) {
        store_row<8>(w + k, v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i >= 0 && k + i < g.K) w[k + i] = from_float<T>(v[i]);
      }
    }
  }
}

constexpr int64_t kMaxDim = int64_t(1) << 30;

// Spans of 256 values that a warp takes of a row: as many as leave every SM its
// 64 warps. (8192 x 8192 of 8, 4, 1: 37, 39, 74 us; 4096 x 4096 18, 16, 22; 16
// rows of 8192 10, 8, 6, flushed and with the launch.)
int spans_of(int64_t rows, int64_t spans, int sms) {
  const int64_t warps = (int64_t)sms * 64;
  return rows * spans >= warps * 8 ? 8 : rows * spans >= warps * 4 ? 4 : 1;
}

template <typename T, bool TOKENS>
int quantize(QuantArgs g, int64_t E, cudaStream_t stream) {
  DeviceInfo* dev = nullptr;
  if (const int rc = device_info(&dev)) return rc;
  const int64_t rows = TOKENS ? g.rows : (g.rows + 127) / 128 * 128, spans = (g.tiles + 1) / 2;
  g.spans = std::max<int>(spans_of(rows * E, spans, dev->sm_count), (int)((spans + 65534) / 65535));
  const bool vec = (reinterpret_cast<uintptr_t>(g.X) & 15u) == 0 && (g.ldx * sizeof(T)) % 16 == 0 &&
                   (E == 1 || (g.x_stride * sizeof(T)) % 16 == 0);
  PdlLaunch l(dim3((unsigned)((rows + WARPS - 1) / WARPS), (unsigned)((spans + g.spans - 1) / g.spans), (unsigned)E),
              dim3(THREADS), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(
      &l.cfg, vec ? quantize_f4_kernel<T, true, TOKENS> : quantize_f4_kernel<T, false, TOKENS>, (const QuantArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "quantize_f4 launch");
}

template <bool TOKENS>
int quantize_any(int dtype, const QuantArgs& g, int64_t E, cudaStream_t s) {
  return dtype == KEBAB_F16    ? quantize<__half, TOKENS>(g, E, s)
         : dtype == KEBAB_BF16 ? quantize<__nv_bfloat16, TOKENS>(g, E, s)
                               : quantize<float, TOKENS>(g, E, s);
}

template <typename T>
int dequantize(DequantArgs g, int64_t E, cudaStream_t stream) {
  DeviceInfo* dev = nullptr;
  if (const int rc = device_info(&dev)) return rc;
  const bool vec = (reinterpret_cast<uintptr_t>(g.W) & 15u) == 0 && g.K % 8 == 0;
  const int64_t spans = (g.K + (vec ? 0 : 7) + 255) / 256;  // a granule may begin before the row
  g.spans = std::max<int>(spans_of(g.rows * E, spans, dev->sm_count), (int)((spans + 65534) / 65535));
  PdlLaunch l(dim3((unsigned)((g.rows + WARPS - 1) / WARPS), (unsigned)((spans + g.spans - 1) / g.spans), (unsigned)E),
              dim3(THREADS), 0, stream);
  const cudaError_t e =
      cudaLaunchKernelEx(&l.cfg, vec ? dequantize_f4_kernel<T, false> : dequantize_f4_kernel<T, true>, (const DequantArgs)g);
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
    const QuantArgs g = {W, ldw, w_stride, codes, scales, N, (int)K, (int)((K + 127) / 128), 0, 0};
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
    const QuantArgs g = {X, ldx, 0, codes, scales, R, (int)K, (int)((K + 127) / 128), 0, R + F4_SLACK};
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
    const DequantArgs g = {codes, scales, W, N, (int)K, (int)((K + 127) / 128), 0};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == KEBAB_F16 ? dequantize<__half>(g, E, s) : dtype == KEBAB_BF16 ? dequantize<__nv_bfloat16>(g, E, s) : dequantize<float>(g, E, s);
  });
}

}  // extern "C"
