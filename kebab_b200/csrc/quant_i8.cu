// Quantisation of rows to 8-bit integers with one scale a row.
//
// One block a row: the row is read once, 16 bytes a thread and step, and kept
// in registers while the block finds its largest magnitude (as the largest
// bit pattern of |x|, so that a NaN stands above everything and is not lost);
// the codes are then made from the registers. Rows longer than the registers
// hold are read a second time, from L2. Bound by memory: 2 bytes read and 1
// written for each 16-bit value.
//
// The code is x * (127 / amax), one multiplication by a once-rounded quotient:
// a division of every value would cost about ten instructions each, and the
// two roundings differ only where x / scale lies within 2^-22 of a tie.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grouped.h"
#include "kebab/int8.h"
#include "quant_i8.cuh"

namespace kb {
namespace {
constexpr int THREADS = 256;

// VEC: 8 values a step in 16-byte (F32: 2 x 16-byte) loads and 8-byte stores;
// otherwise one value a step. HELD steps are kept in registers.
template <typename T, bool VEC, int HELD>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                                                           int cols) {
  constexpr int W = VEC ? 8 : 1;
  __shared__ uint32_t part[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const T* x = X + (int64_t)blockIdx.x * ldx;
  int8_t* out = q + (int64_t)blockIdx.x * ldq;
  float v[HELD][W];
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = (h * THREADS + threadIdx.x) * W;
    if (c < cols) {
      load_row<W>(x + c, v[h]);
#pragma unroll
      for (int u = 0; u < W; ++u) top = max(top, abs_bits(v[h][u]));
    }
  }
  for (int c = (HELD * THREADS + threadIdx.x) * W; c < cols; c += THREADS * W) {
    float y[W];
    load_row<W>(x + c, y);
#pragma unroll
    for (int u = 0; u < W; ++u) top = max(top, abs_bits(y[u]));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = max(top, part[w]);
  const RowScale s = row_scale(top);
  if (threadIdx.x == 0) scale[blockIdx.x] = s.scale;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = (h * THREADS + threadIdx.x) * W;
    if (c < cols) store_codes<W>(out + c, v[h], s.inv);
  }
  for (int c = (HELD * THREADS + threadIdx.x) * W; c < cols; c += THREADS * W) {
    float y[W];
    load_row<W>(x + c, y);
    store_codes<W>(out + c, y, s.inv);
  }
}

template <typename T, bool VEC>
int launch(const void* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols,
           cudaStream_t stream) {
  constexpr int STEP = THREADS * (VEC ? 8 : 1);
  auto kern = quantize_kernel<T, VEC, VEC ? 4 : 8>;
  if (cols <= STEP) kern = quantize_kernel<T, VEC, 1>;
  else if (cols <= 2 * STEP) kern = quantize_kernel<T, VEC, 2>;
  PdlLaunch l(dim3((unsigned)rows), dim3(THREADS), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, static_cast<const T*>(X), ldx, q, ldq, scale, (int)cols);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "quantize_i8 launch");
}

template <typename T>
int launch_type(const void* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols,
                cudaStream_t stream) {
  const bool vec = (reinterpret_cast<uintptr_t>(X) & 15u) == 0 && (ldx * sizeof(T)) % 16 == 0 && cols % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0;
  return vec ? launch<T, true>(X, ldx, q, ldq, scale, rows, cols, stream)
             : launch<T, false>(X, ldx, q, ldq, scale, rows, cols, stream);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" int kebab_quantize_i8(kebab_dtype dtype, const void* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                                 int64_t rows, int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > (1 << 30))
      return fail(KEBAB_EINVAL, "quantize_i8: invalid dimensions rows=" + std::to_string(rows) +
                                    " cols=" + std::to_string(cols));
    if (ldx < cols || ldq < cols) return fail(KEBAB_EINVAL, "quantize_i8: a row pitch is below the row length");
    if (rows == 0) return KEBAB_OK;
    if (!X || !q || !scale) return fail(KEBAB_EINVAL, "quantize_i8: null pointer");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == KEBAB_F16) return launch_type<__half>(X, ldx, q, ldq, scale, rows, cols, s);
    if (dtype == KEBAB_BF16) return launch_type<__nv_bfloat16>(X, ldx, q, ldq, scale, rows, cols, s);
    if (dtype == KEBAB_F32) return launch_type<float>(X, ldx, q, ldq, scale, rows, cols, s);
    return fail(KEBAB_ENOTSUP, "quantize_i8: only F16, BF16 and F32 are implemented");
  });
}
