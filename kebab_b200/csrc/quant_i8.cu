// Quantisation of rows to 8-bit integers with one scale a row.
//
// One block a row, or (rows of up to 2048) one warp: the row is read once, 16
// bytes a thread and step, and kept in registers as it is stored while they find
// its largest magnitude (as the largest bit pattern of |x|, so that a NaN stands
// above everything and is not lost); the codes are then made from the registers.
// Rows longer than the registers hold are read a second time, from L2. Bound by
// memory: 2 bytes read and 1 written for each 16-bit value; 4093 x 8192 BF16
// 17.5 us, 5.7 TB/s (26.6 with conversion instructions and 8 warps a row), 30000
// x 520 13 us (31 with a block a row).
//
// The code is x * (127 / amax), one multiplication by a once-rounded quotient:
// a division of every value would cost about ten instructions each, and the
// two roundings differ only where x / scale lies within 2^-22 of its own size of
// a tie (2^-15 for codes near 127).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "grouped.h"
#include "kebab/int8.h"
#include "quant_i8.cuh"

namespace kb {
namespace {
constexpr int THREADS = 128;

// VEC: 8 values a step in 16-byte (F32: 2 x 16-byte) loads and 8-byte stores;
// otherwise one value a step. ROW threads take a row (a warp or the block) and
// keep HELD steps in registers.
template <typename T, bool VEC, int HELD, int ROW>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const T* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                                                           int64_t rows, int cols) {
  constexpr int W = VEC ? 8 : 1;
  __shared__ uint32_t part[THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * (THREADS / ROW) + threadIdx.x / ROW;
  if (row >= rows) return;
  const T* x = X + row * ldx;
  int8_t* out = q + row * ldq;
  const int c0 = threadIdx.x % ROW * W;
  Run<T, W> held[HELD];
  uint32_t top = 0;
  float v[W];
#pragma unroll
  for (int h = 0; h < HELD; ++h)
    if (c0 + h * ROW * W < cols) held[h].load(x + c0 + h * ROW * W);
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    if (c0 + h * ROW * W < cols) {
      held[h].values(v);
      top = largest<W>(v, top);
    }
  }
  for (int c = c0 + HELD * ROW * W; c < cols; c += ROW * W) {
    load_row<W>(x + c, v);
    top = largest<W>(v, top);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (ROW > 32) {
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = max(top, part[w]);
  }
  const RowScale s = row_scale(top);
  if (threadIdx.x % ROW == 0) scale[row] = s.scale;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    if (c0 + h * ROW * W < cols) {
      held[h].values(v);
      store_codes<W>(out + c0 + h * ROW * W, v, s.inv);
    }
  }
  for (int c = c0 + HELD * ROW * W; c < cols; c += ROW * W) {
    load_row<W>(x + c, v);
    store_codes<W>(out + c, v, s.inv);
  }
}

template <typename T, bool VEC>
int launch(const void* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols,
           cudaStream_t stream) {
  constexpr int W = VEC ? 8 : 1;
  // A warp a row while there are rows for a warp or two a scheduler.
  const bool warp = cols <= 32 * 8 * W && rows >= 1024;
  const int64_t step = (warp ? 32 : THREADS) * W;
  auto kern = quantize_kernel<T, VEC, 8, THREADS>;
  if (cols <= step) kern = warp ? quantize_kernel<T, VEC, 1, 32> : quantize_kernel<T, VEC, 1, THREADS>;
  else if (cols <= 2 * step) kern = warp ? quantize_kernel<T, VEC, 2, 32> : quantize_kernel<T, VEC, 2, THREADS>;
  else if (cols <= 4 * step) kern = warp ? quantize_kernel<T, VEC, 4, 32> : quantize_kernel<T, VEC, 4, THREADS>;
  else if (warp) kern = quantize_kernel<T, VEC, 8, 32>;
  const int64_t per_block = warp ? THREADS / 32 : 1;
  PdlLaunch l(dim3((unsigned)((rows + per_block - 1) / per_block)), dim3(THREADS), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, static_cast<const T*>(X), ldx, q, ldq, scale, rows, (int)cols);
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
