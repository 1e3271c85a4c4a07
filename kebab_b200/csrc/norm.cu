// C entry points of the root-mean-square norm (include/kebab/norm.h): argument
// checks, where rows start, and the sum of dweight's parts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "grouped.h"
#include "kebab/norm.h"
#include "norm.h"
#include "vec.cuh"

namespace kb {
namespace {

// dweight[c] = the sum of the blocks' partial sums in a fixed order: 32 warps
// take every 32nd of them, 32 columns a block.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_dweight_kernel(const float* partial, int blocks, int cols, TW* dweight) {
  __shared__ float sums[32][33];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 32) sum += partial[(int64_t)b * cols + c];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  sum = sums[lane][warp];  // column `warp`, the sum of warp `lane`
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0 && blockIdx.x * 32 + warp < cols) dweight[blockIdx.x * 32 + warp] = from_float<TW>(sum);
}

int check_norm(const char* what, int dtype, int weight_dtype, int64_t rows, int64_t cols, float eps) {
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16 && dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16, BF16 and F32 are implemented");
  if (weight_dtype != dtype && weight_dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": the weight is of the rows' type or F32");
  if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > (1 << 30))
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions rows=" + std::to_string(rows) +
                                  " cols=" + std::to_string(cols));
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(KEBAB_EINVAL, std::string(what) + ": eps must be finite and not negative");
  return KEBAB_OK;
}

int check_ld(const char* what, const char* name, int64_t ld, int64_t cols) {
  if (ld >= cols) return KEBAB_OK;
  return fail(KEBAB_EINVAL, std::string(what) + ": row pitch of " + name + " (" + std::to_string(ld) +
                                ") is below the row length (" + std::to_string(cols) + ")");
}

// Whether rows from `p` on at a pitch of `ld` start on boundaries of `bytes`.
bool aligned(const void* p, int64_t ld, int es, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && ld * es % bytes == 0;
}

// Whether every row starts at the same place of 16 bytes in both.
bool alike(const void* a, int64_t lda, const void* b, int64_t ldb, int es) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15u) == 0 && (lda - ldb) * es % 16 == 0;
}

int size_of(int dtype) { return dtype == KEBAB_F32 ? 4 : 2; }

int forward(const char* what, int dtype, int weight_dtype, NormArgs g, bool i8, kebab_stream_t stream) {
  int rc;
  if ((rc = check_norm(what, dtype, weight_dtype, g.rows, g.cols, g.eps)) || (rc = check_ld(what, "x", g.ldx, g.cols)))
    return rc;
  if (g.r && ((rc = check_ld(what, "residual", g.ldr, g.cols)) || (rc = check_ld(what, "s", g.lds, g.cols)))) return rc;
  if ((g.y || !i8) && (rc = check_ld(what, "y", g.ldy, g.cols))) return rc;
  if (i8 && (rc = check_ld(what, "q", g.ldq, g.cols))) return rc;
  if (g.rows == 0) return KEBAB_OK;
  if (!g.x || !g.w || (g.r && !g.s) || (i8 ? !g.q || !g.scale : !g.y))
    return fail(KEBAB_EINVAL, std::string(what) + ": null pointer");
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  g.w_f32 = weight_dtype == KEBAB_F32;
  const int es = size_of(dtype);
  RowStart start = RowStart::kAny;
  if (g.cols % 8 == 0 && aligned(g.x, g.ldx, es, 16) && aligned(g.w, 0, 1, 16) &&
      (!g.r || (aligned(g.r, g.ldr, es, 16) && aligned(g.s, g.lds, es, 16))) &&
      (!g.y || aligned(g.y, g.ldy, es, 16)) && (!i8 || aligned(g.q, g.ldq, 1, 8)))
    start = RowStart::kAligned;
  else if ((!g.r || (alike(g.x, g.ldx, g.r, g.ldr, es) && alike(g.x, g.ldx, g.s, g.lds, es))) &&
           (!g.y || alike(g.x, g.ldx, g.y, g.ldy, es)))
    start = RowStart::kAlike;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto run = dtype == KEBAB_F16 ? norm_forward_f16 : dtype == KEBAB_BF16 ? norm_forward_bf16 : norm_forward_f32;
  return run(g, start, i8, dev->sm_count, st);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int kebab_rms_norm(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                   int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                   int64_t rows, int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    if (cols > (1 << 30)) return check_norm("rms_norm", dtype, weight_dtype, rows, cols, eps);
    NormArgs g = {};
    g.x = x, g.ldx = ldx, g.r = residual, g.ldr = ldr, g.w = weight, g.eps = eps, g.s = s, g.lds = lds;
    g.y = y, g.ldy = ldy, g.rows = rows, g.cols = (int)cols;
    return forward("rms_norm", dtype, weight_dtype, g, false, stream);
  });
}

int kebab_rms_norm_i8(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                      int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                      int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    if (cols > (1 << 30)) return check_norm("rms_norm_i8", dtype, weight_dtype, rows, cols, eps);
    NormArgs g = {};
    g.x = x, g.ldx = ldx, g.r = residual, g.ldr = ldr, g.w = weight, g.eps = eps, g.s = s, g.lds = lds;
    g.y = y, g.ldy = ldy, g.q = q, g.ldq = ldq, g.scale = scale, g.rows = rows, g.cols = (int)cols;
    return forward("rms_norm_i8", dtype, weight_dtype, g, true, stream);
  });
}

// The rows' two sums, then the blocks' sums of dweight.
int64_t kebab_rms_norm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > (1 << 30)) return -KEBAB_EINVAL;
  return (rows * 8 + 15) / 16 * 16 + std::min<int64_t>((rows + 7) / 8 * 8, kNormMaxBlocks) * cols * 4;
}

int kebab_rms_norm_backward(kebab_dtype dtype, kebab_dtype weight_dtype, const void* dy, int64_t lddy, const void* s,
                            int64_t lds, const void* weight, float eps, const void* ds, int64_t ldds, void* dx,
                            int64_t lddx, void* dweight, void* workspace, int64_t workspace_bytes, int64_t rows,
                            int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "rms_norm_backward";
    int rc;
    if ((rc = check_norm(what, dtype, weight_dtype, rows, cols, eps)) || (rc = check_ld(what, "dy", lddy, cols)) ||
        (rc = check_ld(what, "s", lds, cols)) || (ds && (rc = check_ld(what, "ds", ldds, cols))) ||
        (dx && (rc = check_ld(what, "dx", lddx, cols))))
      return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows == 0) {
      if (!dweight) return KEBAB_OK;
      const cudaError_t e = cudaMemsetAsync(dweight, 0, cols * size_of(weight_dtype), st);
      return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward memset");
    }
    if (!dy || !s || !weight) return fail(KEBAB_EINVAL, "rms_norm_backward: null pointer");
    if (!dx && !dweight) return KEBAB_OK;
    if (!workspace || workspace_bytes < kebab_rms_norm_backward_workspace(rows, cols) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u))
      return fail(KEBAB_EINVAL, "rms_norm_backward: the workspace is null, too small or not 16-byte aligned");
    DeviceInfo* dev = nullptr;
    if ((rc = device_info(&dev))) return rc;
    GradArgs g = {};
    g.dy = dy, g.lddy = lddy, g.s = s, g.lds = lds, g.w = weight, g.w_f32 = weight_dtype == KEBAB_F32, g.eps = eps;
    g.ds = ds, g.ldds = ldds, g.dx = dx, g.lddx = lddx, g.rows = rows, g.cols = (int)cols;
    g.stats = static_cast<float*>(workspace);
    float* partial = g.stats + (rows * 8 + 15) / 16 * 4;
    g.partial = dweight ? partial : nullptr;
    const int es = size_of(dtype);
    RowStart start = RowStart::kAny;
    if (cols % 8 == 0 && aligned(dy, lddy, es, 16) && aligned(s, lds, es, 16) && aligned(weight, 0, 1, 16) &&
        (!ds || aligned(ds, ldds, es, 16)) && (!dx || aligned(dx, lddx, es, 16)))
      start = RowStart::kAligned;
    else if (alike(s, lds, dy, lddy, es) && (!ds || alike(s, lds, ds, ldds, es)) && (!dx || alike(s, lds, dx, lddx, es)))
      start = RowStart::kAlike;
    int blocks = 0;
    auto run = dtype == KEBAB_F16 ? norm_backward_f16 : dtype == KEBAB_BF16 ? norm_backward_bf16 : norm_backward_f32;
    rc = run(g, start, dev->sm_count, &blocks, st);
    if (rc || !dweight) return rc;
    PdlLaunch l(dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, st);
    cudaError_t e;
    if (weight_dtype == KEBAB_F16) e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<__half>, (const float*)partial, blocks, (int)cols, static_cast<__half*>(dweight));
    else if (weight_dtype == KEBAB_BF16) e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<__nv_bfloat16>, (const float*)partial, blocks, (int)cols, static_cast<__nv_bfloat16*>(dweight));
    else e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<float>, (const float*)partial, blocks, (int)cols, static_cast<float*>(dweight));
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward: dweight launch");
  });
}

}  // extern "C"
