/*
 * Root-mean-square norm of tokens, with the residual's addition before it, an
 * output in 8-bit integers, and the gradients:
 *
 *   s[t, h] = round(x[t, h] + residual[t, h])         (s = x without a residual)
 *   rstd[t] = (mean_h s[t, h]^2 + eps)^(-1/2)
 *   y[t, h] = s[t, h] * rstd[t] * weight[h]
 *
 * The norm is of the sum as it is stored, so that the backward pass, which
 * reads s, differentiates what the forward pass computed. Everything between
 * the loads and the stores is in FP32.
 *
 * Plain C, device pointers, asynchronous on `stream`, status codes and
 * kebab_last_error() as in kebab.h. Rows are contiguous; `ld*` are row pitches
 * in elements. `dtype` (F16, BF16 or F32) is the type of x, residual, s, y and
 * their gradients; `weight_dtype`, of weight and dweight, is that type or F32.
 * No counterpart in kebab.
 */
#ifndef KEBAB_NORM_H_
#define KEBAB_NORM_H_

#include "kebab/kebab.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y and s from x. Without a residual (NULL) s is not written and may be NULL.
 * s may be x or residual themselves. rows = 0 is a no-op. */
int kebab_rms_norm(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                   int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                   int64_t rows, int64_t cols, kebab_stream_t stream);

/* The same with y quantised by row as kebab_quantize_i8 does (kebab/int8.h),
 * from the FP32 values: codes q and scales, operands of kebab_gemm_i8 (zeros, with
 * scale 0, for a row whose largest |s * weight| is under 1e-30). y, in
 * `dtype`, is written too unless it is NULL. */
int kebab_rms_norm_i8(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                      int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                      int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, kebab_stream_t stream);

/* Gradients, with g = dy * weight:
 *   dx[t, h] = ds[t, h] + rstd[t] (g[t, h] - s[t, h] rstd[t]^2 mean_h(g s)[t])
 *   dweight[h] = sum_t dy[t, h] s[t, h] rstd[t]
 * dx is the gradient of x and of the residual; ds (NULL: none) is what reaches
 * s past the norm. dx and dweight may be NULL. The sums have a fixed order: the
 * same call gives the same bits on devices with as many SMs (another boundary of
 * the rows, or dx left out, may choose another order).
 * `workspace` (16-byte aligned) holds
 * kebab_rms_norm_backward_workspace(rows, cols) bytes. rows = 0 gives a
 * dweight of zeros. */
int64_t kebab_rms_norm_backward_workspace(int64_t rows, int64_t cols);
int kebab_rms_norm_backward(kebab_dtype dtype, kebab_dtype weight_dtype, const void* dy, int64_t lddy, const void* s,
                            int64_t lds, const void* weight, float eps, const void* ds, int64_t ldds, void* dx,
                            int64_t lddx, void* dweight, void* workspace, int64_t workspace_bytes, int64_t rows,
                            int64_t cols, kebab_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KEBAB_NORM_H_ */
