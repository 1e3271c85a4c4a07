/*
 * Products in 8-bit integers with one scale a row of activations (token) and
 * one a row of weights (output channel):
 *
 *   q[m, k] = rint(X[m, k] * (127 / amax_m)),  scale[m] = amax_m / 127,
 *   Y[m, n] = scale[m] * w_scale[n] * sum_k q[m, k] * Wq[n, k]  (+ bias[n]),
 *
 * with amax_m the largest magnitude of row m, ties of rint to even, the sum
 * in 32-bit integers and one rounding to the output type. The sum is exact:
 * given codes are any int8 (-128 too), with K <= 131071; the codes made here
 * are -127 .. 127, and kebab_linear_i8 takes K <= 131072.
 *
 * Plain C, device pointers, asynchronous on `stream`, status codes and
 * kebab_last_error() as in kebab.h. Rows are contiguous; `ld*` are row pitches
 * in elements. Y is row-major here (Y[m, n] at Y + m * ldy + n): tokens are
 * rows. No counterpart in kebab.
 */
#ifndef KEBAB_INT8_H_
#define KEBAB_INT8_H_

#include "kebab/kebab.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Quantises each row of X (rows x cols, F16, BF16 or F32). A row whose largest
 * magnitude is under 1e-30 becomes zeros with scale 0 (127 / amax would
 * overflow). A row with an infinity or a NaN gets a scale that is infinite or
 * NaN and codes of 0, so products with it are NaN. rows = 0 is a no-op. */
int kebab_quantize_i8(kebab_dtype dtype, const void* X, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                      int64_t rows, int64_t cols, kebab_stream_t stream);

/* Y (M x N, F16 or BF16) from quantised operands. `bias` (N values of the
 * output type) may be NULL. M = 0 is a no-op. */
int kebab_gemm_i8(kebab_dtype out, const int8_t* q, int64_t ldq, const float* scale, const int8_t* Wq, int64_t ldw,
                  const float* w_scale, const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                  kebab_stream_t stream);

/* The same grouped by expert: rows offsets[e] .. offsets[e + 1] - 1 of q take
 * Wq + e * w_stride (N x K) and w_scale + e * N. See kebab_gemm_grouped. */
int kebab_gemm_grouped_i8(kebab_dtype out, const int8_t* q, int64_t ldq, const float* scale, const int8_t* Wq,
                          int64_t ldw, int64_t w_stride, const float* w_scale, void* Y, int64_t ldy,
                          const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K, kebab_stream_t stream);

/* Quantises X (M x K, F16 or BF16) and multiplies, Y of X's type. offsets NULL
 * (then E = 1): one weight matrix, bias optional; else grouped by expert, no
 * bias. `workspace` (16-byte aligned) holds the codes and scales of X:
 * kebab_linear_i8_workspace(M, K) bytes. */
int64_t kebab_linear_i8_workspace(int64_t M, int64_t K);
int kebab_linear_i8(kebab_dtype dtype, const void* X, int64_t ldx, const int8_t* Wq, int64_t ldw, int64_t w_stride,
                    const float* w_scale, const void* bias, void* Y, int64_t ldy, const int32_t* offsets, int64_t E,
                    int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, kebab_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KEBAB_INT8_H_ */
