/*
 * Microscaled 4-bit floating point: values +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} (one
 * sign, two exponent, one mantissa bit), 32 consecutive ones of a row to a
 * power-of-two scale (a byte b stands for 2^(b - 127), 255 for NaN):
 *
 *   e = the least exponent >= -127 with amax <= 6 * 2^e   (amax of the 32)
 *   code[i] = the nearest value to x[i] / 2^e, ties to the even code
 *   Y[m, n] = sum_k X[m, k] W[n, k]  (+ bias[n])  of the values of the codes
 *
 * No value is clipped, the quantisation is exact arithmetic but for the
 * rounding to a code, and products of codes and scales are exact; they are
 * summed in FP32 and rounded once to the output type. A block with an infinity
 * or a NaN gets the scale NaN, which the outputs of its row then are.
 *
 * Storage. Codes: rows of ceil(K / 32) * 16 bytes, the lower nibble first; a
 * last block that K does not fill holds zeros. Scales of weights: tiles of 128
 * rows and 128 values, each 512 bytes, [ceil(N / 128)][ceil(K / 128)][512]; the
 * scale of row n and block b stands in byte (n % 32) * 16 + n % 128 / 32 * 4 +
 * b % 4 of its tile (what the tensor cores read); places of no row or block are
 * 0. Scales of tokens: [ceil(K / 128)][R + 160] entries of 16 bytes; entry r
 * holds the four scales (of the 128 values) of rows r, r + 32, r + 64 and
 * r + 96, so that a tile may begin at any row; places of no row are not written.
 *
 * Plain C, device pointers, asynchronous on `stream`, status codes and
 * kebab_last_error() as in kebab.h. Codes and scales are 16-byte aligned; `ld*`
 * are row pitches in elements. Y is row-major, [M, N]. At most 2^27 token rows,
 * 1024 matrices, 2^30 values a row. No counterpart in kebab.
 */
#ifndef KEBAB_F4_H_
#define KEBAB_F4_H_

#include "kebab/kebab.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of the codes and scales of N weight rows, or R token rows, of K values. */
int64_t kebab_f4_code_bytes(int64_t rows, int64_t K);
int64_t kebab_f4_weight_scale_bytes(int64_t N, int64_t K);
int64_t kebab_f4_token_scale_bytes(int64_t R, int64_t K);

/* Quantises the rows of E weight matrices (N x K, F16, BF16 or F32, w_stride
 * elements apart; E = 1: any). The matrices' codes and scales follow one
 * another. */
int kebab_quantize_f4(kebab_dtype dtype, const void* W, int64_t ldw, int64_t w_stride, uint8_t* codes, uint8_t* scales,
                      int64_t E, int64_t N, int64_t K, kebab_stream_t stream);

/* Quantises the rows of X (R x K). R = 0 is a no-op. */
int kebab_quantize_f4_tokens(kebab_dtype dtype, const void* X, int64_t ldx, uint8_t* codes, uint8_t* scales, int64_t R,
                             int64_t K, kebab_stream_t stream);

/* The values of quantised weights, rounded to `dtype`, contiguous [E, N, K]. */
int kebab_dequantize_f4(kebab_dtype dtype, const uint8_t* codes, const uint8_t* scales, void* W, int64_t E, int64_t N,
                        int64_t K, kebab_stream_t stream);

/* Y (M x N, F16 or BF16) from quantised tokens and weights. `bias` (N values of
 * the output type) may be NULL. M = 0 is a no-op. */
int kebab_gemm_f4(kebab_dtype out, const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                  const uint8_t* w_scales, const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                  kebab_stream_t stream);

/* The same grouped by expert: rows offsets[e] .. offsets[e + 1] - 1 of X take
 * the e-th of E weight matrices. See kebab_gemm_grouped (kebab/experts.h). */
int kebab_gemm_grouped_f4(kebab_dtype out, const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                          const uint8_t* w_scales, void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t R,
                          int64_t N, int64_t K, kebab_stream_t stream);

/* Quantises X (M x K, F16 or BF16) and multiplies, Y of X's type. offsets NULL
 * (then E = 1): one weight matrix, bias optional; else grouped by expert, no
 * bias. Y may lie on X. `workspace` (16-byte aligned) holds the codes and scales
 * of X: kebab_linear_f4_workspace(M, K) bytes. */
int64_t kebab_linear_f4_workspace(int64_t M, int64_t K);
int kebab_linear_f4(kebab_dtype dtype, const void* X, int64_t ldx, const uint8_t* w_codes, const uint8_t* w_scales,
                    const void* bias, void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t M, int64_t N,
                    int64_t K, void* workspace, int64_t workspace_bytes, kebab_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KEBAB_F4_H_ */
