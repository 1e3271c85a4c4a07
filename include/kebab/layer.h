/*
 * A whole mixture-of-experts feed-forward layer for a few tokens (serving):
 *
 *   logits[t, e] = sum_h x[t, h] router[e, h]
 *   e[t, j], w[t, j] as kebab_route (kebab/experts.h) gives for these logits
 *   g, u = the first and the last D values of w_in[e] x[t]
 *   a[t, j, i] = g_i / (1 + exp(-g_i)) * u_i
 *   y[t, n] = sum_j w[t, j] sum_i w_out[e][n, i] a[t, j, i]
 *
 * for T <= KEBAB_FEW_TOKENS tokens of H values, E <= 1024 experts of D hidden
 * values and k <= 32 choices a token, H and D <= 2^20. Logits, a and every sum
 * are in FP32, with one rounding to the output type. Products with a take all of
 * its 24 bits (F16: 22, or 2^-38 of the largest a[t, j, i] of a choice).
 * The matrix units add up to 512 terms of a sum (their additions cut off bits),
 * the rest is added to nearest.
 *
 * With experts in 8-bit integers (the codes and row scales of
 * kebab_quantize_i8, kebab/int8.h) x[t] and every a[t, j] are quantised by row
 * to the nearest code, scale amax / 127, and the sums of products are exact in
 * 32-bit integers. (A row of x that lies on a tie takes the even code here;
 * kebab_quantize_i8 multiplies by a rounded 127 / amax first.)
 *
 * Plain C, device pointers, asynchronous on `stream`, status codes and
 * kebab_last_error() as in kebab.h. x and y are rows at a pitch; router [E, H]
 * (F32), w_in [E, 2 D, H] (gate rows, then up rows) and w_out [E, H, D] are
 * contiguous; weights whose rows do not start on 16 bytes are copied value by
 * value, which for large ones takes longer than the separate operators. An
 * expert that no token chooses is not read, and what an expert holds reaches the
 * tokens that choose it only. A call is two launches; all of
 * the second's blocks (one a multiprocessor) are on the device at once, so it
 * waits for room among kernels of other streams. T = 0 is a no-op. `workspace`
 * (16-byte aligned) holds kebab_expert_layer_workspace(T, E, k, H, D) bytes.
 * No counterpart in kebab.
 */
#ifndef KEBAB_LAYER_H_
#define KEBAB_LAYER_H_

#include "kebab/kebab.h"

#define KEBAB_FEW_TOKENS 16

#ifdef __cplusplus
extern "C" {
#endif

int64_t kebab_expert_layer_workspace(int64_t T, int64_t E, int k, int64_t H, int64_t D);

/* x, weights and y in `dtype`, F16 or BF16. */
int kebab_expert_layer(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const void* w_in,
                       const void* w_out, void* y, int64_t ldy, int64_t T, int64_t E, int k, int renormalize,
                       int64_t H, int64_t D, void* workspace, int64_t workspace_bytes, kebab_stream_t stream);

/* x and y in `dtype`, experts in 8-bit integers with in_scale [E, 2 D] and
 * out_scale [E, H]. H and D <= 131072. */
int kebab_expert_layer_i8(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const int8_t* w_in,
                          const float* in_scale, const int8_t* w_out, const float* out_scale, void* y, int64_t ldy,
                          int64_t T, int64_t E, int k, int renormalize, int64_t H, int64_t D, void* workspace,
                          int64_t workspace_bytes, kebab_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KEBAB_LAYER_H_ */
