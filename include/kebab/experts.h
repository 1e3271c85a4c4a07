/*
 * Operators of a mixture-of-experts layer: routing, the exchange of rows
 * between token order and expert order, and the products grouped by expert,
 * each with its gradient.
 *
 * Plain C, device pointers, asynchronous on `stream`, status codes and
 * kebab_last_error() as in kebab.h. Rows are contiguous; `ld*` are row pitches
 * in elements; all matrices are row-major (tokens are rows). 1 <= E <= 1024
 * experts, 1 <= k <= min(E, 32) choices a token, T * k < 2^31. Zero rows or
 * tokens are valid. No counterpart in kebab.
 *
 * Device-side integers are not trusted: offsets are clamped to [0, R], and a
 * slot outside [0, R) (a negative one marks a dropped choice) or an expert
 * outside [0, E) contributes nothing.
 */
#ifndef KEBAB_EXPERTS_H_
#define KEBAB_EXPERTS_H_

#include "kebab/kebab.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Top-k routing of T tokens over E experts (logits T x E; F16, BF16 or F32).
 *   experts[t, j]  the j-th largest logit's expert (equal logits: the lower
 *                  expert first; NaN orders above +inf)
 *   weights[t, j]  softmax of the logits over the k chosen experts
 *                  (renormalize != 0) or over all E
 *   offsets[e]     number of choices of experts below e (E + 1 values)
 *   slots[t, j]    place of the choice (t, j) when all T * k choices are sorted
 *                  by expert, in the order of t within one expert
 * A row of logits that are all -inf gets weights 0; NaN or +inf in a row makes
 * its weights NaN. `workspace`: kebab_route_workspace(T, E) bytes, 4-byte
 * aligned. */
int64_t kebab_route_workspace(int64_t T, int64_t E);
int kebab_route(kebab_dtype dtype, const void* logits, int64_t ld, int64_t T, int64_t E, int k, int renormalize,
                float* weights, int32_t* experts, int32_t* offsets, int32_t* slots, void* workspace,
                int64_t workspace_bytes, kebab_stream_t stream);

/* dlogits (T x E, type of logits) from the gradient of the weights. */
int kebab_route_backward(kebab_dtype dtype, const void* logits, int64_t ld, int64_t T, int64_t E, int k,
                         int renormalize, const float* weights, const int32_t* experts, const float* dweights,
                         void* dlogits, int64_t ldd, kebab_stream_t stream);

/* xs[slots[t, j]] = x[t]: tokens (T x H) to expert order (R x H). F16 / BF16.
 * Its gradient is kebab_expert_combine with weights NULL. */
int kebab_expert_dispatch(kebab_dtype dtype, const void* x, int64_t ldx, const int32_t* slots, void* xs, int64_t ldxs,
                          int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream);

/* y[t] = sum_j weights[t, j] ys[slots[t, j]] (weights NULL: 1), summed in
 * order of j in FP32 and rounded once. */
int kebab_expert_combine(kebab_dtype dtype, const void* ys, int64_t ldys, const int32_t* slots, const float* weights,
                         void* y, int64_t ldy, int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream);

/* dys[slots[t, j]] = weights[t, j] dy[t]; dweights[t, j] = <dy[t], ys[slots[t, j]]>. */
int kebab_expert_combine_backward(kebab_dtype dtype, const void* dy, int64_t lddy, const void* ys, int64_t ldys,
                                  const int32_t* slots, const float* weights, void* dys, int64_t lddys,
                                  float* dweights, int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream);

/* Y[r] = X[r] W_e for the rows offsets[e] <= r < offsets[e + 1] of each expert
 * e (X: R x K, Y: R x N, F16 or BF16, FP32 accumulation). opmode "RC": W_e is
 * stored column-major, N rows of K; "RR": row-major, K rows of N; W_e starts
 * at W + e * w_stride. The offsets stay on the device: no copy to the host.
 * Rows of no expert are not written. dX is the same call on dY with the other
 * opmode (and N, K exchanged). */
int kebab_gemm_grouped(kebab_dtype dtype, const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_stride,
                       void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K,
                       const char* opmode, kebab_stream_t stream);

/* dW_e = the gradient of W_e: the sum over the expert's rows of dY[r, n] X[r, k],
 * stored as W is ("RC": N x K, "RR": K x N; contiguous, one after another).
 * An expert without rows gets zeros. */
int kebab_gemm_grouped_dw(kebab_dtype dtype, const void* X, int64_t ldx, const void* dY, int64_t lddy, void* dW,
                          const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K, const char* opmode,
                          kebab_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* KEBAB_EXPERTS_H_ */
