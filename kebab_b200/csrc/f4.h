// Internal declarations of the 4-bit floating-point products.
#pragma once
#include "grouped.h"

namespace kb {

// Y[r, n] = sum_k X[r, k] W_e(n, k) for the rows r of group e, of quantised
// operands stored as include/kebab/f4.h says.
struct F4Problem {
  int out;  // KEBAB_F16 or KEBAB_BF16
  const uint8_t* x_codes;
  const uint8_t* x_scales;
  const uint8_t* w_codes;
  const uint8_t* w_scales;
  const void* bias;  // output type, per n, or null
  void* Y;
  int64_t ldy;
  const int32_t* offsets;  // E + 1 device integers; null: one group of all R rows
  int64_t E, R, N, K;
  bool early;  // the kernel before on the stream makes only the codes and scales of X
  cudaStream_t stream;
  const void* x = nullptr;  // rows of the output type that the product quantises itself (launch_f4_skinny), instead of codes
  int64_t ldx = 0;
};

constexpr int64_t F4_MAX_ROWS = int64_t(1) << 27;  // of tokens
// Rows that a product quantises itself, at most: every CTA does it for its k
// range, and saves the launch before (8192 x 8192, back to back: 1 row 7.4 us
// against 9.0, 4 rows 7.6 against 8.9, 8 rows 9.9 against 8.5; 2048 x 2048 3.9
// against 5.6, 4.0 against 5.7, 4.8 against 5.7; weights from memory: 6 rows 12.1
// and 14.1 a call, 7 rows, in two launches, 11.6 and 16.9).
constexpr int F4_FUSED_ROWS = 6;
constexpr int F4_SLACK = 160;  // entries of token scales past the last row

__host__ __device__ inline int64_t f4_pitch(int64_t K) { return (K + 31) / 32 * 16; }  // bytes of a row's codes

// Tensor maps of the operands. Codes: bytes, boxes of 128 bytes of 128 weight
// rows, or of `rows` token rows. Scales: as pairs of bytes, boxes of two runs of
// 128 values, each 512 bytes, for 128 rows.
int f4_weight_map(const F4Problem& p, CUtensorMap* m);         // {byte, n, e}
int f4_weight_scale_map(const F4Problem& p, CUtensorMap* m);  // {0, run of values, run of rows of all matrices}
int f4_token_map(const F4Problem& p, int rows, CUtensorMap* m);          // {byte, token}
int f4_token_scale_map(const F4Problem& p, CUtensorMap* m);              // {8 * token, run of values}

int launch_f4_umma(const F4Problem& p);
int launch_f4_skinny(const F4Problem& p);

}  // namespace kb
