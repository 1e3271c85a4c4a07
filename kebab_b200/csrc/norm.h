// Internal declarations of the norm's kernels.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace kb {

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* r;  // residual, or null
  int64_t ldr;
  const void* w;
  int w_f32;  // weight in FP32, else in the rows' type
  float eps;
  void* s;
  int64_t lds;
  void* y;
  int64_t ldy;
  int8_t* q;
  int64_t ldq;
  float* scale;
  int64_t rows;
  int cols;
};

struct GradArgs {
  const void* dy;
  int64_t lddy;
  const void* s;
  int64_t lds;
  const void* w;
  int w_f32;
  float eps;
  const void* ds;  // or null
  int64_t ldds;
  void* dx;  // or null
  int64_t lddx;
  float* partial;  // [blocks][cols] sums of dweight, or null
  float* stats;    // [rows][2]: rstd, mean(g s), where there is more than one slab
  int64_t rows;
  int cols;
};

constexpr int kNormMaxBlocks = 1024;  // of the backward kernel, as the workspace is sized

// Where the rows of a call's tensors start: all on 16 bytes (of a length that is
// a multiple of 8), each row of all at the same place of 16 bytes, or anywhere.
enum class RowStart { kAligned, kAlike, kAny };

// For rows of one type; `blocks`: how many partial sums of dweight there are.
#define KEBAB_NORM_TYPE(name)                                                                  \
  int norm_forward_##name(const NormArgs& g, RowStart start, bool i8, int sms, cudaStream_t s); \
  int norm_backward_##name(const GradArgs& g, RowStart start, int sms, int* blocks, cudaStream_t s)
KEBAB_NORM_TYPE(f16);
KEBAB_NORM_TYPE(bf16);
KEBAB_NORM_TYPE(f32);
#undef KEBAB_NORM_TYPE

}  // namespace kb
