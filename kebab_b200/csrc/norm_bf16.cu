// The norm's kernels for rows of BF16.
#include "norm.cuh"

namespace kb {

int norm_forward_bf16(const NormArgs& g, RowStart start, bool i8, int sms, cudaStream_t s) {
  return run_forward<__nv_bfloat16>(g, start, i8, sms, s);
}
int norm_backward_bf16(const GradArgs& g, RowStart start, int sms, int* blocks, cudaStream_t s) {
  return run_backward<__nv_bfloat16>(g, start, sms, blocks, s);
}

}  // namespace kb
