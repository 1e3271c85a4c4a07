// The norm's kernels for rows of F32.
#include "norm.cuh"

namespace kb {

int norm_forward_f32(const NormArgs& g, RowStart start, bool i8, int sms, cudaStream_t s) {
  return run_forward<float>(g, start, i8, sms, s);
}
int norm_backward_f32(const GradArgs& g, RowStart start, int sms, int* blocks, cudaStream_t s) {
  return run_backward<float>(g, start, sms, blocks, s);
}

}  // namespace kb
