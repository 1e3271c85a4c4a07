// The norm's kernels for rows of F16.
#include "norm.cuh"

namespace kb {

int norm_forward_f16(const NormArgs& g, RowStart start, bool i8, int sms, cudaStream_t s) {
  return run_forward<__half>(g, start, i8, sms, s);
}
int norm_backward_f16(const GradArgs& g, RowStart start, int sms, int* blocks, cudaStream_t s) {
  return run_backward<__half>(g, start, sms, blocks, s);
}

}  // namespace kb
