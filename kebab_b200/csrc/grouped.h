// Internal declarations of the grouped and 8-bit integer products.
#pragma once
#include "internal.h"

namespace kb {

constexpr int kMaxExperts = 1024;
constexpr int IN_I8 = 100;  // GroupedProblem::in besides KEBAB_F16 / KEBAB_BF16

// Y[r, n] = sum_k X[r, k] W_e(k, n) for the rows r of group e, or (dw)
// dW_e(n, k) = sum_r dY[r, n] X[r, k].
struct GroupedProblem {
  int in, out;  // operand type (KEBAB_F16, KEBAB_BF16 or IN_I8), output type
  const void* X;
  int64_t ldx;
  const void* W;  // dw: dY
  int64_t ldw;    // row pitch of W_e (dw: of dY)
  int64_t w_stride;
  void* Y;  // dw: dW
  int64_t ldy;
  const int32_t* offsets;  // E + 1 device integers; null: one group of all R rows
  int64_t E, R, N, K;
  bool kn;  // opmode RR: W_e (dw: dW_e) is K x N
  bool dw;
  const float* scale = nullptr;    // IN_I8: per row of X
  const float* w_scale = nullptr;  // IN_I8: per (e, n)
  const void* bias = nullptr;      // IN_I8, output type, per n
  bool early = false;  // the kernel before on the stream makes only X and scale (and waited for its own predecessors)
  cudaStream_t stream;
};

// Rows [begin, begin + count) of group e; whatever the offsets hold, the range
// lies in [0, R].
__device__ __forceinline__ void group_range(const int32_t* offsets, int e, int R, int& begin, int& count) {
  if (offsets == nullptr) {
    begin = 0;
    count = R;
    return;
  }
  const int lo = min(max(offsets[e], 0), R), hi = min(max(offsets[e + 1], 0), R);
  begin = lo;
  count = max(hi - lo, 0);
}

int launch_grouped_simt(const GroupedProblem& p);
int launch_grouped_umma(const GroupedProblem& p);
int launch_grouped_skinny(const GroupedProblem& p);
// Whether TMA can address X and W (and dY): the others take the CUDA cores.
bool grouped_tma_ok(const GroupedProblem& p);

// Runs the body of a C entry point; an exception (host memory) becomes a status.
template <typename F>
int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    try {
      set_error("out of host memory");
    } catch (...) {
    }
    return KEBAB_ECUDA;
  }
}

// Launch attributes of a kernel that takes part in programmatic dependent
// launch (it calls pdl_wait() before it touches global memory).
struct PdlLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  PdlLaunch(dim3 grid, dim3 block, size_t smem, cudaStream_t stream, int cluster = 1) {
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 0;
    if (cluster > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = cluster;
      attr[cfg.numAttrs].val.clusterDim.y = 1;
      attr[cfg.numAttrs].val.clusterDim.z = 1;
      ++cfg.numAttrs;
    }
    if (pdl_enabled()) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
      ++cfg.numAttrs;
    }
  }
};

}  // namespace kb
