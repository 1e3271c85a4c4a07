// Rows between token order and expert order: dispatch copies each token's row
// to its choices' places, combine sums a token's choices with their weights,
// and combine's gradient does both in one pass over the rows.
//
// All three are bound by memory: every row is read or written once, 16 bytes a
// thread. The sum runs over a token's own choices in their order, so there are
// no atomics and the result does not depend on the schedule.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "grouped.h"
#include "kebab/experts.h"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int THREADS = 256;

struct ExchangeArgs {
  const void* a;  // dispatch: x; combine: ys; backward: dy
  const void* b;  // backward: ys
  void* out;      // dispatch: xs; combine: y; backward: dys
  int64_t lda, ldb, ldo;
  const int32_t* slots;
  const float* weights;
  float* dweights;
  int64_t T;
  int k;
  int R;
  int H;
};

// One thread a run of W values of a token.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS) dispatch_kernel(const ExchangeArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int per = g.H / W;
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (i >= g.T * per) return;
  const int64_t t = i / per;
  const int h = (int)(i - t * per) * W;
  const T* src = static_cast<const T*>(g.a) + t * g.lda + h;
  T* out = static_cast<T*>(g.out) + h;
  if constexpr (W == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(src);
    for (int j = 0; j < g.k; ++j) {
      const int s = g.slots[t * g.k + j];
      if ((unsigned)s < (unsigned)g.R) *reinterpret_cast<uint4*>(out + (int64_t)s * g.ldo) = v;
    }
  } else {
    const T v = *src;
    for (int j = 0; j < g.k; ++j) {
      const int s = g.slots[t * g.k + j];
      if ((unsigned)s < (unsigned)g.R) out[(int64_t)s * g.ldo] = v;
    }
  }
}

template <typename T, int W>
__global__ void __launch_bounds__(THREADS) combine_kernel(const ExchangeArgs g) {
  pdl_wait();
  pdl_launch_dependents();
  const int per = g.H / W;
  const int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x;
  if (i >= g.T * per) return;
  const int64_t t = i / per;
  const int h = (int)(i - t * per) * W;
  const T* ys = static_cast<const T*>(g.a) + h;
  float acc[W] = {};
#pragma unroll 4
  for (int j = 0; j < g.k; ++j) {
    const int s = g.slots[t * g.k + j];
    if ((unsigned)s >= (unsigned)g.R) continue;
    const float w = g.weights ? g.weights[t * g.k + j] : 1.f;
    float v[W];
    load_row<W>(ys + (int64_t)s * g.lda, v);
#pragma unroll
    for (int u = 0; u < W; ++u) acc[u] += w * v[u];
  }
  store_row<W>(static_cast<T*>(g.out) + t * g.ldo + h, acc);
}

// One block a token: dys = w dy and the products <dy, ys>, JB choices at a
// time so that their rows are in flight together.
template <typename T, int W>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(const ExchangeArgs g) {
  constexpr int JB = 4;
  __shared__ float part[JB][THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = blockIdx.x;
  const T* dy = static_cast<const T*>(g.a) + t * g.lda;
  for (int j0 = 0; j0 < g.k; j0 += JB) {
    int s[JB];
    float w[JB], sum[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      s[j] = j0 + j < g.k ? g.slots[t * g.k + j0 + j] : -1;
      if ((unsigned)s[j] >= (unsigned)g.R) s[j] = -1;
      w[j] = s[j] >= 0 ? g.weights[t * g.k + j0 + j] : 0.f;
      sum[j] = 0.f;
    }
    for (int h = threadIdx.x * W; h < g.H; h += blockDim.x * W) {
      float d[W], v[JB][W];
      load_row<W>(dy + h, d);
#pragma unroll
      for (int j = 0; j < JB; ++j)
        if (s[j] >= 0) load_row<W>(static_cast<const T*>(g.b) + (int64_t)s[j] * g.ldb + h, v[j]);
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        if (s[j] < 0) continue;
        float o[W];
#pragma unroll
        for (int u = 0; u < W; ++u) {
          sum[j] += d[u] * v[j][u];
          o[u] = w[j] * d[u];
        }
        store_row<W>(static_cast<T*>(g.out) + (int64_t)s[j] * g.ldo + h, o);
      }
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
      if ((threadIdx.x & 31) == 0) part[j][threadIdx.x >> 5] = sum[j];
    }
    __syncthreads();
    if (threadIdx.x < JB && j0 + threadIdx.x < g.k) {
      float total = 0.f;
      for (int x = 0; x < (int)blockDim.x / 32; ++x) total += part[threadIdx.x][x];
      g.dweights[t * g.k + j0 + threadIdx.x] = total;
    }
    __syncthreads();
  }
}

bool aligned(const void* p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0; }

int check(const char* what, int dtype, int64_t T, int k, int64_t R, int64_t H) {
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16 and BF16 are implemented");
  if (k < 1 || k > 32) return fail(KEBAB_EINVAL, std::string(what) + ": k = " + std::to_string(k) + " is not in 1..32");
  if (T < 0 || R < 0 || H <= 0 || T * k >= INT32_MAX || R > INT32_MAX || H > (1 << 24) || T > (1 << 30))
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions T=" + std::to_string(T) +
                                  " R=" + std::to_string(R) + " H=" + std::to_string(H));
  return KEBAB_OK;
}

template <typename K>
int launch_flat(K kern, const ExchangeArgs& g, int64_t items, cudaStream_t stream, const char* what) {
  const int64_t blocks = (items + THREADS - 1) / THREADS;
  if (blocks > INT32_MAX) return fail(KEBAB_EINVAL, std::string(what) + ": too many elements");
  PdlLaunch l(dim3((unsigned)blocks), dim3(THREADS), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, what);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int kebab_expert_dispatch(kebab_dtype dtype, const void* x, int64_t ldx, const int32_t* slots, void* xs, int64_t ldxs,
                          int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream) {
  return guarded([&] {
    int rc = check("expert_dispatch", dtype, T, k, R, H);
    if (rc) return rc;
    if (ldx < H || ldxs < H) return fail(KEBAB_EINVAL, "expert_dispatch: a row pitch is below H");
    if (T == 0 || R == 0) return KEBAB_OK;
    if (!x || !slots || !xs) return fail(KEBAB_EINVAL, "expert_dispatch: null pointer");
    const ExchangeArgs g = {x, nullptr, xs, ldx, 0, ldxs, slots, nullptr, nullptr, T, k, (int)R, (int)H};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    // A copy: both 16-bit types move the same bits.
    if (H % 8 == 0 && aligned(x, ldx) && aligned(xs, ldxs))
      return launch_flat(dispatch_kernel<__half, 8>, g, T * (H / 8), s, "expert_dispatch launch");
    return launch_flat(dispatch_kernel<__half, 1>, g, T * H, s, "expert_dispatch launch");
  });
}

int kebab_expert_combine(kebab_dtype dtype, const void* ys, int64_t ldys, const int32_t* slots, const float* weights,
                         void* y, int64_t ldy, int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream) {
  return guarded([&] {
    int rc = check("expert_combine", dtype, T, k, R, H);
    if (rc) return rc;
    if (ldys < H || ldy < H) return fail(KEBAB_EINVAL, "expert_combine: a row pitch is below H");
    if (T == 0) return KEBAB_OK;
    if ((!ys && R > 0) || !slots || !y) return fail(KEBAB_EINVAL, "expert_combine: null pointer");
    const ExchangeArgs g = {ys, nullptr, y, ldys, 0, ldy, slots, weights, nullptr, T, k, (int)R, (int)H};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool vec = H % 8 == 0 && aligned(ys, ldys) && aligned(y, ldy), h = dtype == KEBAB_F16;
    if (vec)
      return launch_flat(h ? combine_kernel<__half, 8> : combine_kernel<__nv_bfloat16, 8>, g, T * (H / 8), s,
                         "expert_combine launch");
    return launch_flat(h ? combine_kernel<__half, 1> : combine_kernel<__nv_bfloat16, 1>, g, T * H, s,
                       "expert_combine launch");
  });
}

int kebab_expert_combine_backward(kebab_dtype dtype, const void* dy, int64_t lddy, const void* ys, int64_t ldys,
                                  const int32_t* slots, const float* weights, void* dys, int64_t lddys,
                                  float* dweights, int64_t T, int k, int64_t R, int64_t H, kebab_stream_t stream) {
  return guarded([&] {
    int rc = check("expert_combine_backward", dtype, T, k, R, H);
    if (rc) return rc;
    if (lddy < H || ldys < H || lddys < H)
      return fail(KEBAB_EINVAL, "expert_combine_backward: a row pitch is below H");
    if (T == 0) return KEBAB_OK;
    if (!dy || !slots || !weights || !dweights || (R > 0 && (!ys || !dys)))
      return fail(KEBAB_EINVAL, "expert_combine_backward: null pointer");
    const ExchangeArgs g = {dy, ys, dys, lddy, ldys, lddys, slots, weights, dweights, T, k, (int)R, (int)H};
    const bool vec = H % 8 == 0 && aligned(dy, lddy) && aligned(ys, ldys) && aligned(dys, lddys);
    const bool h = dtype == KEBAB_F16;
    auto kern = vec ? (h ? combine_backward_kernel<__half, 8> : combine_backward_kernel<__nv_bfloat16, 8>)
                    : (h ? combine_backward_kernel<__half, 1> : combine_backward_kernel<__nv_bfloat16, 1>);
    const int64_t runs = (H + (vec ? 8 : 1) - 1) / (vec ? 8 : 1);
    PdlLaunch l(dim3((unsigned)T), dim3((unsigned)std::min<int64_t>(THREADS, (runs + 31) / 32 * 32)), 0,
                reinterpret_cast<cudaStream_t>(stream));
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "expert_combine_backward launch");
  });
}

}  // extern "C"
