// Rows between token order and expert order: dispatch copies each token's row
// to its choices' places, combine sums a token's choices with their weights,
// and combine's gradient does both in one pass over the rows.
//
// All three are bound by memory: every row is read or written once, 16 bytes a
// thread, with the loads of four choices in flight together. The sum runs over
// a token's own choices in their order, so there are no atomics and the result
// does not depend on the schedule.
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

// A thread takes a run of W values of a token: threads and blocks in x along
// the row, in y (threads) and x (blocks) over the tokens.
template <int W>
__device__ __forceinline__ bool place(const ExchangeArgs& g, int64_t& t, int& h) {
  t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  h = (blockIdx.y * blockDim.x + threadIdx.x) * W;
  return t < g.T && h < g.H;
}

__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T, int W>
__global__ void __launch_bounds__(THREADS) dispatch_kernel(const ExchangeArgs g) {
  int64_t t;
  int h;
  pdl_wait();
  pdl_launch_dependents();
  if (!place<W>(g, t, h)) return;
  const T* src = static_cast<const T*>(g.a) + t * g.lda + h;
  T* out = static_cast<T*>(g.out) + h;
  if constexpr (W == 8) {
    const uint4 v = load_once(src);
#pragma unroll 4
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

// TOKENS (with few choices each) or JB choices at a time: four loads in flight
// a thread. 16384 tokens of 4 choices x 4096: 110 us, 6.1 TB/s (126 us with a
// branch round each load); of 1 choice: 54 us, 5.0 TB/s.
template <typename T, int W, int TOKENS>
__global__ void __launch_bounds__(THREADS) combine_kernel(const ExchangeArgs g) {
  constexpr int JB = 4 / TOKENS;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * TOKENS;
  const int h = (blockIdx.y * blockDim.x + threadIdx.x) * W;
  if (t0 >= g.T || h >= g.H) return;
  const T* ys = static_cast<const T*>(g.a) + h;
  float acc[TOKENS][W] = {};
  for (int j0 = 0; j0 < g.k; j0 += JB) {
    int s[TOKENS][JB];
    float w[TOKENS][JB];
#pragma unroll
    for (int m = 0; m < TOKENS; ++m) {
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        const bool here = j0 + j < g.k && t0 + m < g.T;
        const int64_t at = (t0 + m) * g.k + j0 + j;
        s[m][j] = here ? g.slots[at] : -1;
        if ((unsigned)s[m][j] >= (unsigned)g.R) s[m][j] = -1;
        w[m][j] = s[m][j] < 0 ? 0.f : g.weights ? g.weights[at] : 1.f;
      }
    }
    if constexpr (W == 8) {
      uint4 raw[TOKENS][JB];
#pragma unroll
      for (int m = 0; m < TOKENS; ++m)
#pragma unroll
        for (int j = 0; j < JB; ++j)
          raw[m][j] = s[m][j] >= 0 ? load_once(ys + (int64_t)s[m][j] * g.lda) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < TOKENS; ++m) {
#pragma unroll
        for (int j = 0; j < JB; ++j) {
          float v[8];
          unpack(ys, raw[m][j], v);
#pragma unroll
          for (int u = 0; u < 8; ++u) acc[m][u] += w[m][j] * v[u];
        }
      }
    } else {
#pragma unroll
      for (int m = 0; m < TOKENS; ++m)
#pragma unroll
        for (int j = 0; j < JB; ++j)
          if (s[m][j] >= 0) acc[m][0] += w[m][j] * to_float(ys[(int64_t)s[m][j] * g.lda]);
    }
  }
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)
    if (t0 + m < g.T) store_row<W>(static_cast<T*>(g.out) + (t0 + m) * g.ldo + h, acc[m]);
}

// W values as they are stored, read once (nothing if not `here`).
template <typename T, int W>
struct Run {
  uint4 raw;
  __device__ __forceinline__ Run() {}
  __device__ __forceinline__ Run(const T* p, bool here) {
    if constexpr (W == 8) raw = here ? load_once(p) : make_uint4(0, 0, 0, 0);
    else raw.x = here ? __float_as_uint(to_float(*p)) : 0u;
  }
  __device__ __forceinline__ void values(float (&v)[W]) const {
    if constexpr (W == 8) unpack((const T*)nullptr, raw, v);
    else v[0] = __uint_as_float(raw.x);
  }
};

// dys = w dy and the products <dy, ys>, JB choices at a time so that their rows
// are in flight together. A warp a token up to rows of 2048, else a block.
// 16384 tokens of 4 choices x 4096: 191 us, 6.3 TB/s; 60000 of 2 x 768: 82 us
// (116 with a block a token and every row's loads behind the one before).
template <typename T, int W, bool WARP, int JB>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(const ExchangeArgs g) {
  __shared__ float part[JB][THREADS / 32];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = WARP ? (int64_t)blockIdx.x * (THREADS / 32) + warp : blockIdx.x;
  if (t >= g.T) return;
  const int first = (WARP ? lane : (int)threadIdx.x) * W, step = (WARP ? 32 : THREADS) * W;
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
#pragma unroll(4 / JB)
    for (int h = first; h < g.H; h += step) {
      Run<T, W> d(dy + h, true), v[JB];
#pragma unroll
      for (int j = 0; j < JB; ++j) v[j] = Run<T, W>(static_cast<const T*>(g.b) + (int64_t)s[j] * g.ldb + h, s[j] >= 0);
      float x[W];
      d.values(x);
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        if (s[j] < 0) continue;
        float y[W];
        v[j].values(y);
#pragma unroll
        for (int u = 0; u < W; ++u) {
          sum[j] += x[u] * y[u];
          y[u] = w[j] * x[u];
        }
        store_row<W>(static_cast<T*>(g.out) + (int64_t)s[j] * g.ldo + h, y);
      }
    }
#pragma unroll
    for (int j = 0; j < JB; ++j) {
#pragma unroll
      for (int d = 16; d; d >>= 1) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], d);
    }
    if constexpr (WARP) {
#pragma unroll
      for (int j = 0; j < JB; ++j)
        if (lane == j && j0 + j < g.k) g.dweights[t * g.k + j0 + j] = sum[j];
    } else {
      if (lane == 0)
#pragma unroll
        for (int j = 0; j < JB; ++j) part[j][warp] = sum[j];
      __syncthreads();
      if (threadIdx.x < JB && j0 + threadIdx.x < g.k) {
        float total = 0.f;
#pragma unroll
        for (int x = 0; x < THREADS / 32; ++x) total += part[threadIdx.x][x];
        g.dweights[t * g.k + j0 + threadIdx.x] = total;
      }
      __syncthreads();
    }
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

// A thread for each run of `w` values of each `tokens` tokens.
template <typename K>
int launch_flat(K kern, const ExchangeArgs& g, int w, int tokens, cudaStream_t stream, const char* what) {
  const int runs = (g.H + w - 1) / w;
  const int x = std::min(THREADS, (runs + 31) / 32 * 32), y = THREADS / x;
  const int64_t rows = (runs + x - 1) / x;
  if (rows > 65535) return fail(KEBAB_EINVAL, std::string(what) + ": rows are too long");
  PdlLaunch l(dim3((unsigned)((g.T + y * tokens - 1) / (y * tokens)), (unsigned)rows), dim3(x, y), 0, stream);
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
      return launch_flat(dispatch_kernel<__half, 8>, g, 8, 1, s, "expert_dispatch launch");
    return launch_flat(dispatch_kernel<__half, 1>, g, 1, 1, s, "expert_dispatch launch");
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
    auto go = [&](auto type) {
      using V = decltype(type);
      const char* what = "expert_combine launch";
      if (!vec) return launch_flat(combine_kernel<V, 1, 1>, g, 1, 1, s, what);
      if (k == 1) return launch_flat(combine_kernel<V, 8, 4>, g, 8, 4, s, what);
      if (k == 2) return launch_flat(combine_kernel<V, 8, 2>, g, 8, 2, s, what);
      return launch_flat(combine_kernel<V, 8, 1>, g, 8, 1, s, what);
    };
    return h ? go(__half()) : go(__nv_bfloat16());
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
    const bool warp = vec && H <= 2048;
    auto pick = [&](auto type) {
      using V = decltype(type);
      if (!vec) return combine_backward_kernel<V, 1, false, 4>;
      if (k == 1) return warp ? combine_backward_kernel<V, 8, true, 1> : combine_backward_kernel<V, 8, false, 1>;
      if (k == 2) return warp ? combine_backward_kernel<V, 8, true, 2> : combine_backward_kernel<V, 8, false, 2>;
      return warp ? combine_backward_kernel<V, 8, true, 4> : combine_backward_kernel<V, 8, false, 4>;
    };
    auto kern = h ? pick(__half()) : pick(__nv_bfloat16());
    PdlLaunch l(dim3((unsigned)(warp ? (T + 7) / 8 : T)), dim3(THREADS), 0, reinterpret_cast<cudaStream_t>(stream));
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "expert_combine_backward launch");
  });
}

}  // extern "C"
