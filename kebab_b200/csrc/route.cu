// Top-k routing: the experts and weights of every token, and the plan that
// sorts all choices by expert (a stable counting sort), and its gradient.
//
// One warp a token; lane l holds the logits of experts l, l + 32, ... as
// unsigned keys in the floats' order. A choice is one warp-wide maximum of the
// keys and one warp-wide minimum of the experts that hold it, so ties go to
// the lower expert. The softmax runs on the chosen logits (renormalised) or on
// all of them, in FP32, from the largest logit.
//
// The sort: a block owns a run of tokens and takes it in steps of 128. In a
// step every choice sets its token's bit in a mask of its expert (OR: the
// order of the atomics does not matter); a choice's rank among the block's
// choices of that expert is then the count of the earlier steps plus the bits
// below its own. Few tokens: one block finishes the sort by itself. Otherwise
// each block writes its counts by expert, and a second launch, with the same
// split, adds the counts of all earlier blocks and all lower experts.
//
// Bound by launch latency for few tokens, and by the keys' arithmetic (about
// 20 instructions a choice and token) for many: the logits' bytes are few.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "grouped.h"
#include "kebab/experts.h"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int STEP = 128;           // tokens a step
constexpr int MASK_WORDS = STEP / 32;
constexpr int MAX_CHOICES = 32;
constexpr int ONE_BLOCK = 128;      // up to this many tokens one block does all
constexpr int BLOCKS = 148;

__device__ __forceinline__ uint32_t key_of(float x) {
  x += 0.f;  // -0 becomes +0: they are equal
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);  // NaN's key gives a NaN
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}

struct RouteArgs {
  const void* logits;
  int64_t ld;
  int T, E, k;
  int renormalize;
  int chunk;  // tokens a block
  float* weights;
  int32_t* experts;
  int32_t* offsets;
  int32_t* slots;
  int32_t* counts;  // [blocks][E]
};

// Sum over the block's E counts before each expert, in shared memory:
// base[e] = sum of total[0 .. e), for E <= 1024; base[E] is the sum of all.
__device__ void exclusive_scan(const int* total, int* base, int E) {
  if (threadIdx.x < 32) {
    const int per = (E + 31) / 32, e0 = threadIdx.x * per;
    int sum = 0;
    for (int i = 0; i < per && e0 + i < E; ++i) sum += total[e0 + i];
    int at = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, at, d);
      if (threadIdx.x >= d) at += up;
    }
    int run = at - sum;
    for (int i = 0; i < per && e0 + i < E; ++i) {
      base[e0 + i] = run;
      run += total[e0 + i];
    }
    if (threadIdx.x == 31) base[E] = at;
  }
  __syncthreads();
}

template <typename T, int VPL, int THREADS, bool ONE>
__global__ void __launch_bounds__(THREADS) route_kernel(const RouteArgs g) {
  extern __shared__ int smem[];
  int* count = smem;                                              // [E] of the steps before
  uint32_t* mask = reinterpret_cast<uint32_t*>(count + g.E);      // [E][MASK_WORDS]
  int* base = reinterpret_cast<int*>(mask + g.E * MASK_WORDS);    // [E + 1], ONE only
  __shared__ uint16_t chosen[STEP * MAX_CHOICES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* logits = static_cast<const T*>(g.logits);
  pdl_wait();
  pdl_launch_dependents();
  for (int e = threadIdx.x; e < g.E; e += THREADS) count[e] = 0;
  const int begin = blockIdx.x * g.chunk, end = min(g.T, begin + g.chunk);
  for (int t0 = begin; t0 < end; t0 += STEP) {
    const int n = min(STEP, end - t0);
    for (int i = threadIdx.x; i < g.E * MASK_WORDS; i += THREADS) mask[i] = 0;
    __syncthreads();
    for (int i = warp; i < n; i += THREADS / 32) {
      const T* row = logits + (int64_t)(t0 + i) * g.ld;
      uint32_t key[VPL];
      float v[VPL];
#pragma unroll
      for (int u = 0; u < VPL; ++u) {
        const int e = lane + 32 * u;
        v[u] = e < g.E ? to_float(row[e]) : 0.f;
        key[u] = e < g.E ? key_of(v[u]) : 0u;  // 0 is below the key of -inf
      }
      uint32_t my_key = 0, top_key = 0;
      int my_expert = 0;
      for (int j = 0; j < g.k; ++j) {
        uint32_t best = key[0];
        int at = lane;
#pragma unroll
        for (int u = 1; u < VPL; ++u) {
          if (key[u] > best) {
            best = key[u];
            at = lane + 32 * u;
          }
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const int e = (int)__reduce_min_sync(0xffffffffu, best == top ? (unsigned)at : 0xffffffffu);
        if (j == 0) top_key = top;
        if (lane == j) {
          my_key = top;
          my_expert = e;
        }
#pragma unroll
        for (int u = 0; u < VPL; ++u)
          if (e == lane + 32 * u) key[u] = 0;
      }
      const float highest = key_value(top_key);
      const float p = lane < g.k ? expf(key_value(my_key) - highest) : 0.f;
      float sum = p;
      if (!g.renormalize) {
        sum = 0.f;
#pragma unroll
        for (int u = 0; u < VPL; ++u)
          if (lane + 32 * u < g.E) sum += expf(v[u] - highest);
      }
      sum = warp_sum(sum);
      if (lane < g.k) {
        const int64_t at = (int64_t)(t0 + i) * g.k + lane;
        g.weights[at] = top_key == 0x007fffffu ? 0.f : p / sum;  // all logits -inf: nothing to weigh
        g.experts[at] = my_expert;
        chosen[i * g.k + lane] = (uint16_t)my_expert;
        atomicOr(&mask[my_expert * MASK_WORDS + (i >> 5)], 1u << (i & 31));
      }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < n * g.k; x += THREADS) {
      const int i = x / g.k, e = chosen[x];
      int rank = count[e] + __popc(mask[e * MASK_WORDS + (i >> 5)] & ((1u << (i & 31)) - 1u));
      for (int w = 0; w < (i >> 5); ++w) rank += __popc(mask[e * MASK_WORDS + w]);
      g.slots[(int64_t)t0 * g.k + x] = rank;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < g.E; e += THREADS) {
      int c = count[e];
#pragma unroll
      for (int w = 0; w < MASK_WORDS; ++w) c += __popc(mask[e * MASK_WORDS + w]);
      count[e] = c;
    }
    __syncthreads();  // the next step clears the masks
  }
  __syncthreads();
  if constexpr (!ONE) {
    for (int e = threadIdx.x; e < g.E; e += THREADS) g.counts[(int64_t)blockIdx.x * g.E + e] = count[e];
  } else {
    exclusive_scan(count, base, g.E);
    for (int e = threadIdx.x; e <= g.E; e += THREADS) g.offsets[e] = base[e];
    // At most one step: `chosen` still holds every choice, and each thread
    // adds to the ranks that it wrote itself.
    for (int x = threadIdx.x; x < (end - begin) * g.k; x += THREADS) g.slots[x] += base[chosen[x]];
  }
}

// Second launch: slots += the choices of lower experts and of earlier blocks.
__global__ void __launch_bounds__(512) route_place_kernel(const RouteArgs g) {
  extern __shared__ int smem[];
  int* total = smem;            // [E]
  int* before = smem + g.E;     // [E]
  int* base = before + g.E;     // [E + 1]
  for (int e = threadIdx.x; e < 2 * g.E; e += blockDim.x) smem[e] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const int n = gridDim.x * g.E;
  for (int x = threadIdx.x; x < n; x += blockDim.x) {
    const int c = g.counts[x], b = x / g.E, e = x - b * g.E;
    if (c) {
      atomicAdd(&total[e], c);
      if (b < blockIdx.x) atomicAdd(&before[e], c);
    }
  }
  __syncthreads();
  exclusive_scan(total, base, g.E);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= g.E; e += blockDim.x) g.offsets[e] = base[e];
  const int64_t begin = (int64_t)blockIdx.x * g.chunk, end = min((int64_t)g.T, begin + g.chunk);
  for (int64_t x = begin * g.k + threadIdx.x; x < end * g.k; x += blockDim.x) {
    const int e = g.experts[x];
    g.slots[x] += base[e] + before[e];
  }
}

struct RouteBackArgs {
  const void* logits;
  int64_t ld, ldd;
  int T, E, k, renormalize;
  const float* weights;
  const int32_t* experts;
  const float* dweights;
  void* dlogits;
};

// Renormalised: dl = w (dw - <w, dw>) at the chosen experts, 0 elsewhere.
// Otherwise, with p the softmax over all: dl = p (dw - <w, dw>), dw 0 where not chosen.
template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteBackArgs g) {
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= g.T) return;
  float w = 0.f, dw = 0.f;
  int expert = -1;
  if (lane < g.k) {
    w = g.weights[t * g.k + lane];
    dw = g.dweights[t * g.k + lane];
    expert = g.experts[t * g.k + lane];
  }
  const float dot = warp_sum(w * dw);
  float p[VPL], d[VPL];
#pragma unroll
  for (int u = 0; u < VPL; ++u) p[u] = 0.f, d[u] = 0.f;
  for (int j = 0; j < g.k; ++j) {
    const int e = __shfl_sync(0xffffffffu, expert, j);
    const float wj = __shfl_sync(0xffffffffu, w, j), dj = __shfl_sync(0xffffffffu, dw, j);
#pragma unroll
    for (int u = 0; u < VPL; ++u)
      if (e == lane + 32 * u) p[u] = wj, d[u] = dj;
  }
  if (!g.renormalize) {
    const T* row = static_cast<const T*>(g.logits) + t * g.ld;
    float v[VPL], top = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < VPL; ++u) {
      const int e = lane + 32 * u;
      v[u] = e < g.E ? to_float(row[e]) : -INFINITY;
      nan |= v[u] != v[u];
      top = fmaxf(top, v[u]);
    }
    top = key_value(__reduce_max_sync(0xffffffffu, key_of(nan ? NAN : top)));
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < VPL; ++u) {
      p[u] = (lane + 32 * u < g.E && top != -INFINITY) ? expf(v[u] - top) : 0.f;
      sum += p[u];
    }
    sum = warp_sum(sum);
    if (top != -INFINITY) {
#pragma unroll
      for (int u = 0; u < VPL; ++u) p[u] /= sum;
    }
  }
  T* out = static_cast<T*>(g.dlogits) + t * g.ldd;
#pragma unroll
  for (int u = 0; u < VPL; ++u)
    if (lane + 32 * u < g.E) out[lane + 32 * u] = from_float<T>(p[u] * (d[u] - dot));
}

template <typename T, int VPL>
int launch_route(RouteArgs& g, cudaStream_t stream) {
  const size_t smem = (size_t)g.E * (1 + MASK_WORDS) * sizeof(int);
  cudaError_t e;
  if (g.T <= ONE_BLOCK) {
    g.chunk = ONE_BLOCK;
    PdlLaunch l(dim3(1), dim3(1024), smem + (g.E + 1) * sizeof(int), stream);
    e = cudaLaunchKernelEx(&l.cfg, route_kernel<T, VPL, 1024, true>, (const RouteArgs)g);
  } else {
    const int blocks = std::min(BLOCKS, (g.T + 63) / 64);
    g.chunk = (g.T + blocks - 1) / blocks;
    const int grid = (g.T + g.chunk - 1) / g.chunk;
    PdlLaunch l(dim3(grid), dim3(512), smem, stream);
    e = cudaLaunchKernelEx(&l.cfg, route_kernel<T, VPL, 512, false>, (const RouteArgs)g);
    if (e == cudaSuccess) {
      PdlLaunch m(dim3(grid), dim3(512), (size_t)(3 * g.E + 1) * sizeof(int), stream);
      e = cudaLaunchKernelEx(&m.cfg, route_place_kernel, (const RouteArgs)g);
    }
  }
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "route launch");
}

template <typename T, int VPL>
int launch_back(const RouteBackArgs& g, cudaStream_t stream) {
  PdlLaunch l(dim3((unsigned)((g.T + 7) / 8)), dim3(256), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, route_backward_kernel<T, VPL>, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "route_backward launch");
}

// Calls f with the logits' type and the values a lane holds as template arguments.
template <typename F>
int dispatch(int dtype, int64_t E, F&& f) {
  auto by_lane = [&](auto t) {
    using T = decltype(t);
    if (E <= 32) return f(T(), std::integral_constant<int, 1>());
    if (E <= 64) return f(T(), std::integral_constant<int, 2>());
    if (E <= 128) return f(T(), std::integral_constant<int, 4>());
    if (E <= 256) return f(T(), std::integral_constant<int, 8>());
    if (E <= 512) return f(T(), std::integral_constant<int, 16>());
    return f(T(), std::integral_constant<int, 32>());
  };
  if (dtype == KEBAB_F16) return by_lane(__half());
  if (dtype == KEBAB_BF16) return by_lane(__nv_bfloat16());
  return by_lane(0.f);
}

int check(const char* what, int dtype, int64_t ld, int64_t T, int64_t E, int k) {
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16 && dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16, BF16 and F32 are implemented");
  if (E < 1 || E > kMaxExperts)
    return fail(KEBAB_EINVAL, std::string(what) + ": number of experts " + std::to_string(E) + " is not in 1.." +
                                  std::to_string(kMaxExperts));
  if (k < 1 || k > E || k > MAX_CHOICES)
    return fail(KEBAB_EINVAL, std::string(what) + ": k = " + std::to_string(k) + " is not in 1..min(E, 32)");
  if (T < 0 || T * k >= INT32_MAX || T > (1 << 30))
    return fail(KEBAB_EINVAL, std::string(what) + ": number of tokens " + std::to_string(T) + " is out of range");
  if (ld < E) return fail(KEBAB_EINVAL, std::string(what) + ": row pitch of the logits is below E");
  return KEBAB_OK;
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int64_t kebab_route_workspace(int64_t T, int64_t E) {
  if (T < 0 || E < 1 || E > kMaxExperts) return -KEBAB_EINVAL;
  return T <= ONE_BLOCK ? 0 : BLOCKS * E * (int64_t)sizeof(int32_t);
}

int kebab_route(kebab_dtype dtype, const void* logits, int64_t ld, int64_t T, int64_t E, int k, int renormalize,
                float* weights, int32_t* experts, int32_t* offsets, int32_t* slots, void* workspace,
                int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    int rc = check("route", dtype, ld, T, E, k);
    if (rc) return rc;
    if (!offsets || (T > 0 && (!logits || !weights || !experts || !slots)))
      return fail(KEBAB_EINVAL, "route: null pointer");
    const int64_t need = kebab_route_workspace(T, E);
    if (need > 0 && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3u)))
      return fail(KEBAB_EINVAL, "route: the workspace is null, too small or not 4-byte aligned");
    RouteArgs g = {logits, ld, (int)T, (int)E, k, renormalize, 0, weights, experts, offsets, slots,
                   static_cast<int32_t*>(workspace)};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dispatch(dtype, E, [&](auto t, auto vpl) { return launch_route<decltype(t), decltype(vpl)::value>(g, s); });
  });
}

int kebab_route_backward(kebab_dtype dtype, const void* logits, int64_t ld, int64_t T, int64_t E, int k,
                         int renormalize, const float* weights, const int32_t* experts, const float* dweights,
                         void* dlogits, int64_t ldd, kebab_stream_t stream) {
  return guarded([&] {
    int rc = check("route_backward", dtype, ld, T, E, k);
    if (rc) return rc;
    if (ldd < E) return fail(KEBAB_EINVAL, "route_backward: row pitch of dlogits is below E");
    if (T == 0) return KEBAB_OK;
    if (!logits || !weights || !experts || !dweights || !dlogits)
      return fail(KEBAB_EINVAL, "route_backward: null pointer");
    const RouteBackArgs g = {logits, ld, ldd, (int)T, (int)E, k, renormalize, weights, experts, dweights, dlogits};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dispatch(dtype, E, [&](auto t, auto vpl) { return launch_back<decltype(t), decltype(vpl)::value>(g, s); });
  });
}

}  // extern "C"
