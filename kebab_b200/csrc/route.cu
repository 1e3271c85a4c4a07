// Top-k routing: the experts and weights of every token, and the plan that
// sorts all choices by expert (a stable counting sort), and its gradient.
//
// 4 to 32 lanes take a token, each 8 of its logits (more above 256 experts),
// as unsigned keys in the floats' order. A choice is the largest key over the
// lanes, ties to the lower expert: a 16-bit logit and its expert share one
// 32-bit key; a 32-bit logit travels with its expert. The softmax runs on the
// chosen logits (renormalised) or on all of them, in FP32, from the largest
// logit.
//
// The sort: a block owns a run of tokens and takes it in steps of 256. In a
// step every choice sets its token's bit in a mask of its expert (OR: the
// order of the atomics does not matter); a choice's rank among the block's
// choices of that expert is then the count of the earlier steps plus the bits
// below its own. Few tokens: one block finishes the sort by itself. Otherwise
// each block writes its counts by expert, and a second launch, with the same
// split, adds the counts of all earlier blocks and all lower experts.
//
// Bound by latency for few tokens and by the choices' instructions for many (32768
// tokens of 64 experts, 6 choices: 917 for a warp's 4 tokens, issued in 65 % of
// the active cycles); the second launch waits for memory (it issues in 11 %). The
// logits' bytes are few. A whole warp a token reduces with the warp-wide
// instructions, fewer lanes with shuffles: 1 token of 128 experts, 8 choices,
// 3.7 us with 32 lanes and 5.9 with 16; 32768 tokens of 64 experts, 6 choices,
// 29 with 32 and 17 with 8.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "grouped.h"
#include "kebab/experts.h"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int STEP = 256;           // tokens a step
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

// The keys that a maximum is taken over, with the expert in the low half where
// it fits (lower experts higher). 0 is below every expert's key.
template <typename T>
struct Key {
  static constexpr bool PACKED = sizeof(T) == 2;
  static __device__ __forceinline__ uint32_t make(T v, int e) {
    if constexpr (PACKED) {
      uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
      const float x = to_float(v);
      if (x == 0.f) b = 0;
      b = (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
      if (x != x) b = 0xffffu;
      return b << 16 | (0xffffu - e);
    } else {
      return key_of(v);
    }
  }
  // The larger of two (ties: the lower expert).
  static __device__ __forceinline__ void take(uint32_t& key, int& e, uint32_t other, int other_e) {
    if constexpr (PACKED) {
      key = max(key, other);
    } else if (other > key || (other == key && other_e < e)) {
      key = other;
      e = other_e;
    }
  }
  static __device__ __forceinline__ float value(uint32_t key) {
    if constexpr (PACKED) {
      const uint32_t k = key >> 16;
      const uint16_t b = (uint16_t)((k & 0x8000u) ? (k ^ 0x8000u) : ~k);
      return to_float(*reinterpret_cast<const T*>(&b));
    } else {
      return key_value(key);
    }
  }
};

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

template <typename T, int LANES, int V, bool ONE>
__global__ void __launch_bounds__(1024) route_kernel(const RouteArgs g) {
  constexpr int THREADS = 1024, AT_ONCE = THREADS / LANES;  // tokens of a block at a time
  extern __shared__ int smem[];
  int* count = smem;                                              // [E] of the steps before
  uint32_t* mask = reinterpret_cast<uint32_t*>(count + g.E);      // [E][MASK_WORDS]
  int* base = reinterpret_cast<int*>(mask + g.E * MASK_WORDS);    // [E + 1], ONE only
  float* part = reinterpret_cast<float*>(base + (ONE ? g.E + 1 : 0));  // [STEP][k]: weights times their sum
  uint16_t* chosen = reinterpret_cast<uint16_t*>(part + STEP * g.k);   // [STEP][k]
  __shared__ float s_sum[STEP];
  const int lane = threadIdx.x % LANES;
  const T* logits = static_cast<const T*>(g.logits);
  const int begin = blockIdx.x * g.chunk, end = min(g.T, begin + g.chunk);
  for (int e = threadIdx.x; e < g.E; e += THREADS) count[e] = 0;
  for (int i = threadIdx.x; i < g.E * MASK_WORDS; i += THREADS) mask[i] = 0;
  pdl_wait();
  pdl_launch_dependents();
  __syncthreads();
  for (int t0 = begin; t0 < end; t0 += STEP) {
    const int n = min(STEP, end - t0);
    // Whole warps go round together: the shuffles need all their lanes.
    for (int i0 = threadIdx.x / 32 * (32 / LANES); i0 < n; i0 += AT_ONCE) {
      const int i = i0 + threadIdx.x % 32 / LANES;
      // Past the end: the last token again, whose result is not kept.
      const T* row = logits + (int64_t)(t0 + min(i, n - 1)) * g.ld;
      uint32_t key[V];
#pragma unroll
      for (int u = 0; u < V; ++u) {
        const int e = lane + LANES * u;
        key[u] = e < g.E ? Key<T>::make(row[e], e) : 0u;
      }
      float highest = 0.f, sum = 0.f;
      for (int j = 0; j < g.k; ++j) {
        uint32_t top = key[0];
        int e = lane;
#pragma unroll
        for (int u = 1; u < V; ++u) {
          if constexpr (Key<T>::PACKED) {
            top = max(top, key[u]);
          } else if (key[u] > top) {
            top = key[u];
            e = lane + LANES * u;
          }
        }
        if constexpr (LANES == 32) {
          const uint32_t mine = top;
          top = __reduce_max_sync(0xffffffffu, mine);
          if constexpr (!Key<T>::PACKED)
            e = (int)__reduce_min_sync(0xffffffffu, mine == top ? (unsigned)e : 0xffffffffu);
        } else {
#pragma unroll
          for (int d = LANES / 2; d; d >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, top, d);
            const int other_e = Key<T>::PACKED ? 0 : __shfl_xor_sync(0xffffffffu, e, d);
            Key<T>::take(top, e, other, other_e);
          }
        }
        if constexpr (Key<T>::PACKED) e = 0xffff - (top & 0xffffu);
        const float v = Key<T>::value(top);
        if (j == 0) {
          highest = v;
          if (!g.renormalize) {
#pragma unroll
            for (int u = 0; u < V; ++u)
              if (lane + LANES * u < g.E) sum += expf(Key<T>::value(key[u]) - highest);
#pragma unroll
            for (int d = LANES / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          }
        }
        // All logits -inf: nothing to weigh.
        const float p = highest == -INFINITY ? 0.f : expf(v - highest);
        if (g.renormalize) sum += p;
        if (lane == 0 && i < n) {
          part[i * g.k + j] = p;
          chosen[i * g.k + j] = (uint16_t)e;
          atomicOr(&mask[e * MASK_WORDS + (i >> 5)], 1u << (i & 31));
        }
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (e == lane + LANES * u) key[u] = 0;
      }
      if (lane == 0 && i < n) s_sum[i] = highest == -INFINITY ? 1.f : sum;
    }
    __syncthreads();
    if constexpr (ONE) {
      // The only step.
      for (int e = threadIdx.x; e < g.E; e += THREADS) {
        int c = 0;
#pragma unroll
        for (int w = 0; w < ONE_BLOCK / 32; ++w) c += __popc(mask[e * MASK_WORDS + w]);
        count[e] = c;
      }
      __syncthreads();
      exclusive_scan(count, base, g.E);
    }
    for (int x = threadIdx.x; x < n * g.k; x += THREADS) {
      const int i = x / g.k, e = chosen[x];
      int rank = (ONE ? base[e] : count[e]) + __popc(mask[e * MASK_WORDS + (i >> 5)] & ((1u << (i & 31)) - 1u));
      for (int w = 0; w < (i >> 5); ++w) rank += __popc(mask[e * MASK_WORDS + w]);
      const int64_t at = (int64_t)t0 * g.k + x;
      g.weights[at] = part[x] / s_sum[i];
      g.experts[at] = e;
      g.slots[at] = rank;
    }
    if constexpr (!ONE) {
      __syncthreads();
      for (int e = threadIdx.x; e < g.E; e += THREADS) {
        int c = count[e];
#pragma unroll
        for (int w = 0; w < MASK_WORDS; ++w) {
          c += __popc(mask[e * MASK_WORDS + w]);
          mask[e * MASK_WORDS + w] = 0;
        }
        count[e] = c;
      }
      __syncthreads();
    }
  }
  if constexpr (ONE) {
    if (begin >= end) {  // no tokens
      __syncthreads();
      exclusive_scan(count, base, g.E);
    }
    for (int e = threadIdx.x; e <= g.E; e += THREADS) g.offsets[e] = base[e];
  } else {
    for (int e = threadIdx.x; e < g.E; e += THREADS) g.counts[(int64_t)blockIdx.x * g.E + e] = count[e];
  }
}

// Second launch: slots += the choices of lower experts and of earlier blocks.
// A thread sums the counts of one expert over every `slices`-th block.
constexpr int PLACE_THREADS = 512;
__global__ void __launch_bounds__(PLACE_THREADS) route_place_kernel(const RouteArgs g) {
  extern __shared__ int smem[];
  const int slices = max(1, PLACE_THREADS / g.E);
  int* total = smem;            // [slices][E]
  int* before = total + slices * g.E;  // [slices][E]
  int* base = before + slices * g.E;   // [E + 1]
  pdl_wait();
  pdl_launch_dependents();
  // The first choices of this thread are on their way while the counts are summed.
  constexpr int HELD = 4;
  const int64_t begin = (int64_t)blockIdx.x * g.chunk * g.k;
  const int64_t end = min((int64_t)g.T, (int64_t)(blockIdx.x + 1) * g.chunk) * g.k;
  int expert[HELD], rank[HELD];
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int64_t x = begin + h * PLACE_THREADS + threadIdx.x;
    expert[h] = x < end ? g.experts[x] : 0;
    rank[h] = x < end ? g.slots[x] : 0;
  }
  for (int x = threadIdx.x; x < slices * g.E; x += PLACE_THREADS) {
    const int slice = x / g.E, e = x - slice * g.E;
    int all = 0, early = 0;
#pragma unroll 20
    for (int b = slice; b < (int)gridDim.x; b += slices) {
      const int c = g.counts[b * g.E + e];
      all += c;
      if (b < (int)blockIdx.x) early += c;
    }
    total[x] = all;
    before[x] = early;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < g.E; e += PLACE_THREADS) {
    for (int s = 1; s < slices; ++s) {
      total[e] += total[s * g.E + e];
      before[e] += before[s * g.E + e];
    }
  }
  __syncthreads();
  exclusive_scan(total, base, g.E);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= g.E; e += PLACE_THREADS) g.offsets[e] = base[e];
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int64_t x = begin + h * PLACE_THREADS + threadIdx.x;
    if (x < end) g.slots[x] = rank[h] + base[expert[h]] + before[expert[h]];
  }
  for (int64_t x = begin + HELD * PLACE_THREADS + threadIdx.x; x < end; x += PLACE_THREADS) {
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
// Otherwise, with p the softmax over all: dl = p (dw - <w, dw>), dw 0 where not
// chosen. The lanes write the row as if nothing were chosen, and then the k
// chosen places (w is p there).
// 32768 tokens of 64 experts, 6 choices: 8.6 us, bound by its instructions (issued
// in 71 % of the cycles).
// Tokens that a warp has in flight, by the logits a lane holds of each.
template <int VPL>
struct BackShape {
  static constexpr int TOKENS = VPL <= 2 ? 4 : VPL <= 8 ? 2 : 1;
};

template <typename T, int VPL>
__global__ void __launch_bounds__(256) route_backward_kernel(const RouteBackArgs g) {
  constexpr int TOKENS = BackShape<VPL>::TOKENS;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_launch_dependents();
  const int64_t t0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * TOKENS;
  if (t0 >= g.T) return;
  float w[TOKENS], dw[TOKENS], dot[TOKENS], p[TOKENS][VPL];
  int expert[TOKENS];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) {
    // Past the end: the last token again, whose result is not kept.
    const int64_t t = min(t0 + m, (int64_t)g.T - 1);
    w[m] = dw[m] = 0.f;
    expert[m] = -1;
    if (lane < g.k) {
      expert[m] = g.experts[t * g.k + lane];
      w[m] = g.weights[t * g.k + lane];
      dw[m] = g.dweights[t * g.k + lane];
      // A dropped choice: no part of <w, dw> either.
      if ((unsigned)expert[m] >= (unsigned)g.E) w[m] = dw[m] = 0.f;
    }
    dot[m] = w[m] * dw[m];
    if (!g.renormalize) {
      const T* row = static_cast<const T*>(g.logits) + t * g.ld;
#pragma unroll
      for (int u = 0; u < VPL; ++u) p[m][u] = lane + 32 * u < g.E ? to_float(row[lane + 32 * u]) : -INFINITY;
    }
  }
  float sum[TOKENS], top[TOKENS];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) {
    sum[m] = 0.f;
    top[m] = 0.f;
    if (!g.renormalize) {
      uint32_t key = 0;
#pragma unroll
      for (int u = 0; u < VPL; ++u)
        if (lane + 32 * u < g.E) key = max(key, key_of(p[m][u]));
      top[m] = key_value(__reduce_max_sync(0xffffffffu, key));
#pragma unroll
      for (int u = 0; u < VPL; ++u) {
        p[m][u] = lane + 32 * u < g.E ? expf(p[m][u] - top[m]) : 0.f;
        sum[m] += p[m][u];
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
#pragma unroll
    for (int m = 0; m < TOKENS; ++m) {
      dot[m] += __shfl_xor_sync(0xffffffffu, dot[m], d);
      sum[m] += __shfl_xor_sync(0xffffffffu, sum[m], d);
    }
  }
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) {
    if (t0 + m >= g.T) break;
    T* out = static_cast<T*>(g.dlogits) + (t0 + m) * g.ldd;
    const bool none = g.renormalize || top[m] == -INFINITY;
    const float scale = none ? 0.f : -dot[m] / sum[m];
#pragma unroll
    for (int u = 0; u < VPL; ++u)
      if (lane + 32 * u < g.E) out[lane + 32 * u] = from_float<T>(none ? 0.f : p[m][u] * scale);
  }
  __syncwarp();
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)
    if (t0 + m < g.T && (unsigned)expert[m] < (unsigned)g.E)
      static_cast<T*>(g.dlogits)[(t0 + m) * g.ldd + expert[m]] = from_float<T>(w[m] * (dw[m] - dot[m]));
}

// Dynamic shared memory of a block for E experts and k choices.
constexpr size_t route_smem(int E, int k, bool one) {
  return (size_t)(E * (1 + MASK_WORDS) + (one ? E + 1 : 0)) * sizeof(int) + (size_t)STEP * k * 6;
}

template <typename T, int LANES, int V, bool ONE>
int route_smem_limit() {
  // Once per device, for the most that this kernel is launched with: the limit
  // belongs to the kernel, and other threads may be launching it.
  constexpr size_t most = route_smem(LANES * V, MAX_CHOICES, ONE);
  static std::once_flag once[64];
  static cudaError_t err[64];
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  const int di = dev & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(route_kernel<T, LANES, V, ONE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  });
  return err[di] == cudaSuccess ? KEBAB_OK : cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
}

template <typename T, int LANES, int V>
int launch_route(RouteArgs& g, cudaStream_t stream) {
  const bool one = g.T <= ONE_BLOCK;
  const size_t smem = route_smem(g.E, g.k, one);
  auto kern = one ? route_kernel<T, LANES, V, true> : route_kernel<T, LANES, V, false>;
  // Up to 48 KB, s_sum included, need no opt-in.
  if (smem + STEP * sizeof(float) > 48 * 1024) {
    const int rc = one ? route_smem_limit<T, LANES, V, true>() : route_smem_limit<T, LANES, V, false>();
    if (rc) return rc;
  }
  cudaError_t e = cudaSuccess;
  const int blocks = one ? 1 : std::min(BLOCKS, (g.T + 63) / 64);
  g.chunk = one ? ONE_BLOCK : (g.T + blocks - 1) / blocks;
  const int grid = one ? 1 : (g.T + g.chunk - 1) / g.chunk;
  PdlLaunch l(dim3(grid), dim3(1024), smem, stream);
  e = cudaLaunchKernelEx(&l.cfg, kern, (const RouteArgs)g);
  if (e == cudaSuccess && !one) {
    const size_t place = (size_t)(2 * std::max(1, PLACE_THREADS / g.E) * g.E + g.E + 1) * sizeof(int);
    PdlLaunch m(dim3(grid), dim3(PLACE_THREADS), place, stream);
    e = cudaLaunchKernelEx(&m.cfg, route_place_kernel, (const RouteArgs)g);
  }
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "route launch");
}

template <typename T, int VPL>
int launch_back(const RouteBackArgs& g, cudaStream_t stream) {
  constexpr int PER_BLOCK = 8 * BackShape<VPL>::TOKENS;
  PdlLaunch l(dim3((unsigned)((g.T + PER_BLOCK - 1) / PER_BLOCK)), dim3(256), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, route_backward_kernel<T, VPL>, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "route_backward launch");
}

// Calls f with the logits' type.
template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == KEBAB_F16) return f(__half());
  if (dtype == KEBAB_BF16) return f(__nv_bfloat16());
  return f(0.f);
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
    return by_type(dtype, [&](auto t) {
      using L = decltype(t);
      if (E <= 128 && T <= 32) return launch_route<L, 32, 4>(g, s);  // a warp for each token
      if (E <= 32) return launch_route<L, 4, 8>(g, s);
      if (E <= 64) return launch_route<L, 8, 8>(g, s);
      if (E <= 128) return launch_route<L, 16, 8>(g, s);
      if (E <= 256) return launch_route<L, 32, 8>(g, s);
      if (E <= 512) return launch_route<L, 32, 16>(g, s);
      return launch_route<L, 32, 32>(g, s);
    });
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
    return by_type(dtype, [&](auto t) {
      using L = decltype(t);
      if (E <= 32) return launch_back<L, 1>(g, s);
      if (E <= 64) return launch_back<L, 2>(g, s);
      if (E <= 128) return launch_back<L, 4>(g, s);
      if (E <= 256) return launch_back<L, 8>(g, s);
      if (E <= 512) return launch_back<L, 16>(g, s);
      return launch_back<L, 32>(g, s);
    });
  });
}

}  // extern "C"
