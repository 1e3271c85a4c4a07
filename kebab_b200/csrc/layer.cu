// A mixture-of-experts layer for a few tokens: a warp an output.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "grouped.h"
#include "kebab/experts.h"
#include "kebab/int8.h"
#include "kebab/layer.h"
#include "quant_i8.cuh"

namespace kb {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

template <typename T>
__global__ void logits_kernel(const T* x, int64_t ldx, const float* router, float* logits, int E, int H) {
  const int e = blockIdx.x, t = blockIdx.y;
  float v = 0.f;
  for (int h = threadIdx.x; h < H; h += 32) v += to_float(x[t * ldx + h]) * router[(int64_t)e * H + h];
  v = warp_sum(v);
  if (threadIdx.x == 0) logits[t * E + e] = v;
}

// Codes of the rows of x, nearest with ties to even.
template <typename T>
__global__ void codes_kernel(const T* x, int64_t ldx, int8_t* q, float* scale, int H) {
  const int t = blockIdx.x;
  uint32_t top = 0;
  for (int h = threadIdx.x; h < H; h += 32) top = max(top, abs_bits(to_float(x[t * ldx + h])));
  top = __reduce_max_sync(0xffffffffu, top);
  const RowScale s = row_scale(top);
  for (int h = threadIdx.x; h < H; h += 32)
    q[(int64_t)t * H + h] = s.inv == 0.f ? 0 : (int8_t)rintf(to_float(x[t * ldx + h]) * 127.f / __uint_as_float(top));
  if (threadIdx.x == 0) scale[t] = s.scale;
}

// Row `t` of x against `row` of a weight matrix.
template <typename A, typename W>
__device__ __forceinline__ float dot(const A* a, const W* w, int n) {
  if constexpr (sizeof(W) == 1) {
    int v = 0;
    for (int i = threadIdx.x; i < n; i += 32) v += (int)a[i] * (int)w[i];
    return (float)warp_sum(v);
  } else {
    float v = 0.f;
    for (int i = threadIdx.x; i < n; i += 32) v += to_float(a[i]) * to_float(w[i]);
    return warp_sum(v);
  }
}

template <typename A, typename W>
__global__ void up_kernel(const A* x, int64_t ldx, const W* w_in, const float* in_scale, const float* x_scale,
                          const int32_t* experts, float* a, int k, int H, int D) {
  const int i = blockIdx.x, j = blockIdx.y, t = j / k;
  const int64_t e = experts[j];
  float g = dot(x + t * ldx, w_in + (e * 2 * D + i) * H, H), u = dot(x + t * ldx, w_in + (e * 2 * D + D + i) * H, H);
  if (in_scale) {
    g *= x_scale[t] * in_scale[e * 2 * D + i];
    u *= x_scale[t] * in_scale[e * 2 * D + D + i];
  }
  if (threadIdx.x == 0) a[(int64_t)j * D + i] = g / (1.f + expf(-g)) * u;
}

template <typename T, typename A, typename W>
__global__ void down_kernel(const A* a, const W* w_out, const float* out_scale, const float* a_scale,
                            const int32_t* experts, const float* weights, T* y, int64_t ldy, int k, int H, int D) {
  const int n = blockIdx.x, t = blockIdx.y;
  float sum = 0.f;
  for (int j = t * k; j < (t + 1) * k; ++j) {
    const int64_t e = experts[j];
    float v = dot(a + (int64_t)j * D, w_out + (e * H + n) * D, D);
    if (out_scale) v *= a_scale[j] * out_scale[e * H + n];
    sum += weights[j] * v;
  }
  if (threadIdx.x == 0) y[t * ldy + n] = from_float<T>(sum);
}

struct Sizes {
  int64_t T, E, k, H, D;
};

// logits, weights, a, its scales, those of x (F32); experts, slots, offsets (I32); codes of a and x.
int64_t words(const Sizes& s) { return s.T * s.E + 4 * s.T * s.k + s.T * s.k * s.D + s.T + s.E + 1; }
int64_t bytes(const Sizes& s) { return words(s) * 4 + s.T * s.k * s.D + s.T * s.H; }

int check(const char* what, int dtype, const void* x, int64_t ldx, const void* router, const void* w_in,
          const void* w_out, const void* y, int64_t ldy, const Sizes& s, void* ws, int64_t ws_bytes) {
  const std::string w = what;
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16) return fail(KEBAB_ENOTSUP, w + ": only F16 and BF16 are implemented");
  if (s.T < 0 || s.T > KEBAB_FEW_TOKENS)
    return fail(KEBAB_EINVAL, w + ": " + std::to_string(s.T) + " tokens are not in 0.." + std::to_string(KEBAB_FEW_TOKENS));
  if (s.E < 1 || s.E > kMaxExperts) return fail(KEBAB_EINVAL, w + ": number of experts " + std::to_string(s.E) + " is not in 1..1024");
  if (s.k < 1 || s.k > 32 || s.k > s.E) return fail(KEBAB_EINVAL, w + ": k = " + std::to_string(s.k) + " is not in 1..min(E, 32)");
  if (s.H <= 0 || s.D <= 0 || s.H > (1 << 24) || s.D > (1 << 24))
    return fail(KEBAB_EINVAL, w + ": invalid dimensions H=" + std::to_string(s.H) + " D=" + std::to_string(s.D));
  if (ldx < s.H || ldy < s.H) return fail(KEBAB_EINVAL, w + ": a row pitch is below the row length");
  if (s.T == 0) return KEBAB_OK;
  if (!x || !router || !w_in || !w_out || !y) return fail(KEBAB_EINVAL, w + ": null pointer");
  if (!ws || ws_bytes < bytes(s) || (reinterpret_cast<uintptr_t>(ws) & 15u))
    return fail(KEBAB_EINVAL, w + ": the workspace is null, too small or not 16-byte aligned");
  return KEBAB_OK;
}

template <typename T, typename W>
int run(const T* x, int64_t ldx, const float* router, const W* w_in, const float* in_scale, const W* w_out,
        const float* out_scale, T* y, int64_t ldy, const Sizes& s, int renormalize, void* ws, kebab_stream_t stream) {
  constexpr bool I8 = sizeof(W) == 1;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int Tk = (int)(s.T * s.k), H = (int)s.H, D = (int)s.D, k = (int)s.k;
  float* logits = static_cast<float*>(ws);
  float* weights = logits + s.T * s.E;
  float* a = weights + Tk;
  float* a_scale = a + (int64_t)Tk * D;
  float* x_scale = a_scale + Tk;
  int32_t* experts = reinterpret_cast<int32_t*>(x_scale + s.T);
  int32_t* slots = experts + Tk;
  int32_t* offsets = slots + Tk;
  int8_t* qa = reinterpret_cast<int8_t*>(offsets + s.E + 1);
  int8_t* qx = qa + (int64_t)Tk * D;
  logits_kernel<<<dim3((unsigned)s.E, (unsigned)s.T), 32, 0, st>>>(x, ldx, router, logits, (int)s.E, H);
  int rc = kebab_route(KEBAB_F32, logits, s.E, s.T, s.E, k, renormalize, weights, experts, offsets, slots, nullptr, 0, stream);
  if (rc) return rc;
  if constexpr (I8) {
    codes_kernel<<<(unsigned)s.T, 32, 0, st>>>(x, ldx, qx, x_scale, H);
    up_kernel<<<dim3(D, Tk), 32, 0, st>>>(qx, H, w_in, in_scale, x_scale, experts, a, k, H, D);
    if ((rc = kebab_quantize_i8(KEBAB_F32, a, D, qa, D, a_scale, Tk, D, stream))) return rc;
    down_kernel<<<dim3(H, (unsigned)s.T), 32, 0, st>>>(qa, w_out, out_scale, a_scale, experts, weights, y, ldy, k, H, D);
  } else {
    up_kernel<<<dim3(D, Tk), 32, 0, st>>>(x, ldx, w_in, in_scale, x_scale, experts, a, k, H, D);
    down_kernel<<<dim3(H, (unsigned)s.T), 32, 0, st>>>(a, w_out, out_scale, a_scale, experts, weights, y, ldy, k, H, D);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "expert_layer launch");
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int64_t kebab_expert_layer_workspace(int64_t T, int64_t E, int k, int64_t H, int64_t D) {
  if (T < 0 || T > KEBAB_FEW_TOKENS || E < 1 || E > kMaxExperts || k < 1 || k > 32 || H <= 0 || D <= 0 ||
      H > (1 << 24) || D > (1 << 24))
    return -KEBAB_EINVAL;
  return bytes({T, E, k, H, D});
}

int kebab_expert_layer(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const void* w_in,
                       const void* w_out, void* y, int64_t ldy, int64_t T, int64_t E, int k, int renormalize,
                       int64_t H, int64_t D, void* workspace, int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const Sizes s = {T, E, k, H, D};
    const int rc = check("expert_layer", dtype, x, ldx, router, w_in, w_out, y, ldy, s, workspace, workspace_bytes);
    if (rc || T == 0) return rc;
    auto go = [&](auto t) {
      using V = decltype(t);
      return run(static_cast<const V*>(x), ldx, router, static_cast<const V*>(w_in), nullptr, static_cast<const V*>(w_out),
                 nullptr, static_cast<V*>(y), ldy, s, renormalize, workspace, stream);
    };
    return dtype == KEBAB_F16 ? go(__half()) : go(__nv_bfloat16());
  });
}

int kebab_expert_layer_i8(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const int8_t* w_in,
                          const float* in_scale, const int8_t* w_out, const float* out_scale, void* y, int64_t ldy,
                          int64_t T, int64_t E, int k, int renormalize, int64_t H, int64_t D, void* workspace,
                          int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const Sizes s = {T, E, k, H, D};
    const int rc = check("expert_layer_i8", dtype, x, ldx, router, w_in, w_out, y, ldy, s, workspace, workspace_bytes);
    if (rc || T == 0) return rc;
    if (H > 131072 || D > 131072) return fail(KEBAB_EINVAL, "expert_layer_i8: H or D above 131072 could overflow the 32-bit sums");
    if (!in_scale || !out_scale) return fail(KEBAB_EINVAL, "expert_layer_i8: null pointer");
    auto go = [&](auto t) {
      using V = decltype(t);
      return run(static_cast<const V*>(x), ldx, router, w_in, in_scale, w_out, out_scale, static_cast<V*>(y), ldy, s,
                 renormalize, workspace, stream);
    };
    return dtype == KEBAB_F16 ? go(__half()) : go(__nv_bfloat16());
  });
}

}  // extern "C"
