// C entry points of the grouped and 8-bit integer products
// (include/kebab/experts.h, include/kebab/int8.h): argument checks and the
// choice of kernel.
#include <algorithm>
#include <string>

#include "grouped.h"
#include "kebab/experts.h"
#include "kebab/int8.h"

namespace kb {
namespace {
constexpr int64_t kMaxDim = int64_t(1) << 30;  // leaves room for tile arithmetic in 32 bits

int check_sizes(const char* what, int64_t E, int64_t R, int64_t N, int64_t K) {
  if (E < 1 || E > kMaxExperts)
    return fail(KEBAB_EINVAL, std::string(what) + ": number of experts " + std::to_string(E) + " is not in 1.." +
                                  std::to_string(kMaxExperts));
  if (R < 0 || N <= 0 || K <= 0)
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions rows=" + std::to_string(R) +
                                  " N=" + std::to_string(N) + " K=" + std::to_string(K));
  if (R > kMaxDim || N > kMaxDim || K > kMaxDim)
    return fail(KEBAB_EINVAL, std::string(what) + ": rows, N and K must not exceed 2^30");
  return KEBAB_OK;
}

int check_type(const char* what, int dtype) {
  if (dtype == KEBAB_F16 || dtype == KEBAB_BF16) return KEBAB_OK;
  return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16 and BF16 are implemented");
}

int check_pitch(const char* what, const char* name, int64_t ld, int64_t cols) {
  if (ld >= cols) return KEBAB_OK;
  return fail(KEBAB_EINVAL, std::string(what) + ": row pitch of " + name + " (" + std::to_string(ld) +
                                ") is below its row length (" + std::to_string(cols) + ")");
}

// "RC" (also null) or "RR", either case.
int parse_mode(const char* what, const char* opmode, bool* kn) {
  const std::string m = opmode ? opmode : "RC";
  auto is = [&](size_t i, char c) { return m.size() == 2 && (m[i] == c || m[i] == c + ('a' - 'A')); };
  if (is(0, 'R') && (is(1, 'C') || is(1, 'R'))) {
    *kn = is(1, 'R');
    return KEBAB_OK;
  }
  return fail(KEBAB_EINVAL, std::string(what) + ": opmode must be RC or RR, got " + m);
}

// The skinny kernel up to 128 rows, and where the persistent one would have
// tiles for less than half of its CTA pairs. us, skinny against persistent:
// int8 64 x 8192 x 8192 19.4 and 23.1, 128 rows 24.2 and 25.8, 256 rows (32
// tiles) 28.3 and 34.0, 400 rows (64 tiles) 35.8 and 34.8; 1024 x 1024 x 8192 (16
// tiles) 24.3 and 35.4; 16-bit 200 rows of 16 experts 2048 x 2048 25.1 and 27.2,
// 100 rows of 64 experts 1024 x 1024 27.3 and 26.9.
int run(const GroupedProblem& p) {
  // dw without rows has no operand for a tensor map; it only writes zeros.
  if (p.R == 0 || !grouped_tma_ok(p)) return launch_grouped_simt(p);
  if (p.dw) return launch_grouped_umma(p);
  DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc) return rc;
  const int64_t tiles = (p.N + 255) / 256 * (p.offsets ? p.R / 256 + std::min(p.E, p.R) : (p.R + 255) / 256);
  return p.R <= 128 || tiles <= dev->sm_count / 4 ? launch_grouped_skinny(p) : launch_grouped_umma(p);
}

int run_i8(int out, const int8_t* q, int64_t ldq, const float* scale, const int8_t* Wq, int64_t ldw,
           int64_t w_stride, const float* w_scale, const void* bias, void* Y, int64_t ldy, const int32_t* offsets,
           int64_t E, int64_t R, int64_t N, int64_t K, bool early, kebab_stream_t stream) {
  GroupedProblem p = {};
  p.early = early;
  p.in = IN_I8, p.out = out;
  p.X = q, p.ldx = ldq, p.W = Wq, p.ldw = ldw, p.w_stride = w_stride, p.Y = Y, p.ldy = ldy;
  p.offsets = offsets, p.E = E, p.R = R, p.N = N, p.K = K;
  p.scale = scale, p.w_scale = w_scale, p.bias = bias;
  p.stream = reinterpret_cast<cudaStream_t>(stream);
  return run(p);
}

// The longest K whose 32-bit sums are exact. Any codes: a product is at most
// 2^14 (-128 twice), and 2^17 of them are 2^31. The codes that linear_i8 makes
// are at least -127, products with any weights at most 127 * 2^7.
constexpr int64_t kMaxKAny = (int64_t(1) << 17) - 1, kMaxKQuantized = int64_t(1) << 17;
static_assert(kMaxKAny << 14 <= INT32_MAX && kMaxKQuantized * 127 * 128 <= INT32_MAX, "sums fit 32 bits");

int check_i8(const char* what, int out, const void* X, int64_t ldx, const int8_t* Wq, int64_t ldw, int64_t w_stride,
             const float* w_scale, const void* Y, int64_t ldy, int64_t E, int64_t R, int64_t N, int64_t K,
             int64_t max_k) {
  int rc;
  if ((rc = check_type(what, out)) || (rc = check_sizes(what, E, R, N, K))) return rc;
  if (K > max_k)
    return fail(KEBAB_EINVAL, std::string(what) + ": K above " + std::to_string(max_k) +
                                  " could overflow the 32-bit sums");
  if ((rc = check_pitch(what, "X", ldx, K)) || (rc = check_pitch(what, "W", ldw, K)) ||
      (rc = check_pitch(what, "Y", ldy, N)))
    return rc;
  if (E > 1 && w_stride < (N - 1) * ldw + K)
    return fail(KEBAB_EINVAL, std::string(what) + ": the experts' weights overlap");
  if (!Wq || !w_scale || (R > 0 && (!X || !Y))) return fail(KEBAB_EINVAL, std::string(what) + ": null pointer");
  return KEBAB_OK;
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int kebab_gemm_grouped(kebab_dtype dtype, const void* X, int64_t ldx, const void* W, int64_t ldw, int64_t w_stride,
                       void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K,
                       const char* opmode, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "gemm_grouped";
    GroupedProblem p = {};
    int rc;
    if ((rc = check_type(what, dtype)) || (rc = check_sizes(what, E, R, N, K)) || (rc = parse_mode(what, opmode, &p.kn)))
      return rc;
    const int64_t wr = p.kn ? K : N, wc = p.kn ? N : K;
    if ((rc = check_pitch(what, "X", ldx, K)) || (rc = check_pitch(what, "W", ldw, wc)) ||
        (rc = check_pitch(what, "Y", ldy, N)))
      return rc;
    if (E > 1 && w_stride < (wr - 1) * ldw + wc) return fail(KEBAB_EINVAL, "gemm_grouped: the experts' weights overlap");
    if (R == 0) return KEBAB_OK;
    if (!X || !W || !Y || !offsets) return fail(KEBAB_EINVAL, "gemm_grouped: null pointer");
    p.in = p.out = dtype;
    p.X = X, p.ldx = ldx, p.W = W, p.ldw = ldw, p.w_stride = w_stride, p.Y = Y, p.ldy = ldy;
    p.offsets = offsets, p.E = E, p.R = R, p.N = N, p.K = K;
    p.stream = reinterpret_cast<cudaStream_t>(stream);
    return run(p);
  });
}

int kebab_gemm_grouped_dw(kebab_dtype dtype, const void* X, int64_t ldx, const void* dY, int64_t lddy, void* dW,
                          const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K, const char* opmode,
                          kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "gemm_grouped_dw";
    GroupedProblem p = {};
    int rc;
    if ((rc = check_type(what, dtype)) || (rc = check_sizes(what, E, R, N, K)) || (rc = parse_mode(what, opmode, &p.kn)))
      return rc;
    if ((rc = check_pitch(what, "X", ldx, K)) || (rc = check_pitch(what, "dY", lddy, N))) return rc;
    if (!dW || !offsets || (R > 0 && (!X || !dY))) return fail(KEBAB_EINVAL, "gemm_grouped_dw: null pointer");
    p.dw = true;
    p.in = p.out = dtype;
    p.X = X, p.ldx = ldx, p.W = dY, p.ldw = lddy, p.Y = dW, p.ldy = p.kn ? N : K;
    p.offsets = offsets, p.E = E, p.R = R, p.N = N, p.K = K;
    p.stream = reinterpret_cast<cudaStream_t>(stream);
    return run(p);
  });
}

int kebab_gemm_i8(kebab_dtype out, const int8_t* q, int64_t ldq, const float* scale, const int8_t* Wq, int64_t ldw,
                  const float* w_scale, const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                  kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "gemm_i8";
    int rc = check_i8(what, out, q, ldq, Wq, ldw, 0, w_scale, Y, ldy, 1, M, N, K, kMaxKAny);
    if (rc || M == 0) return rc;
    if (!scale) return fail(KEBAB_EINVAL, "gemm_i8: null pointer");
    return run_i8(out, q, ldq, scale, Wq, ldw, 0, w_scale, bias, Y, ldy, nullptr, 1, M, N, K, false, stream);
  });
}

int kebab_gemm_grouped_i8(kebab_dtype out, const int8_t* q, int64_t ldq, const float* scale, const int8_t* Wq,
                          int64_t ldw, int64_t w_stride, const float* w_scale, void* Y, int64_t ldy,
                          const int32_t* offsets, int64_t E, int64_t R, int64_t N, int64_t K, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "gemm_grouped_i8";
    int rc = check_i8(what, out, q, ldq, Wq, ldw, w_stride, w_scale, Y, ldy, E, R, N, K, kMaxKAny);
    if (rc || R == 0) return rc;
    if (!scale || !offsets) return fail(KEBAB_EINVAL, "gemm_grouped_i8: null pointer");
    return run_i8(out, q, ldq, scale, Wq, ldw, w_stride, w_scale, nullptr, Y, ldy, offsets, E, R, N, K, false, stream);
  });
}

// Codes with rows padded to 16 bytes, then the scales.
int64_t kebab_linear_i8_workspace(int64_t M, int64_t K) {
  if (M < 0 || K <= 0 || M > kMaxDim || K > kMaxDim) return -KEBAB_EINVAL;
  return M * ((K + 15) / 16 * 16) + M * (int64_t)sizeof(float);
}

int kebab_linear_i8(kebab_dtype dtype, const void* X, int64_t ldx, const int8_t* Wq, int64_t ldw, int64_t w_stride,
                    const float* w_scale, const void* bias, void* Y, int64_t ldy, const int32_t* offsets, int64_t E,
                    int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "linear_i8";
    int rc = check_i8(what, dtype, X, ldx, Wq, ldw, w_stride, w_scale, Y, ldy, E, M, N, K, kMaxKQuantized);
    if (rc) return rc;
    if (offsets ? bias != nullptr : E != 1)
      return fail(KEBAB_EINVAL, offsets ? "linear_i8: a grouped product takes no bias"
                                        : "linear_i8: without offsets there is one weight matrix (E = 1)");
    if (M == 0) return KEBAB_OK;
    if (!workspace || workspace_bytes < kebab_linear_i8_workspace(M, K) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u))
      return fail(KEBAB_EINVAL, "linear_i8: the workspace is null, too small or not 16-byte aligned");
    const int64_t ldq = (K + 15) / 16 * 16;
    int8_t* q = static_cast<int8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(q + M * ldq);
    if ((rc = kebab_quantize_i8(dtype, X, ldx, q, ldq, scale, M, K, stream))) return rc;
    return run_i8(dtype, q, ldq, scale, Wq, ldw, w_stride, w_scale, bias, Y, ldy, offsets, E, M, N, K, true, stream);
  });
}

}  // extern "C"
