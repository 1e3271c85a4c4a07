// C entry points of the 4-bit floating-point products (include/kebab/f4.h):
// argument checks and the choice of kernel.
#include <algorithm>
#include <string>

#include "f4.h"
#include "kebab/f4.h"

namespace kb {

int f4_weight_map(const F4Problem& p, CUtensorMap* m) {
  const uint64_t pitch = f4_pitch(p.K);
  const uint64_t dims[3] = {pitch, (uint64_t)p.N, (uint64_t)p.E}, strides[2] = {pitch, pitch * p.N};
  const uint32_t box[3] = {128, 128, 1};
  return make_tmap(m, p.w_codes, TMAP_U8, 3, dims, strides, box, 128);
}

int f4_weight_scale_map(const F4Problem& p, CUtensorMap* m) {
  const uint64_t k_tiles = (p.K + 127) / 128, n_tiles = (p.N + 127) / 128;
  const uint64_t dims[3] = {256, k_tiles, p.E * n_tiles}, strides[2] = {512, k_tiles * 512};
  const uint32_t box[3] = {256, 2, 1};
  return make_tmap(m, p.w_scales, KEBAB_F16, 3, dims, strides, box, 0);
}

int f4_token_map(const F4Problem& p, int rows, CUtensorMap* m) {
  const uint64_t pitch = f4_pitch(p.K);
  const uint64_t dims[2] = {pitch, (uint64_t)p.R}, strides[1] = {pitch};
  const uint32_t box[2] = {128, (uint32_t)rows};
  return make_tmap(m, p.x_codes, TMAP_U8, 2, dims, strides, box, 128);
}

int f4_token_scale_map(const F4Problem& p, CUtensorMap* m) {
  const uint64_t dims[2] = {(uint64_t)(p.R + F4_SLACK) * 8, (uint64_t)((p.K + 127) / 128)};
  const uint64_t strides[1] = {(uint64_t)(p.R + F4_SLACK) * 16};
  const uint32_t box[2] = {256, 2};
  return make_tmap(m, p.x_scales, KEBAB_F16, 2, dims, strides, box, 0);
}

namespace {
constexpr int64_t kMaxDim = int64_t(1) << 30;  // leaves room for tile arithmetic in 32 bits

int run(const char* what, const F4Problem& p) {
  if (p.out != KEBAB_F16 && p.out != KEBAB_BF16)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16 and BF16 are implemented");
  if (p.E < 1 || p.E > kMaxExperts)
    return fail(KEBAB_EINVAL, std::string(what) + ": number of experts " + std::to_string(p.E) + " is not in 1.." +
                                  std::to_string(kMaxExperts));
  if (p.R < 0 || p.N <= 0 || p.K <= 0 || p.R > kMaxDim || p.N > kMaxDim || p.K > kMaxDim)
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions rows=" + std::to_string(p.R) +
                                  " N=" + std::to_string(p.N) + " K=" + std::to_string(p.K));
  // Coordinates of the scales' tensor maps are 32 bits.
  if (p.R > F4_MAX_ROWS || p.E * ((p.N + 127) / 128) > (1 << 30))
    return fail(KEBAB_EINVAL, std::string(what) + ": more than 2^27 rows, or than 2^30 runs of 128 weight rows");
  if (p.ldy < p.N)
    return fail(KEBAB_EINVAL, std::string(what) + ": row pitch of Y (" + std::to_string(p.ldy) +
                                  ") is below its row length (" + std::to_string(p.N) + ")");
  if (!p.w_codes || !p.w_scales || (p.R > 0 && ((!p.x && (!p.x_codes || !p.x_scales)) || !p.Y)))
    return fail(KEBAB_EINVAL, std::string(what) + ": null pointer");
  auto off16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) != 0; };
  if (off16(p.w_codes) || off16(p.w_scales) || off16(p.x_codes) || off16(p.x_scales))
    return fail(KEBAB_EINVAL, std::string(what) + ": codes and scales must be 16-byte aligned");
  if (p.R == 0) return KEBAB_OK;
  DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc) return rc;
  // The few-rows kernel up to 128 rows (28672 x 8192: 64 rows 37 us against 43, 128
  // rows 39 against 43; from 144 on, two shares, 57 against 43), and where the
  // persistent one would have tiles for less than half of its CTA pairs (4096 x
  // 14336, 192 rows, 16 tiles: 25 us against 29; 512 rows, 48 tiles: 31 both; 8192
  // x 8192, 384 rows, 64 tiles: 29 against 27).
  const int64_t tiles = (p.N + 255) / 256 * (p.offsets ? p.R / 240 + std::min(p.E, p.R) : (p.R + 239) / 240);
  return p.R <= 128 || tiles <= dev->sm_count / 4 ? launch_f4_skinny(p) : launch_f4_umma(p);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int kebab_gemm_f4(kebab_dtype out, const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                  const uint8_t* w_scales, const void* bias, void* Y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                  kebab_stream_t stream) {
  return guarded([&] {
    return run("gemm_f4", {out, x_codes, x_scales, w_codes, w_scales, bias, Y, ldy, nullptr, 1, M, N, K, false,
                           reinterpret_cast<cudaStream_t>(stream)});
  });
}

int kebab_gemm_grouped_f4(kebab_dtype out, const uint8_t* x_codes, const uint8_t* x_scales, const uint8_t* w_codes,
                          const uint8_t* w_scales, void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t R,
                          int64_t N, int64_t K, kebab_stream_t stream) {
  return guarded([&] {
    if (R > 0 && !offsets) return fail(KEBAB_EINVAL, "gemm_grouped_f4: null pointer");
    return run("gemm_grouped_f4", {out, x_codes, x_scales, w_codes, w_scales, nullptr, Y, ldy, offsets, E, R, N, K,
                                   false, reinterpret_cast<cudaStream_t>(stream)});
  });
}

// Codes (a multiple of 16 bytes), then the scales.
int64_t kebab_linear_f4_workspace(int64_t M, int64_t K) {
  const int64_t codes = kebab_f4_code_bytes(M, K);
  return codes < 0 ? codes : codes + kebab_f4_token_scale_bytes(M, K);
}

int kebab_linear_f4(kebab_dtype dtype, const void* X, int64_t ldx, const uint8_t* w_codes, const uint8_t* w_scales,
                    const void* bias, void* Y, int64_t ldy, const int32_t* offsets, int64_t E, int64_t M, int64_t N,
                    int64_t K, void* workspace, int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "linear_f4";
    if (offsets ? bias != nullptr : E != 1)
      return fail(KEBAB_EINVAL, offsets ? "linear_f4: a grouped product takes no bias"
                                        : "linear_f4: without offsets there is one weight matrix (E = 1)");
    F4Problem p = {dtype, nullptr, nullptr, w_codes, w_scales, bias, Y, ldy, offsets, E, 0, N, K, false,
                   reinterpret_cast<cudaStream_t>(stream)};
    int rc = run(what, p);  // the checks
    if (rc) return rc;
    if (M < 0 || M > F4_MAX_ROWS) return fail(KEBAB_EINVAL, "linear_f4: invalid dimensions rows=" + std::to_string(M));
    if (ldx < K) return fail(KEBAB_EINVAL, "linear_f4: row pitch of X is below its row length");
    if (M == 0) return KEBAB_OK;
    if (!X || !Y) return fail(KEBAB_EINVAL, "linear_f4: null pointer");
    if (!workspace || workspace_bytes < kebab_linear_f4_workspace(M, K) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u))
      return fail(KEBAB_EINVAL, "linear_f4: the workspace is null, too small or not 16-byte aligned");
    // (Where Y may lie on X, X is quantised before the product writes.)
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(X), y0 = reinterpret_cast<uintptr_t>(Y);
    const bool apart = x0 >= y0 + 2 * ((M - 1) * ldy + N) || y0 >= x0 + 2 * ((M - 1) * ldx + K);
    if (M <= F4_FUSED_ROWS && apart) {
      p.x = X, p.ldx = ldx, p.R = M;
      return run(what, p);
    }
    uint8_t* codes = static_cast<uint8_t*>(workspace);
    uint8_t* scales = codes + kebab_f4_code_bytes(M, K);
    if ((rc = kebab_quantize_f4_tokens(dtype, X, ldx, codes, scales, M, K, stream))) return rc;
    p.x_codes = codes, p.x_scales = scales, p.R = M, p.early = true;
    return run(what, p);
  });
}

}  // extern "C"
