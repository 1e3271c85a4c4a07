// 4-bit floating-point products on the CUDA cores: a thread an output, the
// blocks' sums in integers (twice a code's value is one).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "f4.h"
#include "vec.cuh"

namespace kb {
namespace {

__device__ __forceinline__ int twice(uint32_t code) {
  const int m = (int)(0xC8643210u >> (code & 7u) * 4 & 15u);
  return code & 8u ? -m : m;
}

__device__ __forceinline__ float power(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255u ? 0x7fffffffu : byte << 23);
}

template <typename TO>
__global__ void f4_simt_kernel(const F4Problem p) {
  const int64_t n = (int64_t)blockIdx.x * 128 + threadIdx.x, r = blockIdx.y;
  if (n >= p.N) return;
  int e = 0;
  if (p.offsets) {
    for (e = 0; e < p.E; ++e) {
      int begin, rows;
      group_range(p.offsets, e, (int)p.R, begin, rows);
      if (r >= begin && r < begin + rows) break;
    }
    if (e == p.E) return;
  }
  const int64_t pitch = f4_pitch(p.K), tiles = (p.K + 127) / 128;
  const uint8_t* x = p.x_codes + r * pitch;
  const uint8_t* w = p.w_codes + (e * p.N + n) * pitch;
  const uint8_t* ws = p.w_scales + (e * ((p.N + 127) / 128) + n / 128) * tiles * 512 + n % 32 * 16 + n % 128 / 32 * 4;
  float sum = 0.f;
  for (int64_t b = 0; b < pitch / 16; ++b) {
    int s = 0;
    for (int i = 0; i < 16; ++i) {
      const uint32_t cx = x[b * 16 + i], cw = w[b * 16 + i];
      s += twice(cx & 15u) * twice(cw & 15u) + twice(cx >> 4) * twice(cw >> 4);
    }
    const uint8_t* xs = p.x_scales + ((b / 4) * (p.R + F4_SLACK) + r) * 16;
    sum += (float)s * 0.25f * power(xs[b % 4]) * power(ws[b / 4 * 512 + b % 4]);
  }
  if (p.bias) sum += to_float(static_cast<const TO*>(p.bias)[n]);
  static_cast<TO*>(p.Y)[r * p.ldy + n] = from_float<TO>(sum);
}
}  // namespace

int launch_f4_simt(const F4Problem& p) {
  const dim3 grid((unsigned)((p.N + 127) / 128), (unsigned)p.R);
  if (p.out == KEBAB_F16) f4_simt_kernel<__half><<<grid, 128, 0, p.stream>>>(p);
  else f4_simt_kernel<__nv_bfloat16><<<grid, 128, 0, p.stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "gemm_f4 launch");
}

}  // namespace kb
