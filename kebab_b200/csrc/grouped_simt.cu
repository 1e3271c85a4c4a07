// Grouped and 8-bit integer products on the CUDA cores, for operands that TMA
// cannot address (base addresses or row pitches that are no multiples of 16
// bytes): any size, pitch and alignment.
//
// Every form is C[i, j] = sum_p A(i, p) B(j, p) with operands given by two
// strides each:
//   forward  i = row of the group, j = n, p = k
//   dw       i = n, j = k, p = row of the group   ("RR": i = k, j = n)
// A block computes a 64 x 64 tile with 16 x 16 threads of 4 x 4 outputs each,
// 16 terms of p at a time from shared memory. It is bound by its loads and
// shared-memory reads (two 16-byte reads feed 16 multiply-adds): 4096 rows over 8
// groups, 4096 x 4100, 16 bits, 5970 us where 4096 x 4096 take 133 on the tensor
// cores. Products of 8 bits come here where K is short (grouped_api.cu).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "group_search.cuh"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int TILE = 64, TP = 16;

__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ int to_acc(int8_t v) { return v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
struct Acc {
  using type = float;
};
template <>
struct Acc<int8_t> {
  using type = int;
};

template <typename T, typename TO>
struct SimtArgs {
  const T* a;
  const T* b;
  TO* c;
  int64_t a_i, a_p, b_j, b_p, c_i;  // strides; c_j = 1
  int64_t a_e, b_e, c_e;            // from one group to the next (0: by rows)
  int64_t a_r, b_r, c_r;            // from one row of a group to the next (0: by group)
  const int32_t* offsets;
  int E, R, I, J, P;  // I (forward) or P (dw) is the group's row count
  const float* scale;
  const float* w_scale;
  const TO* bias;
};

template <typename T, typename TO, bool DW>
__global__ void __launch_bounds__(256) grouped_simt_kernel(const SimtArgs<T, TO> g) {
  using A = typename Acc<T>::type;
  __shared__ A sa[TP][TILE + 4], sb[TP][TILE + 4];
  // Which group, and which of its 64-row tiles (dw: of dW_e's).
  int e = 0, tile = blockIdx.x, begin = 0, rows = 0;
  if constexpr (DW) {
    const int per = (g.I + TILE - 1) / TILE;
    e = tile / per;
    tile -= e * per;
    group_range(g.offsets, e, g.R, begin, rows);
  } else {
    if (!nth_tile<256, TILE>(g.offsets, g.E, g.R, tile, e, begin, rows, tile)) return;
  }
  const int I = DW ? g.I : rows, P = DW ? rows : g.P;
  const int i0 = tile * TILE, j0 = blockIdx.y * TILE;
  const T* a = g.a + e * g.a_e + begin * g.a_r;
  const T* b = g.b + e * g.b_e + begin * g.b_r;
  TO* c = g.c + e * g.c_e + begin * g.c_r;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  A acc[4][4] = {};
  for (int p0 = 0; p0 < P; p0 += TP) {
    // Neighbouring threads follow the stride of 1.
    for (int x = threadIdx.x; x < TILE * TP; x += 256) {
      const int i = g.a_p == 1 ? x / TP : x % TILE, p = g.a_p == 1 ? x % TP : x / TILE;
      sa[p][i] = (i0 + i < I && p0 + p < P) ? to_acc(a[(i0 + i) * g.a_i + (p0 + p) * g.a_p]) : A(0);
      const int j = g.b_p == 1 ? x / TP : x % TILE, pb = g.b_p == 1 ? x % TP : x / TILE;
      sb[pb][j] = (j0 + j < g.J && p0 + pb < P) ? to_acc(b[(j0 + j) * g.b_j + (p0 + pb) * g.b_p]) : A(0);
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < TP; ++p) {
      A x[4], y[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        x[u] = sa[p][ty * 4 + u];
        y[u] = sb[p][tx * 4 + u];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] += x[u] * y[v];
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int i = i0 + ty * 4 + u;
    if (i >= I) continue;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int j = j0 + tx * 4 + v;
      if (j >= g.J) continue;
      float y = (float)acc[u][v];
      // (As the other 8-bit kernels, for the same bits.)
      if constexpr (sizeof(T) == 1)
        y = __fmaf_rn(y, g.w_scale[(int64_t)e * g.J + j] * g.scale[begin + i], g.bias ? to_float(g.bias[j]) : 0.f);
      put(c + i * g.c_i + j, y);
    }
  }
}

template <typename T, typename TO>
int launch(const GroupedProblem& p) {
  SimtArgs<T, TO> g = {};
  const T* X = static_cast<const T*>(p.X);
  const T* W = static_cast<const T*>(p.W);
  g.c = static_cast<TO*>(p.Y);
  g.offsets = p.offsets;
  g.E = (int)p.E;
  g.R = (int)p.R;
  g.scale = p.scale;
  g.w_scale = p.w_scale;
  g.bias = static_cast<const TO*>(p.bias);
  int64_t tiles;
  if (!p.dw) {
    g.a = X, g.a_i = p.ldx, g.a_p = 1, g.a_r = p.ldx;
    g.b = W, g.b_j = p.kn ? 1 : p.ldw, g.b_p = p.kn ? p.ldw : 1, g.b_e = p.w_stride;
    g.c_i = p.ldy, g.c_r = p.ldy;
    g.I = 0, g.J = (int)p.N, g.P = (int)p.K;
    tiles = p.R / TILE + std::min(p.E, p.R);  // upper bound over all splits of R rows
  } else {
    // dW_e: N x K, or K x N with the two operands exchanged.
    g.a = p.kn ? X : W, g.b = p.kn ? W : X;
    g.a_i = 1, g.a_p = g.a_r = p.kn ? p.ldx : p.ldw;
    g.b_j = 1, g.b_p = g.b_r = p.kn ? p.ldw : p.ldx;
    g.I = (int)(p.kn ? p.K : p.N), g.J = (int)(p.kn ? p.N : p.K);
    g.c_i = g.J, g.c_e = p.N * p.K;
    tiles = p.E * ((g.I + TILE - 1) / TILE);
  }
  const int64_t cols = (g.J + TILE - 1) / TILE;
  if (tiles > INT32_MAX || cols > 65535) return fail(KEBAB_EINVAL, "grouped product: too many tiles");
  const dim3 grid((unsigned)tiles, (unsigned)cols);
  if constexpr (sizeof(T) != 1) {
    if (p.dw) grouped_simt_kernel<T, TO, true><<<grid, 256, 0, p.stream>>>(g);
    else grouped_simt_kernel<T, TO, false><<<grid, 256, 0, p.stream>>>(g);
  } else {
    grouped_simt_kernel<T, TO, false><<<grid, 256, 0, p.stream>>>(g);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "grouped SIMT launch");
}
}  // namespace

int launch_grouped_simt(const GroupedProblem& p) {
  const bool h = p.out == KEBAB_F16;
  if (p.in == IN_I8) return h ? launch<int8_t, __half>(p) : launch<int8_t, __nv_bfloat16>(p);
  return h ? launch<__half, __half>(p) : launch<__nv_bfloat16, __nv_bfloat16>(p);
}

}  // namespace kb
