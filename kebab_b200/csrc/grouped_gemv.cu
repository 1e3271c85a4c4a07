// Grouped and 8-bit integer products for a few rows (serving single tokens):
// every weight is read once, straight into registers, so the kernel is bound
// by the weights' bytes.
//
// Weights N x K (RC): a warp takes four rows n and strides over k, 16 bytes a
// lane, row and step; x comes through L1, shared by the four rows. Where N
// leaves too few warps to keep the memory busy, several warps of a block share
// the rows and split k. Weights K x N (RR): a lane takes eight columns n, a
// warp several rows k, a block all of k. Partial sums meet in a fixed order,
// in FP32 or 32-bit integers.
//
// grid.y is a row of X; the block of a group's first row does the group, the
// other rows' blocks leave at once. That needs no sorting and no list of the
// groups in use, whose number only the device knows.
//
// The loads of the next step are issued before the current one is used. In
// linear_i8 the kernel before this one only makes the codes and scales of X, so
// the first weights are on their way while it still runs (`early`).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "grouped.h"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int NR = 4;     // RC: weight rows a warp
constexpr int WARPS = 8;  // RC: warps a block
constexpr int MAX_ROWS = 8;

struct GemvArgs {
  const void* X;
  int64_t ldx;
  const void* W;
  int64_t ldw, w_stride;
  void* Y;
  int64_t ldy;
  const int32_t* offsets;
  int E, R, N, K;
  int splits;  // RC: warps that share rows and split k
  const float* scale;
  const float* w_scale;
  const void* bias;
  int early, pdl;
};

// 16 bytes of weights, read once.
__device__ __forceinline__ uint4 load_once(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// The group of row blockIdx.y if that is its first row. All threads of the
// block take part.
__device__ bool first_row_group(const GemvArgs& g, int& e, int& rows) {
  __shared__ int s_group, s_rows;
  const int row = blockIdx.y;
  if (g.offsets == nullptr) {
    e = 0;
    rows = g.R;
    return row == 0;
  }
  if (threadIdx.x == 0) s_rows = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < g.E; i += blockDim.x) {
    int begin, count;
    group_range(g.offsets, i, g.R, begin, count);
    if (count > 0 && begin == row) {
      s_group = i;
      s_rows = count;
    }
  }
  __syncthreads();
  e = s_group;
  rows = s_rows;
  return rows > 0;
}

template <typename T>
struct Sum {
  using type = float;
};
template <>
struct Sum<int8_t> {
  using type = int;
};

// acc += the products of 16 bytes of W and of X.
__device__ __forceinline__ void dot16(const int8_t*, int& acc, const uint4& w, const uint4& x) {
  acc = __dp4a((int)w.x, (int)x.x, acc);
  acc = __dp4a((int)w.y, (int)x.y, acc);
  acc = __dp4a((int)w.z, (int)x.z, acc);
  acc = __dp4a((int)w.w, (int)x.w, acc);
}

template <typename T, typename TO>
__device__ __forceinline__ void put(const GemvArgs& g, int e, int64_t row, int n, typename Sum<T>::type acc) {
  float y = (float)acc;
  if constexpr (sizeof(T) == 1) {
    y *= g.w_scale[(int64_t)e * g.N + n] * g.scale[row];
    if (g.bias) y += to_float(static_cast<const TO*>(g.bias)[n]);
  }
  static_cast<TO*>(g.Y)[row * g.ldy + n] = from_float<TO>(y);
}

// Rows m0 .. m0 + MT - 1 of the group (those below `rows`) against this warp's
// weight rows. The weights of a later pass over more rows come from L2.
template <typename T, typename TO, int MT>
__device__ __forceinline__ void rc_rows(const GemvArgs& g, int e, int64_t row0, int rows, int n0, int split, bool wait,
                                        typename Sum<T>::type* part) {
  using A = typename Sum<T>::type;
  constexpr int V = 16 / sizeof(T);  // elements of 16 bytes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* W = static_cast<const T*>(g.W) + (int64_t)e * g.w_stride;
  const T* wrow[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) wrow[i] = W + (int64_t)min(n0 + i, g.N - 1) * g.ldw;
  // This warp's share of k, in steps of 32 lanes x 16 bytes.
  const int step = 32 * V, steps = (g.K + step - 1) / step;
  const int per = (steps + g.splits - 1) / g.splits;
  int k = split * per * step + lane * V;
  const int k_end = min(g.K, (split + 1) * per * step);
  A acc[NR][MT] = {};
  uint4 next[NR] = {};
  if (k < k_end) {
#pragma unroll
    for (int i = 0; i < NR; ++i) next[i] = load_once(wrow[i] + k);
  }
  uint4 next2[NR] = {};
  if (k + step < k_end) {
#pragma unroll
    for (int i = 0; i < NR; ++i) next2[i] = load_once(wrow[i] + k + step);
  }
  if (wait) pdl_wait();
  const T* x0 = static_cast<const T*>(g.X) + row0 * g.ldx;
  for (; k < k_end; k += step) {
    uint4 w[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) w[i] = next[i], next[i] = next2[i];
    if (k + 2 * step < k_end) {
#pragma unroll
      for (int i = 0; i < NR; ++i) next2[i] = load_once(wrow[i] + k + 2 * step);
    }
    if constexpr (sizeof(T) == 1) {
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= rows) break;
        const uint4 x = *reinterpret_cast<const uint4*>(x0 + m * g.ldx + k);
#pragma unroll
        for (int i = 0; i < NR; ++i) dot16(wrow[0], acc[i][m], w[i], x);
      }
    } else {
      float f[NR][8];
#pragma unroll
      for (int i = 0; i < NR; ++i) unpack(wrow[0], w[i], f[i]);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= rows) break;
        float x[8];
        load_row<8>(x0 + m * g.ldx + k, x);
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int u = 0; u < 8; ++u) acc[i][m] += f[i][u] * x[u];
      }
    }
  }
  // Sum over the lanes, then (in order) over the warps that split k.
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int d = 16; d; d >>= 1) acc[i][m] += __shfl_xor_sync(0xffffffffu, acc[i][m], d);
      if (g.splits > 1) {
        if (lane == 0) part[warp * NR * MAX_ROWS + m * NR + i] = acc[i][m];
      } else if (lane == m * NR + i && m < rows && n0 + i < g.N) {
        put<T, TO>(g, e, row0 + m, n0 + i, acc[i][m]);
      }
    }
  if (g.splits > 1) {
    __syncthreads();
    if (split == 0 && lane < NR * MT) {
      const int m = lane / NR, i = lane % NR;
      A sum = 0;
      for (int s = 0; s < g.splits; ++s) sum += part[(warp + s) * NR * MAX_ROWS + lane];
      if (m < rows && n0 + i < g.N) put<T, TO>(g, e, row0 + m, n0 + i, sum);
    }
  }
}

template <typename T, typename TO>
__global__ void __launch_bounds__(WARPS * 32) gemv_rc_kernel(const GemvArgs g) {
  __shared__ typename Sum<T>::type part[WARPS * NR * MAX_ROWS];
  const bool early = g.early && g.pdl;
  // A kernel that touches memory before its predecessor is done must not let
  // its successor start.
  if (!early) {
    pdl_wait();
    pdl_launch_dependents();
  }
  int e, rows;
  if (!first_row_group(g, e, rows)) {
    if (early) pdl_wait();
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int n0 = (blockIdx.x * (WARPS / g.splits) + warp / g.splits) * NR, split = warp % g.splits;
  const int64_t row = blockIdx.y;
  if (n0 >= g.N && g.splits == 1) return;
  if (rows == 1) rc_rows<T, TO, 1>(g, e, row, rows, n0, split, early, part);
  else if (rows == 2) rc_rows<T, TO, 2>(g, e, row, rows, n0, split, early, part);
  else if (rows <= 4) rc_rows<T, TO, 4>(g, e, row, rows, n0, split, early, part);
  else rc_rows<T, TO, 8>(g, e, row, rows, n0, split, early, part);
}

// Weights K x N: LN lanes of 8 columns side by side, 32 / LN rows k a warp.
constexpr int RR_WARPS = 16, LN = 8;

template <typename T, int MT>
__device__ __forceinline__ void rr_rows(const GemvArgs& g, int e, int64_t row0, int rows, float* part) {
  constexpr int KL = 32 / LN * RR_WARPS;  // rows k in flight a block and step
  constexpr int U = MT <= 2 ? 8 : 4;      // steps whose loads are issued together
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = (blockIdx.x * LN + lane % LN) * 8;
  const int kl = warp * (32 / LN) + lane / LN;
  const T* W = static_cast<const T*>(g.W) + (int64_t)e * g.w_stride + n;
  const T* x0 = static_cast<const T*>(g.X) + row0 * g.ldx;
  float acc[MT][8] = {};
  if (n < g.N) {
    for (int k0 = kl; k0 < g.K; k0 += KL * U) {
      uint4 w[U];
      float x[U][MT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = k0 + u * KL;
        w[u] = k < g.K ? load_once(W + (int64_t)k * g.ldw) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) x[u][m] = k < g.K && m < rows ? to_float(x0[m * g.ldx + k]) : 0.f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[8];
        unpack(W, w[u], f);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[m][c] += x[u][m] * f[c];
      }
    }
  }
  // Over the lanes of a warp that share columns, then over the warps.
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
#pragma unroll
      for (int d = LN; d < 32; d <<= 1) acc[m][c] += __shfl_xor_sync(0xffffffffu, acc[m][c], d);
      if (lane < LN) part[(warp * MAX_ROWS + m) * LN * 8 + lane * 8 + c] = acc[m][c];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < MT * LN * 8; i += RR_WARPS * 32) {
    const int m = i / (LN * 8), c = i % (LN * 8), col = blockIdx.x * LN * 8 + c;
    float sum = 0.f;
    for (int w = 0; w < RR_WARPS; ++w) sum += part[(w * MAX_ROWS + m) * LN * 8 + c];
    if (m < rows && col < g.N) static_cast<T*>(g.Y)[(row0 + m) * g.ldy + col] = from_float<T>(sum);
  }
}

template <typename T>
__global__ void __launch_bounds__(RR_WARPS * 32) gemv_rr_kernel(const GemvArgs g) {
  __shared__ float part[RR_WARPS * MAX_ROWS * LN * 8];
  pdl_wait();
  pdl_launch_dependents();
  int e, rows;
  if (!first_row_group(g, e, rows)) return;
  const int64_t row = blockIdx.y;
  if (rows == 1) rr_rows<T, 1>(g, e, row, rows, part);
  else if (rows == 2) rr_rows<T, 2>(g, e, row, rows, part);
  else if (rows <= 4) rr_rows<T, 4>(g, e, row, rows, part);
  else rr_rows<T, 8>(g, e, row, rows, part);
}

template <typename T, typename TO>
int launch(const GroupedProblem& p) {
  DeviceInfo* dev = nullptr;
  const int rc = device_info(&dev);
  if (rc) return rc;
  GemvArgs g = {};
  g.X = p.X, g.ldx = p.ldx, g.W = p.W, g.ldw = p.ldw, g.w_stride = p.w_stride, g.Y = p.Y, g.ldy = p.ldy;
  g.offsets = p.offsets, g.E = (int)p.E, g.R = (int)p.R, g.N = (int)p.N, g.K = (int)p.K;
  g.scale = p.scale, g.w_scale = p.w_scale, g.bias = p.bias;
  g.early = p.early, g.pdl = pdl_enabled();
  const unsigned groups = p.offsets ? (unsigned)p.R : 1u;
  cudaError_t e;
  if constexpr (sizeof(T) == 2) {
    if (p.kn) {
      PdlLaunch l(dim3((unsigned)((p.N + LN * 8 - 1) / (LN * 8)), groups), dim3(RR_WARPS * 32), 0, p.stream);
      e = cudaLaunchKernelEx(&l.cfg, gemv_rr_kernel<T>, (const GemvArgs)g);
      return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "few-rows product launch");
    }
  }
  // Split k until there are 16 warps an SM, of at least two steps each.
  const int64_t units = (p.N + NR - 1) / NR * std::min<int64_t>(groups, p.E);
  const int64_t steps = (p.K * (int64_t)sizeof(T) + 511) / 512;
  g.splits = 1;
  while (g.splits < WARPS && units * g.splits < 16 * dev->sm_count && steps >= 4 * g.splits) g.splits *= 2;
  if (getenv("KB_SPLITS")) g.splits = atoi(getenv("KB_SPLITS"));
  const int per_block = WARPS / g.splits * NR;
  PdlLaunch l(dim3((unsigned)((p.N + per_block - 1) / per_block), groups), dim3(WARPS * 32), 0, p.stream);
  e = cudaLaunchKernelEx(&l.cfg, gemv_rc_kernel<T, TO>, (const GemvArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "few-rows product launch");
}
}  // namespace

bool grouped_gemv_ok(const GroupedProblem& p) {
  const int64_t v = p.in == IN_I8 ? 16 : 8;
  return !p.dw && p.R <= (getenv("KB_GEMV") ? atoi(getenv("KB_GEMV")) : MAX_ROWS) && (p.kn ? p.N : p.K) % v == 0 && grouped_tma_ok(p);
}

int launch_grouped_gemv(const GroupedProblem& p) {
  const bool h = p.out == KEBAB_F16;
  if (p.in == IN_I8) return h ? launch<int8_t, __half>(p) : launch<int8_t, __nv_bfloat16>(p);
  return h ? launch<__half, __half>(p) : launch<__nv_bfloat16, __nv_bfloat16>(p);
}

}  // namespace kb
