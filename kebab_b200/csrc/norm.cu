// Root-mean-square norm with the residual's addition, its form with 8-bit
// output, and its gradients.
//
// Forward: ROW threads take a row, read it once (x and the residual), keep the
// sum in registers as it is stored, and find the sum of squares (and, for 8
// bits, the largest |y|) by shuffles and shared memory. Rows longer than the
// registers hold are read a second time, from L2. Bound by memory for many rows
// and by latency for few: a row then has 1024 threads.
//
// Backward: a block takes every gridDim-th row. A thread has the same columns
// of all of them, so that its share of dweight stays in registers; the blocks'
// sums are added in a fixed order by a second, small kernel. Rows longer than a
// block's registers hold are taken in slabs of columns: the first slab's pass
// also finds the row's two sums (over all columns) and leaves them in the
// workspace.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "grouped.h"
#include "kebab/norm.h"
#include "quant_i8.cuh"

namespace kb {
namespace {

struct NormArgs {
  const void* x;
  int64_t ldx;
  const void* r;  // residual, or null
  int64_t ldr;
  const void* w;
  int w_f32;  // weight in FP32, else in the rows' type
  float eps;
  void* s;
  int64_t lds;
  void* y;
  int64_t ldy;
  int8_t* q;
  int64_t ldq;
  float* scale;
  int64_t rows;
  int cols;
};

// W weights from column c on.
template <typename T, int W>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int c, float (&v)[W]) {
  if (sizeof(T) == 4 || w_f32) load_row<W>(static_cast<const float*>(w) + c, v);
  else load_row<W>(static_cast<const T*>(w) + c, v);
}

// Sums of N values over the ROW threads of a row (a warp or whole warps of the
// block); `part`: N floats a warp.
template <int ROW, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*part)[N]) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
  }
  if constexpr (ROW > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
#pragma unroll
      for (int n = 0; n < N; ++n) part[warp][n] = v[n];
    }
    __syncthreads();
    // Every warp adds the warps' sums in the same way.
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane < ROW / 32 ? part[lane][n] : 0.f;
#pragma unroll
    for (int d = ROW / 64; d; d >>= 1) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], d);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, v[n], 0);
  }
}

// W = 8: 16-byte accesses; W = 1: rows on any boundary. HELD runs of W columns
// a thread in registers.
template <typename T, int W, int HELD, int ROW, bool I8>
__global__ void __launch_bounds__(ROW < 128 ? 128 : ROW) norm_kernel(const NormArgs g) {
  constexpr int PER_BLOCK = (ROW < 128 ? 128 : ROW) / ROW;
  __shared__ float part[32][1];
  __shared__ uint32_t tops[32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * PER_BLOCK + threadIdx.x / ROW;
  if (row >= g.rows) return;
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  const T* r = static_cast<const T*>(g.r) + row * g.ldr;
  T* s = static_cast<T*>(g.s) + row * g.lds;
  const bool add = g.r != nullptr;
  const int c0 = threadIdx.x % ROW * W;
  Run<T, W> held[HELD], other[HELD];
  float v[W], u[W];
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = c0 + h * ROW * W;
    if (c < g.cols) {
      held[h].load(x + c);
      if (add) other[h].load(r + c);
    }
  }
  float sum[1] = {0.f};
  auto square = [&] {
#pragma unroll
    for (int i = 0; i < W; ++i) sum[0] += v[i] * v[i];
  };
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = c0 + h * ROW * W;
    if (c >= g.cols) break;
    held[h].values(v);
    if (add) {
      other[h].values(u);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += u[i];
      held[h].set(v);
      held[h].store(s + c);
      held[h].values(v);
    }
    square();
  }
  for (int c = c0 + HELD * ROW * W; c < g.cols; c += ROW * W) {
    Run<T, W> a;
    a.load(x + c);
    a.values(v);
    if (add) {
      load_row<W>(r + c, u);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += u[i];
      a.set(v);
      a.store(s + c);
      a.values(v);
    }
    square();
  }
  row_sum<ROW, 1>(sum, part);
  const float rstd = rsqrtf(sum[0] / (float)g.cols + g.eps);
  const T* again = add ? s : x;  // the columns past the registers, which this thread wrote
  T* y = static_cast<T*>(g.y) + row * g.ldy;
  // v becomes the columns' output.
  auto output = [&](int c) {
    load_weight<T, W>(g.w, g.w_f32, c, u);
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = v[i] * rstd * u[i];
  };
  if constexpr (!I8) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = c0 + h * ROW * W;
      if (c >= g.cols) break;
      held[h].values(v);
      output(c);
      store_row<W>(y + c, v);
    }
    for (int c = c0 + HELD * ROW * W; c < g.cols; c += ROW * W) {
      load_row<W>(again + c, v);
      output(c);
      store_row<W>(y + c, v);
    }
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = c0 + h * ROW * W;
      if (c >= g.cols) break;
      held[h].values(v);
      output(c);
      top = largest<W>(v, top);
    }
    for (int c = c0 + HELD * ROW * W; c < g.cols; c += ROW * W) {
      load_row<W>(again + c, v);
      output(c);
      top = largest<W>(v, top);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (ROW > 32) {
      const int lane = threadIdx.x & 31;
      if (lane == 0) tops[threadIdx.x >> 5] = top;
      __syncthreads();
      top = __reduce_max_sync(0xffffffffu, lane < ROW / 32 ? tops[lane] : 0u);
    }
    const RowScale code = row_scale(top);
    if (threadIdx.x % ROW == 0) g.scale[row] = code.scale;
    int8_t* q = g.q + row * g.ldq;
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = c0 + h * ROW * W;
      if (c >= g.cols) break;
      held[h].values(v);
      output(c);
      store_codes<W>(q + c, v, code.inv);
      if (g.y) store_row<W>(y + c, v);
    }
    for (int c = c0 + HELD * ROW * W; c < g.cols; c += ROW * W) {
      load_row<W>(again + c, v);
      output(c);
      store_codes<W>(q + c, v, code.inv);
      if (g.y) store_row<W>(y + c, v);
    }
  }
}

template <typename T, int W, bool I8>
int launch_forward(const NormArgs& g, int sms, cudaStream_t stream) {
  const int64_t runs = (g.cols + W - 1) / W;
  // Few rows: 1024 threads a row. Short rows, many of them: a warp a row.
  const bool few = g.rows <= 2 * sms && runs > 256;
  const bool warp = !few && runs <= 128 && g.rows >= 1024;
  const int row = few ? 1024 : warp ? 32 : 128;
  const int64_t held = (runs + row - 1) / row;
  auto kern = norm_kernel<T, W, 8, 128, I8>;
  if (few) kern = held <= 1 ? norm_kernel<T, W, 1, 1024, I8> : norm_kernel<T, W, 2, 1024, I8>;
  else if (warp) kern = held <= 1 ? norm_kernel<T, W, 1, 32, I8> : held <= 2 ? norm_kernel<T, W, 2, 32, I8> : norm_kernel<T, W, 4, 32, I8>;
  else if (held <= 1) kern = norm_kernel<T, W, 1, 128, I8>;
  else if (held <= 2) kern = norm_kernel<T, W, 2, 128, I8>;
  else if (held <= 4) kern = norm_kernel<T, W, 4, 128, I8>;
  const int64_t per_block = warp ? 4 : 1;
  PdlLaunch l(dim3((unsigned)((g.rows + per_block - 1) / per_block)), dim3(few ? 1024 : 128), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm launch");
}

struct GradArgs {
  const void* dy;
  int64_t lddy;
  const void* s;
  int64_t lds;
  const void* w;
  int w_f32;
  float eps;
  const void* ds;  // or null
  int64_t ldds;
  void* dx;  // or null
  int64_t lddx;
  float* partial;  // [blocks][cols] sums of dweight, or null
  float* stats;    // [rows][2]: rstd, mean(g s), where there is more than one slab
  int64_t rows;
  int cols;
};

// AHEAD: the next row of the first slab is loaded before the sums of this one
// are exchanged (where the registers hold two).
template <typename T, int W, int HELD, int THREADS, bool AHEAD>
__global__ void __launch_bounds__(THREADS, AHEAD ? 512 / THREADS : 1) norm_backward_kernel(const GradArgs g) {
  constexpr int SLAB = THREADS * W * HELD;
  __shared__ float part[2][THREADS / 32][2];
  pdl_wait();
  pdl_launch_dependents();
  const bool add = g.ds && g.dx;
  int turn = 0;
  for (int base = 0; base < g.cols; base += SLAB) {
    const int c0 = base + threadIdx.x * W;
    float acc[HELD][W];
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
      for (int i = 0; i < W; ++i) acc[h][i] = 0.f;
    Run<T, W> rs[HELD], rd[HELD], re[HELD], ns[HELD], nd[HELD], ne[HELD];
    auto load = [&](int64_t row, Run<T, W> (&ls)[HELD], Run<T, W> (&ld)[HELD], Run<T, W> (&le)[HELD]) {
      const T* s = static_cast<const T*>(g.s) + row * g.lds + c0;
      const T* dy = static_cast<const T*>(g.dy) + row * g.lddy + c0;
      const T* ds = static_cast<const T*>(g.ds) + row * g.ldds + c0;
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        if (c0 + h * THREADS * W < g.cols) {
          ls[h].load(s + h * THREADS * W);
          ld[h].load(dy + h * THREADS * W);
          if (add) le[h].load(ds + h * THREADS * W);
        }
      }
    };
    if (AHEAD) load(blockIdx.x, ns, nd, ne);
    for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
      if (AHEAD) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) rs[h] = ns[h], rd[h] = nd[h], re[h] = ne[h];
        if (row + gridDim.x < g.rows) load(row + gridDim.x, ns, nd, ne);
      } else {
        load(row, rs, rd, re);
      }
      float a[W], b[W], w[W], sum[2] = {0.f, 0.f};
      auto count = [&](int c) {
        load_weight<T, W>(g.w, g.w_f32, c, w);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          sum[0] += a[i] * a[i];
          sum[1] += b[i] * w[i] * a[i];
        }
      };
      if (base == 0) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
          const int c = c0 + h * THREADS * W;
          if (c >= g.cols) break;
          rs[h].values(a);
          rd[h].values(b);
          count(c);
        }
        for (int c = c0 + SLAB; c < g.cols; c += THREADS * W) {
          load_row<W>(static_cast<const T*>(g.s) + row * g.lds + c, a);
          load_row<W>(static_cast<const T*>(g.dy) + row * g.lddy + c, b);
          count(c);
        }
        row_sum<THREADS, 2>(sum, part[turn]);  // two buffers in turn: one barrier a row
        turn ^= 1;
        sum[0] = rsqrtf(sum[0] / (float)g.cols + g.eps);
        sum[1] = sum[1] / (float)g.cols;
        if (g.cols > SLAB && threadIdx.x == 0) {
          g.stats[2 * row] = sum[0];
          g.stats[2 * row + 1] = sum[1];
        }
      } else {
        sum[0] = g.stats[2 * row];
        sum[1] = g.stats[2 * row + 1];
      }
      const float rstd = sum[0], k = sum[1] * rstd * rstd;
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        const int c = c0 + h * THREADS * W;
        if (c >= g.cols) break;
        rs[h].values(a);
        rd[h].values(b);
#pragma unroll
        for (int i = 0; i < W; ++i) acc[h][i] += b[i] * (a[i] * rstd);
        if (g.dx) {
          load_weight<T, W>(g.w, g.w_f32, c, w);
#pragma unroll
          for (int i = 0; i < W; ++i) a[i] = rstd * (b[i] * w[i] - a[i] * k);
          if (add) {
            re[h].values(b);
#pragma unroll
            for (int i = 0; i < W; ++i) a[i] += b[i];
          }
          store_row<W>(static_cast<T*>(g.dx) + row * g.lddx + c, a);
        }
      }
    }
    if (g.partial) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        const int c = c0 + h * THREADS * W;
        if (c >= g.cols) break;
#pragma unroll
        for (int i = 0; i < W; ++i) g.partial[(int64_t)blockIdx.x * g.cols + c + i] = acc[h][i];
      }
    }
    __syncthreads();  // stats[] of the first slab, written by one thread
  }
}

// dweight[c] = the sum of the blocks' partial sums in a fixed order: 32 warps
// take every 32nd of them, 32 columns a block.
template <typename TW>
__global__ void __launch_bounds__(1024) norm_dweight_kernel(const float* partial, int blocks, int cols, TW* dweight) {
  __shared__ float sums[32][33];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += 32) sum += partial[(int64_t)b * cols + c];
  }
  sums[warp][lane] = sum;
  __syncthreads();
  sum = sums[lane][warp];  // column `warp`, the sum of warp `lane`
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (lane == 0 && blockIdx.x * 32 + warp < cols) dweight[blockIdx.x * 32 + warp] = from_float<TW>(sum);
}

constexpr int kMaxBlocks = 1024;  // of the backward kernel, as the workspace is sized

// Threads of a block by the runs of a row, and the blocks that an SM holds.
template <typename T, int W>
int launch_backward(const GradArgs& g, int sms, int* blocks, cudaStream_t stream) {
  const int64_t runs = (g.cols + W - 1) / W;
  // (F32 rows: registers for half as many runs, and not for the next row's.)
  constexpr bool F32 = sizeof(T) == 4;
  auto kern = norm_backward_kernel<T, W, F32 ? 2 : 4, 512, false>;
  int threads = 512;
  if (runs <= 128) kern = norm_backward_kernel<T, W, 1, 128, true>, threads = 128;
  else if (runs <= 256) kern = norm_backward_kernel<T, W, 1, 256, true>, threads = 256;
  else if (runs <= 512) kern = norm_backward_kernel<T, W, 2, 256, true>, threads = 256;
  else if (runs <= 1024) kern = norm_backward_kernel<T, W, 2, 512, !F32>;
  *blocks = (int)std::min<int64_t>({g.rows, kMaxBlocks, (int64_t)sms * (512 / threads)});
  PdlLaunch l(dim3(*blocks), dim3(threads), 0, stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward launch");
}

int check_norm(const char* what, int dtype, int weight_dtype, int64_t rows, int64_t cols, float eps) {
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16 && dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": only F16, BF16 and F32 are implemented");
  if (weight_dtype != dtype && weight_dtype != KEBAB_F32)
    return fail(KEBAB_ENOTSUP, std::string(what) + ": the weight is of the rows' type or F32");
  if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > (1 << 30))
    return fail(KEBAB_EINVAL, std::string(what) + ": invalid dimensions rows=" + std::to_string(rows) +
                                  " cols=" + std::to_string(cols));
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(KEBAB_EINVAL, std::string(what) + ": eps must be finite and not negative");
  return KEBAB_OK;
}

int check_ld(const char* what, const char* name, int64_t ld, int64_t cols) {
  if (ld >= cols) return KEBAB_OK;
  return fail(KEBAB_EINVAL, std::string(what) + ": row pitch of " + name + " (" + std::to_string(ld) +
                                ") is below the row length (" + std::to_string(cols) + ")");
}

// Whether rows from `p` on at a pitch of `ld` start on boundaries of `bytes`.
bool aligned(const void* p, int64_t ld, int es, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0 && ld * es % bytes == 0;
}

int size_of(int dtype) { return dtype == KEBAB_F32 ? 4 : 2; }

int forward(const char* what, int dtype, int weight_dtype, NormArgs g, bool i8, kebab_stream_t stream) {
  int rc;
  if ((rc = check_norm(what, dtype, weight_dtype, g.rows, g.cols, g.eps)) || (rc = check_ld(what, "x", g.ldx, g.cols)))
    return rc;
  if (g.r && ((rc = check_ld(what, "residual", g.ldr, g.cols)) || (rc = check_ld(what, "s", g.lds, g.cols)))) return rc;
  if ((g.y || !i8) && (rc = check_ld(what, "y", g.ldy, g.cols))) return rc;
  if (i8 && (rc = check_ld(what, "q", g.ldq, g.cols))) return rc;
  if (g.rows == 0) return KEBAB_OK;
  if (!g.x || !g.w || (g.r && !g.s) || (i8 ? !g.q || !g.scale : !g.y))
    return fail(KEBAB_EINVAL, std::string(what) + ": null pointer");
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  g.w_f32 = weight_dtype == KEBAB_F32;
  const int es = size_of(dtype);
  const bool vec = g.cols % 8 == 0 && aligned(g.x, g.ldx, es, 16) && aligned(g.w, 0, 1, 16) &&
                   (!g.r || (aligned(g.r, g.ldr, es, 16) && aligned(g.s, g.lds, es, 16))) &&
                   (!g.y || aligned(g.y, g.ldy, es, 16)) && (!i8 || aligned(g.q, g.ldq, 1, 8));
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int sms = dev->sm_count;
  auto run = [&](auto t) {
    using T = decltype(t);
    if (i8) return vec ? launch_forward<T, 8, true>(g, sms, st) : launch_forward<T, 1, true>(g, sms, st);
    return vec ? launch_forward<T, 8, false>(g, sms, st) : launch_forward<T, 1, false>(g, sms, st);
  };
  return dtype == KEBAB_F16 ? run(__half()) : dtype == KEBAB_BF16 ? run(__nv_bfloat16()) : run(0.f);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int kebab_rms_norm(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                   int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                   int64_t rows, int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    if (cols > (1 << 30)) return check_norm("rms_norm", dtype, weight_dtype, rows, cols, eps);
    NormArgs g = {};
    g.x = x, g.ldx = ldx, g.r = residual, g.ldr = ldr, g.w = weight, g.eps = eps, g.s = s, g.lds = lds;
    g.y = y, g.ldy = ldy, g.rows = rows, g.cols = (int)cols;
    return forward("rms_norm", dtype, weight_dtype, g, false, stream);
  });
}

int kebab_rms_norm_i8(kebab_dtype dtype, kebab_dtype weight_dtype, const void* x, int64_t ldx, const void* residual,
                      int64_t ldr, const void* weight, float eps, void* s, int64_t lds, void* y, int64_t ldy,
                      int8_t* q, int64_t ldq, float* scale, int64_t rows, int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    if (cols > (1 << 30)) return check_norm("rms_norm_i8", dtype, weight_dtype, rows, cols, eps);
    NormArgs g = {};
    g.x = x, g.ldx = ldx, g.r = residual, g.ldr = ldr, g.w = weight, g.eps = eps, g.s = s, g.lds = lds;
    g.y = y, g.ldy = ldy, g.q = q, g.ldq = ldq, g.scale = scale, g.rows = rows, g.cols = (int)cols;
    return forward("rms_norm_i8", dtype, weight_dtype, g, true, stream);
  });
}

// The rows' two sums, then the blocks' sums of dweight.
int64_t kebab_rms_norm_backward_workspace(int64_t rows, int64_t cols) {
  if (rows < 0 || cols <= 0 || rows > INT32_MAX || cols > (1 << 30)) return -KEBAB_EINVAL;
  return (rows * 8 + 15) / 16 * 16 + std::min<int64_t>(rows, kMaxBlocks) * cols * 4;
}

int kebab_rms_norm_backward(kebab_dtype dtype, kebab_dtype weight_dtype, const void* dy, int64_t lddy, const void* s,
                            int64_t lds, const void* weight, float eps, const void* ds, int64_t ldds, void* dx,
                            int64_t lddx, void* dweight, void* workspace, int64_t workspace_bytes, int64_t rows,
                            int64_t cols, kebab_stream_t stream) {
  return guarded([&] {
    const char* what = "rms_norm_backward";
    int rc;
    if ((rc = check_norm(what, dtype, weight_dtype, rows, cols, eps)) || (rc = check_ld(what, "dy", lddy, cols)) ||
        (rc = check_ld(what, "s", lds, cols)) || (ds && (rc = check_ld(what, "ds", ldds, cols))) ||
        (dx && (rc = check_ld(what, "dx", lddx, cols))))
      return rc;
    const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (rows == 0) {
      if (!dweight) return KEBAB_OK;
      const cudaError_t e = cudaMemsetAsync(dweight, 0, cols * size_of(weight_dtype), st);
      return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward memset");
    }
    if (!dy || !s || !weight) return fail(KEBAB_EINVAL, "rms_norm_backward: null pointer");
    if (!dx && !dweight) return KEBAB_OK;
    if (!workspace || workspace_bytes < kebab_rms_norm_backward_workspace(rows, cols) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u))
      return fail(KEBAB_EINVAL, "rms_norm_backward: the workspace is null, too small or not 16-byte aligned");
    DeviceInfo* dev = nullptr;
    if ((rc = device_info(&dev))) return rc;
    GradArgs g = {};
    g.dy = dy, g.lddy = lddy, g.s = s, g.lds = lds, g.w = weight, g.w_f32 = weight_dtype == KEBAB_F32, g.eps = eps;
    g.ds = ds, g.ldds = ldds, g.dx = dx, g.lddx = lddx, g.rows = rows, g.cols = (int)cols;
    g.stats = static_cast<float*>(workspace);
    float* partial = g.stats + (rows * 8 + 15) / 16 * 4;
    g.partial = dweight ? partial : nullptr;
    const int es = size_of(dtype);
    const bool vec = cols % 8 == 0 && aligned(dy, lddy, es, 16) && aligned(s, lds, es, 16) &&
                     aligned(weight, 0, 1, 16) && (!ds || aligned(ds, ldds, es, 16)) &&
                     (!dx || aligned(dx, lddx, es, 16));
    int blocks = 0;
    auto run = [&](auto t) {
      using T = decltype(t);
      return vec ? launch_backward<T, 8>(g, dev->sm_count, &blocks, st) : launch_backward<T, 1>(g, dev->sm_count, &blocks, st);
    };
    rc = dtype == KEBAB_F16 ? run(__half()) : dtype == KEBAB_BF16 ? run(__nv_bfloat16()) : run(0.f);
    if (rc || !dweight) return rc;
    PdlLaunch l(dim3((unsigned)((cols + 31) / 32)), dim3(1024), 0, st);
    cudaError_t e;
    if (weight_dtype == KEBAB_F16) e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<__half>, (const float*)partial, blocks, (int)cols, static_cast<__half*>(dweight));
    else if (weight_dtype == KEBAB_BF16) e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<__nv_bfloat16>, (const float*)partial, blocks, (int)cols, static_cast<__nv_bfloat16*>(dweight));
    else e = cudaLaunchKernelEx(&l.cfg, norm_dweight_kernel<float>, (const float*)partial, blocks, (int)cols, static_cast<float*>(dweight));
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward: dweight launch");
  });
}

}  // extern "C"
