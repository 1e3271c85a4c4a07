// Root-mean-square norm with the residual's addition, its form with 8-bit
// output, and its gradients: the kernels and their choice for one type of rows
// (norm_f16.cu and its neighbours).
//
// Forward: ROW threads take a row, read it once (x and the residual), keep the
// sum in registers as it is stored, and find the sum of squares (and, for 8
// bits, the largest |s w|) by shuffles and shared memory. Longer rows than the
// registers hold are read a second time, from L2. Bound by memory for many rows
// (16381 x 4096 BF16 with a residual 77 us, 6.9 TB/s) and by latency for few: a
// row then has 1024 threads (1 x 8192 2.6 us).
//
// Backward: a block takes every gridDim-th row (or group of short rows). A thread
// has the same columns of all of them, so that its share of dweight and its
// weights stay in registers; the blocks' sums are added in a fixed order by a
// second, small kernel (16381 x 4096 BF16 with ds 105 us, 5.1 TB/s, and 4 us for
// the sums; with 512 threads a row and two blocks an SM 130). Longer rows than a
// block's registers hold are taken in slabs of columns: the first slab's pass also
// finds the row's two sums (over all columns) and leaves them in the workspace.
//
// Rows that do not start on 16 bytes (SHIFT): a thread takes the eight columns
// of a 16-byte granule, c0 = 8 j - off for a row that starts `off` values into
// its first granule; the first and the last granule are taken value by value. In
// the backward pass a thread's rows are a multiple of 8 apart, so that they have
// the same `off` (16381 x 8191 with ds 372 us, 2.9 TB/s). Rows of several
// tensors that start differently take one value a step.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "grouped.h"
#include "norm.h"
#include "quant_i8.cuh"

namespace kb {
namespace {

// W weights from column c on, which may reach past the row's ends.
template <typename T, int W, bool SHIFT>
__device__ __forceinline__ void load_weight(const void* w, int w_f32, int c, int cols, float (&v)[W]) {
  if constexpr (SHIFT) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const bool in = c + i >= 0 && c + i < cols;
      if (sizeof(T) == 4 || w_f32) v[i] = in ? static_cast<const float*>(w)[c + i] : 0.f;
      else v[i] = in ? to_float(static_cast<const T*>(w)[c + i]) : 0.f;
    }
  } else {
    if (sizeof(T) == 4 || w_f32) load_row<W>(static_cast<const float*>(w) + c, v);
    else load_row<W>(static_cast<const T*>(w) + c, v);
  }
}

// W values of a row from column c on. A granule across the row's ends is loaded
// whole, and with it the neighbouring rows' values (`inner`: rows with seven
// neighbours on both sides in the tensor, as a granule may reach over seven rows
// of one value); row_values makes zeros of them.
template <typename T, int W, bool SHIFT>
__device__ __forceinline__ void load_run(const T* row, int c, int cols, bool inner, Run<T, W>& run) {
  if (!SHIFT || inner || (c >= 0 && c + W <= cols)) {
    run.load(row + c);
  } else {
    float v[W];
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = c + i >= 0 && c + i < cols ? to_float(row[c + i]) : 0.f;
    run.set(v);
  }
}
template <typename T, int W, bool SHIFT>
__device__ __forceinline__ void row_values(const Run<T, W>& run, int c, int cols, float (&v)[W]) {
  run.values(v);
  if (SHIFT && (c < 0 || c + W > cols)) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (c + i < 0 || c + i >= cols) v[i] = 0.f;
  }
}

// Places past the row's ends are not written.
template <typename T, int W, bool SHIFT>
__device__ __forceinline__ void store_run(T* row, int c, int cols, const float (&v)[W]) {
  if (!SHIFT || (c >= 0 && c + W <= cols)) {
    store_row<W>(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (c + i >= 0 && c + i < cols) row[c + i] = from_float<T>(v[i]);
  }
}
// Values of a 16-byte granule before the row's first.
template <typename T, bool SHIFT>
__device__ __forceinline__ int row_offset(const T* row) {
  return SHIFT ? (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T)) : 0;
}

// Sums of N values over the ROW threads of a row: part of a warp, a warp, or all
// of a block (`part`: N floats a warp).
template <int ROW, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float (*part)[N]) {
#pragma unroll
  for (int d = ROW < 32 ? ROW / 2 : 16; d; d >>= 1) {
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

// The largest of a value over the same threads, before row_sum's barrier (in
// `tops`) and after it.
template <int ROW>
__device__ __forceinline__ uint32_t warp_top(uint32_t top, uint32_t* tops) {
#pragma unroll
  for (int d = ROW < 32 ? ROW / 2 : 16; d; d >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (ROW > 32 && (threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  return top;
}
template <int ROW>
__device__ __forceinline__ uint32_t row_top(uint32_t top, const uint32_t* tops) {
  if constexpr (ROW > 32) {
    const int lane = threadIdx.x & 31;
    top = __reduce_max_sync(0xffffffffu, lane < ROW / 32 ? tops[lane] : 0u);
  }
  return top;
}

// What is in flight is what the resident blocks have loaded: for 8 bits (less to
// load a row, and more to keep) registers are held down to fit four or more.
template <typename T, int W, int HELD, int ROW, bool I8, bool SHIFT>
__global__ void __launch_bounds__(ROW < 128 ? 128 : ROW, I8 && sizeof(T) == 2 && ROW <= 256 ? (HELD > 4 ? 768 : 1024) / (ROW < 128 ? 128 : ROW) : 1)
    norm_kernel(const NormArgs g) {
  constexpr int PER_BLOCK = (ROW < 128 ? 128 : ROW) / ROW;
  __shared__ float part[32][1];
  __shared__ uint32_t tops[32];
  pdl_wait();
  pdl_launch_dependents();
  const int64_t row = (int64_t)blockIdx.x * PER_BLOCK + threadIdx.x / ROW;
  const int cols = row < g.rows ? g.cols : -8;  // before every granule: nothing is read or written
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  const T* r = static_cast<const T*>(g.r) + row * g.ldr;
  T* s = static_cast<T*>(g.s) + row * g.lds;
  const bool add = g.r != nullptr;
  const int c0 = threadIdx.x % ROW * W - row_offset<T, SHIFT>(x);
  const bool inner = row >= 7 && row + 7 < g.rows;
  Run<T, W> held[HELD], other[HELD];
  float v[W], u[W], sum[1] = {0.f};
  uint32_t top = 0;
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = c0 + h * ROW * W;
    if (c < cols) {
      load_run<T, W, SHIFT>(x, c, cols, inner, held[h]);
      if (add) load_run<T, W, SHIFT>(r, c, cols, inner, other[h]);
    }
  }
  // The stored sum of the run's columns in v; squares, and largest products with the weight.
  auto take = [&](Run<T, W>& a, const Run<T, W>& b, int c) {
    row_values<T, W, SHIFT>(a, c, cols, v);
    if (add) {
      row_values<T, W, SHIFT>(b, c, cols, u);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] += u[i];
      a.set(v);
      a.values(v);
      store_run<T, W, SHIFT>(s, c, cols, v);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) sum[0] += v[i] * v[i];
    if constexpr (I8) {
      load_weight<T, W, SHIFT>(g.w, g.w_f32, c, cols, u);
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] *= u[i];
      top = largest<W>(v, top);
    }
  };
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = c0 + h * ROW * W;
    if (c >= cols) break;
    take(held[h], other[h], c);
  }
  for (int c = c0 + HELD * ROW * W; c < cols; c += ROW * W) {
    Run<T, W> a, b;
    load_run<T, W, SHIFT>(x, c, cols, inner, a);
    if (add) load_run<T, W, SHIFT>(r, c, cols, inner, b);
    take(a, b, c);
  }
  if constexpr (I8) top = warp_top<ROW>(top, tops);
  row_sum<ROW, 1>(sum, part);
  const float rstd = rsqrtf(sum[0] / (float)g.cols + g.eps);
  // Codes: s w 127 / max |s w|, in which rstd cancels.
  RowScale code = {0.f, 0.f};
  if constexpr (I8) {
    code = row_scale(row_top<ROW>(top, tops));
    if (threadIdx.x % ROW == 0 && row < g.rows) g.scale[row] = code.scale * rstd;
  }
  T* y = static_cast<T*>(g.y) + row * g.ldy;
  auto give = [&](const Run<T, W>& a, int c) {
    load_weight<T, W, SHIFT>(g.w, g.w_f32, c, cols, u);
    a.values(v);  // (what is outside the row is not written)
    if (!I8 || g.y) {
      float o[W];
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = v[i] * rstd * u[i];
      store_run<T, W, SHIFT>(y, c, cols, o);
    }
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] *= u[i];
      store_codes<W>(g.q + row * g.ldq + c, v, code.inv);
    }
  };
#pragma unroll
  for (int h = 0; h < HELD; ++h) {
    const int c = c0 + h * ROW * W;
    if (c >= cols) break;
    give(held[h], c);
  }
  const T* again = add ? s : x;  // the columns past the registers, which this thread wrote
  for (int c = c0 + HELD * ROW * W; c < cols; c += ROW * W) {
    Run<T, W> a;
    load_run<T, W, SHIFT>(again, c, cols, inner, a);
    give(a, c);
  }
}

template <typename T, int W, bool I8, bool SHIFT>
int launch_forward(const NormArgs& g, int sms, cudaStream_t stream) {
  const int64_t runs = (g.cols + W - 1) / W + SHIFT;
  auto run = [&](auto kern, int row) {
    const int threads = std::max(row, 128), per_block = threads / row;
    PdlLaunch l(dim3((unsigned)((g.rows + per_block - 1) / per_block)), dim3(threads), 0, stream);
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm launch");
  };
  if constexpr (W == 1) {
    // What the registers hold is read once (4093 x 8191 to 8 bits with 256 threads: 168 us; 1024 112).
    return g.cols <= 2048 ? run(norm_kernel<T, W, 8, 256, I8, SHIFT>, 256) : run(norm_kernel<T, W, 8, 1024, I8, SHIFT>, 1024);
  } else {
    // Few rows: 1024 threads a row (1 x 4096 to 8 bits 8 us, with 128 threads 10,
    // flushed and with the launch; 592 rows 14 against 10). Many short rows: 8 to 32
    // lanes a row (65536 x 64 10 us, with 128 threads 74).
    if (g.rows <= 2 * sms && runs > 256)
      return runs <= 1024 ? run(norm_kernel<T, W, 1, 1024, I8, SHIFT>, 1024) : run(norm_kernel<T, W, 2, 1024, I8, SHIFT>, 1024);
    if (g.rows >= 1024 && runs <= 128) {
      if (runs <= 8) return run(norm_kernel<T, W, 1, 8, I8, SHIFT>, 8);
      if (runs <= 16) return run(norm_kernel<T, W, 1, 16, I8, SHIFT>, 16);
      if (runs <= 32) return run(norm_kernel<T, W, 1, 32, I8, SHIFT>, 32);
      if (runs <= 64) return run(norm_kernel<T, W, 2, 32, I8, SHIFT>, 32);
      return run(norm_kernel<T, W, 4, 32, I8, SHIFT>, 32);
    }
    if (runs <= 128) return run(norm_kernel<T, W, 1, 128, I8, SHIFT>, 128);
    if (runs <= 256) return run(norm_kernel<T, W, 2, 128, I8, SHIFT>, 128);
    if (runs <= 512) return run(norm_kernel<T, W, 4, 128, I8, SHIFT>, 128);
    if (runs <= 1024) return run(norm_kernel<T, W, 4, 256, I8, SHIFT>, 256);
    // (4093 x 8200 with 8 runs a thread, for 8 bits 512 threads: 51 us, 83; with 5 43, 48.)
    if (runs <= 1280) return run(norm_kernel<T, W, 5, 256, I8, SHIFT>, 256);
    return run(norm_kernel<T, W, I8 ? 4 : 8, I8 ? 512 : 256, I8, SHIFT>, I8 ? 512 : 256);
  }
}

// AHEAD: the next row of a slab is loaded before the sums of this one are
// exchanged. KEEP: a slab's weights stay in registers. (Where those hold them.)
template <typename T, int W, int HELD, int ROW, bool SHIFT, bool AHEAD, bool KEEP>
__global__ void __launch_bounds__(ROW < 256 && ROW > 32 ? ROW : ROW <= 32 ? 256 : ROW, 512 / (ROW <= 32 ? 256 : ROW))
    norm_backward_kernel(const GradArgs g) {
  constexpr int THREADS = ROW <= 32 ? 256 : ROW, GROUPS = THREADS / ROW;  // rows at a time
  constexpr int SLAB = ROW * W * HELD;
  __shared__ float part[2][THREADS / 32][2];
  __shared__ float sums[GROUPS > 1 ? GROUPS * SLAB : 1];
  pdl_wait();
  pdl_launch_dependents();
  const bool add = g.ds && g.dx;
  const int group = threadIdx.x / ROW;
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group, step = (int64_t)gridDim.x * GROUPS;
  const int off = row_offset<T, SHIFT>(static_cast<const T*>(g.s) + first * g.lds);
  const int end = g.cols + (SHIFT ? 7 : 0);  // granules may begin before the first column
  int turn = 0;
  for (int base = 0; base < end; base += SLAB) {
    const int c0 = base + threadIdx.x % ROW * W - off;
    float acc[HELD][W], weight[KEEP ? HELD : 1][W];
#pragma unroll
    for (int h = 0; h < HELD; ++h)
#pragma unroll
      for (int i = 0; i < W; ++i) acc[h][i] = 0.f;
    if constexpr (KEEP) {
#pragma unroll
      for (int h = 0; h < HELD; ++h)
        if (c0 + h * ROW * W < g.cols) load_weight<T, W, SHIFT>(g.w, g.w_f32, c0 + h * ROW * W, g.cols, weight[h]);
    }
    Run<T, W> rs[HELD], rd[HELD], re[HELD], ns[HELD], nd[HELD], ne[HELD];
    auto load = [&](int64_t row, Run<T, W> (&ls)[HELD], Run<T, W> (&ld)[HELD], Run<T, W> (&le)[HELD]) {
      if (row >= g.rows) return;
      const bool inner = row >= 7 && row + 7 < g.rows;
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        const int c = c0 + h * ROW * W;
        if (c < g.cols) {
          load_run<T, W, SHIFT>(static_cast<const T*>(g.s) + row * g.lds, c, g.cols, inner, ls[h]);
          load_run<T, W, SHIFT>(static_cast<const T*>(g.dy) + row * g.lddy, c, g.cols, inner, ld[h]);
          if (add) load_run<T, W, SHIFT>(static_cast<const T*>(g.ds) + row * g.ldds, c, g.cols, inner, le[h]);
        }
      }
    };
    if (AHEAD) load(first, ns, nd, ne);
    // Groups of a warp go round together: the shuffles need all lanes.
    for (int64_t row = first; row - group < g.rows; row += step) {
      const int cols = row < g.rows ? g.cols : -8;  // before every granule
      if (AHEAD) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) rs[h] = ns[h], rd[h] = nd[h], re[h] = ne[h];
        load(row + step, ns, nd, ne);
      } else {
        load(row, rs, rd, re);
      }
      float a[W], b[W], w[W], sum[2] = {0.f, 0.f};
      auto weights = [&](int h, int c) {
        if constexpr (KEEP) {
#pragma unroll
          for (int i = 0; i < W; ++i) w[i] = weight[h][i];
        } else {
          load_weight<T, W, SHIFT>(g.w, g.w_f32, c, g.cols, w);
        }
      };
      auto count = [&] {
#pragma unroll
        for (int i = 0; i < W; ++i) {
          sum[0] += a[i] * a[i];
          sum[1] += b[i] * w[i] * a[i];
        }
      };
      if (base == 0) {
#pragma unroll
        for (int h = 0; h < HELD; ++h) {
          const int c = c0 + h * ROW * W;
          if (c >= cols) break;
          row_values<T, W, SHIFT>(rs[h], c, cols, a);
          row_values<T, W, SHIFT>(rd[h], c, cols, b);
          weights(h, c);
          count();
        }
        for (int c = c0 + SLAB; c < cols; c += ROW * W) {
          Run<T, W> s, d;
          load_run<T, W, SHIFT>(static_cast<const T*>(g.s) + row * g.lds, c, cols, false, s);
          load_run<T, W, SHIFT>(static_cast<const T*>(g.dy) + row * g.lddy, c, cols, false, d);
          s.values(a);
          d.values(b);
          load_weight<T, W, SHIFT>(g.w, g.w_f32, c, cols, w);
          count();
        }
        row_sum<ROW, 2>(sum, part[turn]);  // two buffers in turn: one barrier a row
        turn ^= 1;
        sum[0] = rsqrtf(sum[0] / (float)g.cols + g.eps);
        sum[1] = sum[1] / (float)g.cols;
        if (end > SLAB && threadIdx.x % ROW == 0 && row < g.rows) {
          g.stats[2 * row] = sum[0];
          g.stats[2 * row + 1] = sum[1];
        }
      } else if (row < g.rows) {
        sum[0] = g.stats[2 * row];
        sum[1] = g.stats[2 * row + 1];
      }
      const float rstd = sum[0], k = sum[1] * rstd * rstd;
#pragma unroll
      for (int h = 0; h < HELD; ++h) {
        const int c = c0 + h * ROW * W;
        if (c >= cols) break;
        rs[h].values(a);  // (what is outside the row goes nowhere)
        rd[h].values(b);
#pragma unroll
        for (int i = 0; i < W; ++i) acc[h][i] += b[i] * (a[i] * rstd);
        if (g.dx) {
          weights(h, c);
#pragma unroll
          for (int i = 0; i < W; ++i) a[i] = rstd * (b[i] * w[i] - a[i] * k);
          if (add) {
            re[h].values(b);
#pragma unroll
            for (int i = 0; i < W; ++i) a[i] += b[i];
          }
          store_run<T, W, SHIFT>(static_cast<T*>(g.dx) + row * g.lddx, c, cols, a);
        }
      }
    }
    if (g.partial) {
      // By column: the groups' granules may begin at different ones.
      float* to = GROUPS > 1 ? sums + group * SLAB : g.partial + (int64_t)blockIdx.x * g.cols;
#pragma unroll
      for (int h = 0; h < HELD; ++h)
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const int c = c0 + h * ROW * W + i;
          if (c >= 0 && c < g.cols) to[c] = acc[h][i];
        }
      if constexpr (GROUPS > 1) {  // one slab
        __syncthreads();
        for (int c = threadIdx.x; c < g.cols; c += THREADS) {
          float sum = 0.f;
          for (int i = 0; i < GROUPS; ++i) sum += sums[i * SLAB + c];
          g.partial[(int64_t)blockIdx.x * g.cols + c] = sum;
        }
      }
    }
    __syncthreads();  // stats[] of the first slab, written by one thread
  }
}

// Blocks: as many as an SM's 512 threads of each, in multiples of 8 (SHIFT).
template <typename T, int W, bool SHIFT>
int launch_backward(const GradArgs& g, int sms, int* blocks, cudaStream_t stream) {
  const int64_t runs = (g.cols + W - 1) / W + SHIFT;
  auto run = [&](auto kern, int row) {
    const int threads = row <= 32 ? 256 : row, groups = threads / row;
    int64_t n = std::min<int64_t>(kNormMaxBlocks, sms * (512 / threads)) / 8 * 8;
    n = std::min<int64_t>(n, ((g.rows + groups - 1) / groups + 7) / 8 * 8);
    *blocks = (int)n;
    PdlLaunch l(dim3((unsigned)n), dim3(threads), 0, stream);
    const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, g);
    return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "rms_norm_backward launch");
  };
  constexpr bool F32 = sizeof(T) == 4;  // registers for half as many runs
  if constexpr (W == 1) {
    return run(norm_backward_kernel<T, W, 8, 256, SHIFT, false, false>, 256);
  } else {
    if (runs <= 8) return run(norm_backward_kernel<T, W, 1, 8, SHIFT, true, true>, 8);
    if (runs <= 16) return run(norm_backward_kernel<T, W, 1, 16, SHIFT, true, true>, 16);
    if (runs <= 32) return run(norm_backward_kernel<T, W, 1, 32, SHIFT, true, true>, 32);
    if (runs <= 64) return run(norm_backward_kernel<T, W, 2, 32, SHIFT, !F32, true>, 32);
    if (runs <= 128) return run(norm_backward_kernel<T, W, 1, 128, SHIFT, true, true>, 128);
    if (runs <= 256) return run(norm_backward_kernel<T, W, 1, 256, SHIFT, true, true>, 256);
    if (runs <= 512) return run(norm_backward_kernel<T, W, 2, 256, SHIFT, !F32, !F32>, 256);
    if (runs <= 1024) return run(norm_backward_kernel<T, W, 2, 512, SHIFT, !F32, !F32>, 512);
    // (4093 x 8191 with 4 runs, whose weights do not stay: 145 us; with 3 104.)
    if (runs <= 1536 && !F32) return run(norm_backward_kernel<T, W, 3, 512, SHIFT, false, true>, 512);
    return run(norm_backward_kernel<T, W, F32 ? 2 : 4, 512, SHIFT, false, false>, 512);
  }
}

template <typename T>
int run_forward(const NormArgs& g, RowStart start, bool i8, int sms, cudaStream_t st) {
  if (start == RowStart::kAligned)
    return i8 ? launch_forward<T, 8, true, false>(g, sms, st) : launch_forward<T, 8, false, false>(g, sms, st);
  // (Codes have a granule of their own: 8191 wide rows one value a step 110 us, with scattered codes 310.)
  if (start == RowStart::kAlike && !i8) return launch_forward<T, 8, false, true>(g, sms, st);
  return i8 ? launch_forward<T, 1, true, false>(g, sms, st) : launch_forward<T, 1, false, false>(g, sms, st);
}

template <typename T>
int run_backward(const GradArgs& g, RowStart start, int sms, int* blocks, cudaStream_t st) {
  if (start == RowStart::kAligned) return launch_backward<T, 8, false>(g, sms, blocks, st);
  if (start == RowStart::kAlike) return launch_backward<T, 8, true>(g, sms, blocks, st);
  return launch_backward<T, 1, false>(g, sms, blocks, st);
}
}  // namespace
}  // namespace kb
