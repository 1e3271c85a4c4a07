// 8-bit integer products, dense and grouped, of operands that TMA cannot address
// (base addresses or row pitches that are no multiples of 16 bytes).
//
// A CTA multiplies 128 weight rows n (the MMA's row side, so that a lane of TMEM
// is a column of Y) with up to 128 rows of a group. All threads copy: 16 bytes of
// a row are cut from two aligned granules (selects and four funnel shifts) and
// stored where TMA would place them; the next K-block's are in flight while this
// one's are multiplied. Pieces whose granules reach past an operand's ends are
// copied byte by byte, and bytes past K are zeros. Sums are exact in 32 bits, so
// that the results are those of the other 8-bit kernels. Bound by the copies'
// instructions, with few warps to hide their latency: 1 row of 4096 x 4100 38 us,
// 4096 rows 205, 4093 x 1024 x 1000 26; rows on 16 bytes, by TMA, take 6, 64 and
// 11. (Pieces away from an operand's ends take a path without conditions: with one
// for each, 68, 327 and 30.) All threads look for the block's group together: 1021
// rows of 1024 experts, 512 x 301, 111 us (one after the other 1637), of 256
// experts, 1024 x 1001, 112 (255).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "gemm_umma.cuh"
#include "group_search.cuh"
#include "grouped.h"
#include "vec.cuh"

namespace kb {
namespace {
constexpr int THREADS = 256, TILE = 128, BLOCK = TILE * 128;  // bytes of an operand's K-block
constexpr int STAGES = 2, TASKS = 8;                          // 16-byte pieces that a thread copies a K-block
// More than a third of an SM's: no more than two CTAs that allocate TMEM share one.
constexpr int SMEM = 83 * 1024;
static_assert(BLOCK == 4 * 32 * 128, "the second operand's rows follow the first's");
static_assert(STAGES * 2 * BLOCK + 1024 <= SMEM, "the stages fit");

struct Operand {
  const uint8_t* base;
  const uint8_t* end;  // past its last byte
  int64_t pitch, stride;
};

struct AnyArgs {
  Operand w, x;
  const int32_t* offsets;
  int E, R, N, K, n_tiles;
  void* Y;
  int64_t ldy;
  const float* scale;
  const float* w_scale;
  const void* bias;
  int pdl;
  WaitCtx ctx;
};

// 16 bytes of a row on any boundary: the two granules that hold them.
struct Piece {
  uint4 a, b;
};

__device__ __forceinline__ uint4 piece_bytes(const Piece& p, uint32_t off) {
  uint32_t w[8] = {p.a.x, p.a.y, p.a.z, p.a.w, p.b.x, p.b.y, p.b.z, p.b.w}, v[4];
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = off & 8u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = off & 4u ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __funnelshift_r(w[i], w[i + 1], (off & 3u) * 8u);
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename TO>
__global__ void __launch_bounds__(THREADS, 2) grouped_i8_any_kernel(const AnyArgs g) {
  if (g.pdl) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const int n0 = (int)(blockIdx.x % g.n_tiles) * TILE;
  int e, begin, rows;
  if (!nth_share<THREADS, TILE>(g.offsets, g.E, g.R, (int)(blockIdx.x / g.n_tiles), e, begin, rows)) return;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t done[STAGES];
  __shared__ uint32_t tmem_slot;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&done[s], 1);
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc<1>(&tmem_slot, TILE);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // Pieces of this thread: rows r, r + 32, .. of both operands, the same 16 bytes
  // of a K-block of each, from the granule on that `row` points at (its offset in
  // `offs`, 4 bits each). Past the last row it is the last row again, whose results
  // are not used. `free`: rows whose granules lie in the operand wherever in the row.
  const int r0 = threadIdx.x >> 3, part = (threadIdx.x & 7) * 16;
  const uint8_t* row[TASKS];
  uint32_t offs = 0, free = 0;
#pragma unroll
  for (int u = 0; u < TASKS; ++u) {
    const Operand& o = u < 4 ? g.w : g.x;
    const int r = r0 + 32 * (u & 3);
    const int64_t at = u < 4 ? min(n0 + r, g.N - 1) : begin + min(r, rows - 1);
    row[u] = o.base + e * o.stride + at * o.pitch;
    if (row[u] - 15 >= o.base && row[u] + g.K + 15 <= o.end) free |= 1u << u;
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row[u]) & 15u;
    offs |= off << (4 * u);
    row[u] += part - (int)off;
  }
  auto off_of = [&](int u) { return offs >> (4 * u) & 15u; };
  // Whether all pieces at k lie within their rows with both granules; and, where
  // not, whether the granules that hold a piece's bytes lie in the operand. (What
  // does not is copied byte by byte.)
  auto inner = [&](int k) { return k > 0 && k + 32 <= g.K; };
  auto by_granules = [&](int u, int k) {
    return (free >> u & 1u) || (k > 0 && k + 31 <= g.K) || (off_of(u) == 0 && k + 16 <= g.K);
  };
  Piece next[TASKS];
  auto load = [&](int kb) {
    const int k = kb * 128 + part;
    if (inner(k)) {
#pragma unroll
      for (int u = 0; u < TASKS; ++u) {
        const uint4* from = reinterpret_cast<const uint4*>(row[u] + kb * 128);
        next[u].a = from[0];
        next[u].b = from[1];
      }
    } else {
      const int valid = min(16, g.K - k);
#pragma unroll
      for (int u = 0; u < TASKS; ++u) {
        const uint4* from = reinterpret_cast<const uint4*>(row[u] + kb * 128);
        const bool in = valid > 0 && by_granules(u, k);
        next[u].a = next[u].b = make_uint4(0, 0, 0, 0);
        if (in) next[u].a = from[0];
        if (in && valid > 16 - (int)off_of(u)) next[u].b = from[1];
      }
    }
  };
  const int blocks = (g.K + 127) / 128;
  const uint32_t idesc = umma_idesc_i8(128, (rows + 15) / 16 * 16);
  bool ok = true;
  load(0);
  for (int kb = 0; kb < blocks; ++kb) {
    const int s = kb % STAGES;
    if (kb >= STAGES) ok = mbar_wait(&done[s], kb / STAGES - 1 & 1, g.ctx, SITE_EMPTY);
    uint8_t* stage = smem + s * 2 * BLOCK;
    if (ok) {
      const int k = kb * 128 + part, valid = max(0, min(16, g.K - k));
      // (Rows of a thread are 32 apart: the same place in the swizzle.)
      uint8_t* to = stage + r0 * 128 + (((part >> 4) ^ (r0 & 7)) << 4);
      if (inner(k)) {
#pragma unroll
        for (int u = 0; u < TASKS; ++u) *reinterpret_cast<uint4*>(to + u * 32 * 128) = piece_bytes(next[u], off_of(u));
      } else {
#pragma unroll
        for (int u = 0; u < TASKS; ++u, to += 32 * 128) {
          uint4 v = piece_bytes(next[u], off_of(u));
          auto keep = [&](int i) { return valid >= 4 * i + 4 ? ~0u : valid <= 4 * i ? 0u : (1u << (8 * (valid - 4 * i))) - 1u; };
          v.x &= keep(0), v.y &= keep(1), v.z &= keep(2), v.w &= keep(3);  // zeros past K
          *reinterpret_cast<uint4*>(to) = v;
          if (by_granules(u, k)) continue;
          const uint8_t* src = row[u] + kb * 128 + off_of(u);
#pragma unroll 1
          for (int b = 0; b < valid; b += 8) {
            uint8_t t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = b + i < valid ? src[b + i] : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[b + i] = t[i];
          }
        }
      }
      if (kb + 1 < blocks) load(kb + 1);
    }
    fence_proxy_async_smem();
    if (!__syncthreads_and(ok)) {
      ok = false;
      break;
    }
    if (warp == 0) {
      tc_fence_after();
      const uint32_t at = smem_u32(stage);
      const uint64_t a = umma_desc_sw128(at), b = umma_desc_sw128(at + BLOCK);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_i8<1>(tmem, a + k * 2, b + k * 2, idesc, kb == 0 && k == 0 ? 0u : 1u);
        umma_commit_cg1(&done[s]);
      }
      __syncwarp();
    }
  }
  if (ok) ok = mbar_wait(&done[(blocks - 1) % STAGES], (blocks - 1) / STAGES & 1, g.ctx, SITE_TMEM_FULL);
  ok = __all_sync(0xffffffffu, ok) != 0;
  tc_fence_after();

  // Two warps a quarter of the lanes, half of the columns each.
  const int q = warp & 3, n = n0 + q * 32 + lane;
  const bool mine = ok && n < g.N;
  const float sw = mine ? g.w_scale[(int64_t)e * g.N + n] : 0.f;
  const float bias = mine && g.bias ? to_float(static_cast<const TO*>(g.bias)[n]) : 0.f;
  TO* y = static_cast<TO*>(g.Y) + (int64_t)begin * g.ldy + n;
#pragma unroll 1
  for (int c = warp / 4 * 16; ok && c < rows; c += 32) {
    uint32_t v[16];
    tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (!mine || c + j >= rows) continue;
      const float o = (float)(int)v[j] * (sw * g.scale[begin + c + j]) + bias;
      y[(int64_t)(c + j) * g.ldy] = from_float<TO>(o);
    }
  }
  __syncwarp();
  tc_fence_before();
  if (__syncthreads_or(!ok)) settle();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, TILE);
  }
}

template <typename TO>
int launch(const GroupedProblem& p) {
  int rc;
  DeviceInfo* dev = nullptr;
  AnyArgs g = {};
  if ((rc = device_info(&dev)) || (rc = wait_ctx(&g.ctx))) return rc;
  const uint8_t* w = static_cast<const uint8_t*>(p.W);
  const uint8_t* x = static_cast<const uint8_t*>(p.X);
  const int64_t stride = p.E > 1 ? p.w_stride : 0;
  g.w = {w, w + (p.E - 1) * stride + (p.N - 1) * p.ldw + p.K, p.ldw, stride};
  g.x = {x, x + (p.R - 1) * p.ldx + p.K, p.ldx, 0};
  g.offsets = p.offsets;
  g.E = (int)p.E, g.R = (int)p.R, g.N = (int)p.N, g.K = (int)p.K;
  g.n_tiles = (int)((p.N + TILE - 1) / TILE);
  g.Y = p.Y, g.ldy = p.ldy, g.scale = p.scale, g.w_scale = p.w_scale, g.bias = p.bias;
  g.pdl = pdl_enabled();
  const int64_t tiles = g.n_tiles * (p.offsets ? p.R / TILE + std::min(p.E, p.R) : (p.R + TILE - 1) / TILE);
  if (tiles > INT32_MAX) return fail(KEBAB_EINVAL, "grouped product: too many tiles");
  auto kern = grouped_i8_any_kernel<TO>;
  static std::once_flag once[64];
  static cudaError_t err[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] { err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM); });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  PdlLaunch l(dim3((unsigned)tiles), dim3(THREADS), SMEM, p.stream);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, (const AnyArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "8-bit product launch");
}
}  // namespace

int launch_grouped_i8_any(const GroupedProblem& p) {
  return p.out == KEBAB_F16 ? launch<__half>(p) : launch<__nv_bfloat16>(p);
}

}  // namespace kb
