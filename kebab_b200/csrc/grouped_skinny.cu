// Grouped and 8-bit integer products for few rows, or few tiles, on the tensor
// cores: bound by the weights' bytes, or by how many SMs have work.
//
// A CTA multiplies 128 weight rows n (the MMA's row side, so that a lane of
// TMEM is a column of Y) with up to 128 rows of one group (equal shares of a
// larger group, padded to a multiple of 16). Where that gives too few CTAs, a
// cluster of S of them splits k: each ends with a partial sum in TMEM, sends
// every other CTA the 128 / S of its rows that that one finishes (st.async,
// counted on the receiver's barrier), and adds up its own rows over the S
// partials in rank order. No workspace, no atomics, and the same bits every
// time.
//
// Ring: a stage is two 128-byte K-blocks (256 contiguous bytes a weight row) up
// to 64 rows of X, else one; with one CTA an SM or two, up to 190 KB are in
// flight.
//
// In linear_i8 the kernel before this one only makes the codes and scales of X
// (`early`): the first weights are fetched while it still runs.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "gemm_umma.cuh"
#include "grouped.h"
#include "vec.cuh"

namespace kb {
namespace {
// Warps: copies of W, MMA issuer, 8 epilogue warps, copies of X. The epilogue is
// bound by latency, a warp or two a scheduler: of 256 x 1024 x 8192 int8 (8
// splits) the exchange and the output took 6.1 us with 4 warps, 4.8 with 8.
constexpr int EPI = 8, X_WARP = 2 + EPI, THREADS = 32 * (3 + EPI);
constexpr int SUB = 128 * 128;
constexpr int MAX_STAGES = 8, MAX_WIDTH = 128;

struct SkinnyArgs {
  const int32_t* offsets;
  int E, R, N, K;
  int splits;
  int kps, stages, x_rows;  // K-blocks a stage, stages, rows of X that a stage has room for
  void* Y;
  int64_t ldy;
  const float* scale;
  const float* w_scale;
  const void* bias;
  int early, pdl;
  WaitCtx ctx;
};

// Boxes of 64, 32 and 16 rows of X.
struct RowMaps {
  CUtensorMap box[3];
};

// 16 bytes into a peer's shared memory; the bytes count towards the peer's
// mbarrier (both given as shared::cluster addresses).
__device__ __forceinline__ void send16(uint32_t dst, uint32_t bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(dst),
               "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
               : "memory");
}

// Rows begin .. begin + rows - 1 of group e: the `nth` of the shares (of at most
// MAX_WIDTH rows) of all groups, by all threads of the block; false if there
// are fewer.
__device__ bool nth_share(const SkinnyArgs& g, int nth, int& e, int& begin, int& rows) {
  __shared__ int s_count[THREADS / 32], s_found[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int at = nth;  // the share within its group
  if (g.offsets == nullptr) {
    e = 0;
    begin = 0;
    rows = g.R;
  } else {
    if (threadIdx.x == 0) s_found[0] = -1;
    int before = 0;
    for (int e0 = 0; e0 < g.E; e0 += THREADS) {
      int b = 0, n = 0;
      if (e0 + (int)threadIdx.x < g.E) group_range(g.offsets, e0 + threadIdx.x, g.R, b, n);
      const int shares = (n + MAX_WIDTH - 1) / MAX_WIDTH;
      int sum = shares;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (lane == 31) s_count[warp] = sum;
      __syncthreads();
      int first = before + sum - shares;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) first += s_count[w];
        before += s_count[w];
      }
      if (first <= nth && nth < first + shares) {
        s_found[0] = e0 + threadIdx.x;
        s_found[1] = b;
        s_found[2] = n;
        s_found[3] = nth - first;
      }
      __syncthreads();
      if (before > nth) break;
    }
    e = s_found[0];
    if (e < 0) return false;
    begin = s_found[1];
    rows = s_found[2];
    at = s_found[3];
  }
  const int shares = (rows + MAX_WIDTH - 1) / MAX_WIDTH;
  if (at >= shares) return false;
  const int share = (rows + shares - 1) / shares;
  begin += at * share;
  rows = min(share, rows - at * share);
  return rows > 0;
}

template <typename TO, bool I8, bool RR>
__global__ void __launch_bounds__(THREADS)
    grouped_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ RowMaps tmX,
                          const SkinnyArgs g) {
  constexpr int EPB = I8 ? 128 : 64;
  constexpr uint32_t IDESC = (I8 ? umma_idesc_i8(128, 0) : umma_idesc_f16(128, 0, ElemTraits<TO>::kBf16)) |
                             (RR ? (1u << 15) : 0u);
  const bool early = g.early && g.pdl;
  // A kernel that touches memory before its predecessor is done must not let
  // its successor start. The successor of others may start before this CTA has
  // allocated TMEM: beside its 83 KB or more of shared memory only another CTA
  // of this kernel fits, and their 128 columns each.
  if (!early && g.pdl) {
    pdl_wait();
    pdl_launch_dependents();
  }
  int e, begin, rows;
  if (!nth_share(g, blockIdx.y, e, begin, rows)) {  // the whole cluster leaves
    if (early) pdl_wait();
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full, recv_full;
  __shared__ uint32_t tmem_slot;
  __shared__ float s_scale[MAX_WIDTH];
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = g.splits, kps = g.kps, stages = g.stages;
  const int width = (rows + 15) / 16 * 16;  // columns of the MMA
  const int w_bytes = kps * SUB, x_block = g.x_rows * 128, stage_bytes = w_bytes + kps * x_block;
  float* recv = reinterpret_cast<float*>(smem + stages * stage_bytes);  // [S][128 / S][stride]
  const int stride = width + 4, share = 128 / S;                        // floats of a row; rows this CTA finishes
  const int rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)(blockIdx.x / S) * 128;
  const WaitCtx& ctx = g.ctx;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&recv_full, 1);
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc<1>(&tmem_slot, 128);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  // First half of a cluster barrier: the peers wait for it before they send.
  if (S > 1) cluster_arrive_release();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // This CTA's K-blocks, a multiple of kps but at the end.
  const int total = (g.K + EPB - 1) / EPB;
  const int per = ((total + S - 1) / S + kps - 1) / kps * kps;
  const int kb0 = min(total, rank * per), kb1 = min(total, kb0 + per);
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  bool ok = true;  // of every wait of this warp

  if (warp == 0 || warp == X_WARP) {
    // ---------------------------------------- producers: of W (warp 0), of X
    // (the last warp). One warp for both took 1.2 us longer to fill the ring. A stage's
    // bytes are all announced by the first; those of X may land before that.
    const bool of_w = warp == 0;
    const uint32_t block_bytes = SUB + width * 128;
    if (early && !of_w) pdl_wait();
    int stage = 0;
    uint32_t phase = 1;
    for (int kb = kb0; kb < kb1; kb += kps) {
      ok = all_ok(mbar_wait(&empty[stage], phase, ctx, SITE_EMPTY));
      if (!ok) break;
      const int nq = min(kps, kb1 - kb);
      if (elect_one()) {
        if (of_w) mbar_arrive_expect_tx(&full[stage], nq * block_bytes);
        uint8_t* dst = smem + stage * stage_bytes + (of_w ? 0 : w_bytes);
        for (int q = 0; q < nq; ++q) {
          const int k0 = (kb + q) * EPB;
          if (of_w) {
            if constexpr (RR) {
              tma_load_3d(dst, &tmW, &full[stage], n0, k0, e);
              tma_load_3d(dst + 8192, &tmW, &full[stage], n0 + 64, k0, e);
            } else {
              tma_load_3d(dst, &tmW, &full[stage], k0, n0, e);
            }
            dst += SUB;
          } else {
            int r = 0;
            if (width == 128) {
              tma_load_2d(dst, &tmX.box[0], &full[stage], k0, begin);
              r = 64;
            }
#pragma unroll
            for (int m = 0; m < 3; ++m) {
              if ((width - r) & (64 >> m)) {
                tma_load_2d(dst + r * 128, &tmX.box[m], &full[stage], k0, begin + r);
                r += 64 >> m;
              }
            }
            dst += x_block;
          }
        }
      }
      __syncwarp();
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (early && of_w) pdl_wait();  // every path of a grid waits before it ends
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issuer
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t ring = smem_u32(smem), d_tmem = __shfl_sync(0xffffffffu, tmem, 0);
    const uint32_t idesc = IDESC | (uint32_t)(__shfl_sync(0xffffffffu, width, 0) >> 3) << 17;
    for (int kb = kb0; kb < kb1; kb += kps) {
      ok = all_ok(mbar_wait(&full[stage], phase, ctx, SITE_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t w_addr = ring + stage * stage_bytes, x_addr = w_addr + w_bytes;
      const int nq = min(kps, kb1 - kb);
      const uint64_t a0 = operand_desc<RR>(w_addr, 0), b0 = operand_desc<false>(x_addr, 0);
      const uint64_t a1 = operand_desc<RR>(w_addr + SUB, 0), b1 = operand_desc<false>(x_addr + x_block, 0);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t ad = a0 + k * (RR ? 128 : 2), bd = b0 + k * 2;
          const uint32_t accumulate = k == 0 && kb == kb0 ? 0u : 1u;
          if constexpr (I8) umma_i8<1>(d_tmem, ad, bd, idesc, accumulate);
          else umma_f16_cg1(d_tmem, ad, bd, idesc, accumulate);
        }
        if (nq == 2) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint64_t ad = a1 + k * (RR ? 128 : 2), bd = b1 + k * 2;
            if constexpr (I8) umma_i8<1>(d_tmem, ad, bd, idesc, 1u);
            else umma_f16_cg1(d_tmem, ad, bd, idesc, 1u);
          }
        }
        umma_commit_cg1(&empty[stage]);
      }
      __syncwarp();
      if (++stage == stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Also drains what was issued before an abort.
    if (kb1 > kb0 && elect_one()) umma_commit_cg1(&acc_full);
    __syncwarp();
  } else {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3, row = q * 32 + lane;  // TMEM lane quarter of this warp
    const int side = (warp - 2) / 4;              // two warps a quarter take every second run of columns
    const int et = threadIdx.x - 64;
    if (early) pdl_wait();  // the scales
    if (I8 && et < rows) s_scale[et] = g.scale[begin + et];
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (S > 1) {
      // The barrier completes once every peer's rows have landed.
      if (threadIdx.x == 64) mbar_arrive_expect_tx(&recv_full, (uint32_t)((S - 1) * share * width * 4));
      __syncwarp();
      cluster_wait_acquire();  // second half: the peers' barriers are set up
    }
    const bool some = kb1 > kb0;
    ok = all_ok(!some || mbar_wait(&acc_full, 0, ctx, SITE_TMEM_FULL));
    tc_fence_after();
    if (S == 1) {
      const int n = n0 + row;
      float sw = 0.f, bias = 0.f;
      if (I8 && n < g.N) {
        sw = g.w_scale[(int64_t)e * g.N + n];
        if (g.bias) bias = to_float(static_cast<const TO*>(g.bias)[n]);
      }
      TO* y = static_cast<TO*>(g.Y) + (int64_t)begin * g.ldy + n;
#pragma unroll 1
      for (int c = side * 16; c < width; c += EPI / 4 * 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (!ok || n >= g.N || c + j >= rows) continue;
          const float o = I8 ? (float)(int)v[j] * (sw * s_scale[c + j]) + bias : __uint_as_float(v[j]);
          y[(int64_t)(c + j) * g.ldy] = from_float<TO>(o);
        }
      }
    } else {
      // This thread's row goes to the CTA that finishes it.
      const int owner = row / share, place = (rank * share + row % share) * stride;
      const uint32_t bar = mapa_shared(smem_u32(&recv_full), owner);
      const uint32_t dst = mapa_shared(smem_u32(recv + place), owner);
#pragma unroll 1
      for (int c = side * 16; c < width; c += EPI / 4 * 16) {
        uint32_t v[16];
        if (some && ok) {
          tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0u;
        }
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (owner == rank) *reinterpret_cast<uint4*>(recv + place + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
          else send16(dst + (c + j) * 4, bar, v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
      }
      ok = all_ok(mbar_wait_cluster(&recv_full, 0, ctx, SITE_PARTIAL)) && ok;
      // The rows that this CTA keeps were written by some of its warps.
      asm volatile("bar.sync 1, 256;" ::: "memory");
      // Neighbouring threads take neighbouring n of one column of Y's.
      const int r = et % share, n = n0 + rank * share + r;
      float sw = 0.f, bias = 0.f;
      if (I8 && n < g.N) {
        sw = g.w_scale[(int64_t)e * g.N + n];
        if (g.bias) bias = to_float(static_cast<const TO*>(g.bias)[n]);
      }
      if (ok && n < g.N) {
        // Four columns at a time from every partial: with one warp a scheduler
        // only independent loads hide each other's latency (64 rows, column by
        // column: 7.4 us of 24).
        TO* y = static_cast<TO*>(g.Y) + (int64_t)begin * g.ldy + n;
#pragma unroll 2
        for (int c = et / share * 4; c < rows; c += EPI / 4 * S * 4) {
          uint4 part[8];
#pragma unroll
          for (int s = 0; s < 8; ++s)
            if (s < S) part[s] = *reinterpret_cast<const uint4*>(recv + (s * share + r) * stride + c);
          uint32_t sum[4] = {part[0].x, part[0].y, part[0].z, part[0].w};
#pragma unroll
          for (int s = 1; s < 8; ++s) {
            if (s >= S) break;
            const uint32_t v[4] = {part[s].x, part[s].y, part[s].z, part[s].w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              sum[j] = I8 ? sum[j] + v[j] : __float_as_uint(__uint_as_float(sum[j]) + __uint_as_float(v[j]));
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (c + j >= rows) break;
            const float o = I8 ? (float)(int)sum[j] * (sw * s_scale[c + j]) + bias : __uint_as_float(sum[j]);
            y[(int64_t)(c + j) * g.ldy] = from_float<TO>(o);
          }
        }
      }
    }
  }
  if ((warp < 2 || warp == X_WARP) && S > 1) {
    __syncwarp();
    cluster_wait_acquire();
  }
  // Peers finish writing into this CTA before its recv_full completes, which
  // every epilogue thread has waited for, so the CTA may end after this.
  __syncwarp();
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    // Some wait ran out. Every CTA sends its rows whatever its waits gave, so
    // recv_full completes soon after the last of the peers has given up too.
    if (S > 1) mbar_drain(&recv_full, 0, ctx.timeout_ns + 1000000000ull);
    settle();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, 128);
  }
}

template <typename TO, bool I8, bool RR>
int launch(const GroupedProblem& p) {
  constexpr int EPB = I8 ? 128 : 64, ES = I8 ? 1 : 2;
  const int type = I8 ? TMAP_U8 : p.in;
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  SkinnyArgs g = {};
  if ((rc = wait_ctx(&g.ctx))) return rc;
  g.offsets = p.offsets;
  g.E = (int)p.E, g.R = (int)p.R, g.N = (int)p.N, g.K = (int)p.K;
  g.Y = p.Y, g.ldy = p.ldy, g.scale = p.scale, g.w_scale = p.w_scale, g.bias = p.bias;
  g.pdl = pdl_enabled();
  g.early = p.early;
  CUtensorMap tW;
  RowMaps tX;
  const uint64_t wd[3] = {(uint64_t)(RR ? p.N : p.K), (uint64_t)(RR ? p.K : p.N), (uint64_t)p.E};
  const uint64_t ws[2] = {(uint64_t)(p.ldw * ES), (uint64_t)((p.E > 1 ? p.w_stride : p.ldw * (RR ? p.K : p.N)) * ES)};
  const uint32_t wb[3] = {(uint32_t)EPB, RR ? 64u : 128u, 1};
  if ((rc = make_tmap(&tW, p.W, type, 3, wd, ws, wb, 128))) return rc;
  const uint64_t xd[2] = {(uint64_t)p.K, (uint64_t)p.R};
  const uint64_t xs[1] = {(uint64_t)(p.ldx * ES)};
  for (int m = 0; m < 3; ++m) {
    const uint32_t xb[2] = {(uint32_t)EPB, 64u >> m};
    if ((rc = make_tmap(&tX.box[m], p.X, type, 2, xd, xs, xb, 128))) return rc;
  }
  // Once per device and instantiation: the shared-memory opt-in, and how many
  // clusters of 2, 4 and 8 such CTAs the device holds at once (fewer than its
  // SMs would give: a cluster stays within a GPC).
  auto kern = grouped_skinny_kernel<TO, I8, RR>;
  constexpr int ONE_CTA = 221 * 1024;
  static std::once_flag once[64];
  static cudaError_t err[64];
  static int clusters[64][9];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
    for (int s = 2; s <= 8 && err[di] == cudaSuccess; s *= 2) {
      PdlLaunch q(dim3(dev->sm_count / s * s), dim3(THREADS), ONE_CTA, nullptr, s);
      q.cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &q.cfg) == cudaSuccess) clusters[di][s] = n;
      (void)cudaGetLastError();
    }
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  // As many splits as run in one wave (a power of two, at least four K-blocks
  // each), for the shares that the groups can have.
  const int64_t shares = p.offsets ? p.R / MAX_WIDTH + std::min(p.R, p.E) : (p.R + MAX_WIDTH - 1) / MAX_WIDTH;
  const int64_t tiles = (p.N + 127) / 128 * shares, blocks = (p.K + EPB - 1) / EPB;
  g.splits = 1;
  while (g.splits < 8 && tiles <= clusters[di][g.splits * 2] && blocks >= g.splits * 8) g.splits *= 2;
  const int width = (int)std::min<int64_t>(MAX_WIDTH, (p.R + 15) / 16 * 16);  // of the widest share there can be
  g.x_rows = width;
  g.kps = width <= 64 ? 2 : 1;
  const int stage = g.kps * (SUB + width * 128);
  const int recv = g.splits > 1 ? 128 * (width + 4) * 4 : 0;
  // One CTA an SM takes most of the shared memory; with more CTAs than SMs two share it.
  const int budget = (tiles * g.splits > dev->sm_count ? 110 : 220) * 1024 - recv;
  g.stages = std::max(2, std::min(MAX_STAGES, budget / stage));
  const int smem = g.stages * stage + recv + 1024;
  const int64_t x = (p.N + 127) / 128 * g.splits;
  if (x > INT32_MAX || shares > 65535) return fail(KEBAB_EINVAL, "grouped product: too many tiles");
  PdlLaunch l(dim3((unsigned)x, (unsigned)shares), dim3(THREADS), smem, p.stream, g.splits);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, tW, tX, (const SkinnyArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "few-rows tcgen05 launch");
}

template <typename TO>
int launch_type(const GroupedProblem& p) {
  if (p.in == IN_I8) return launch<TO, true, false>(p);
  return p.kn ? launch<TO, false, true>(p) : launch<TO, false, false>(p);
}
}  // namespace

int launch_grouped_skinny(const GroupedProblem& p) {
  return p.out == KEBAB_F16 ? launch_type<__half>(p) : launch_type<__nv_bfloat16>(p);
}

}  // namespace kb
