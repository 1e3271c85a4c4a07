// 4-bit floating-point products for few rows, or few tiles, on the tensor cores:
// bound by the weights' bytes, or by how many SMs have work.
//
// A CTA multiplies 128 weight rows n (the MMA's row side, so that a lane of
// TMEM is a column of Y) with up to 128 rows of one group (equal shares of a
// larger group, padded to a multiple of 16). Where that gives too few CTAs, a
// cluster of S of them splits k: each ends with a partial sum in TMEM, sends
// every other CTA the 128 / S of its rows that that one finishes (st.async,
// counted on the receiver's barrier), and adds up its own rows over the S
// partials in rank order. No workspace, no atomics, and the same bits every
// time. With the quantisation, 1 row of 8192 x 8192 takes 9.6 us and 61 rows
// 14.4 (3.7 and 2.6 TB/s; with codes at hand 61 rows 13.0): latency of the first
// copies and of the exchange. Several accumulators in turn gave nothing.
//
// A K-block is 256 values: 128 bytes of codes a row, and two runs of 128 whose
// scales (512 bytes for 128 rows, as they are stored) the issuer copies into
// TMEM before their MMAs. Copies and MMAs of one thread execute in order, so
// that two places in turn suffice for the scales.
//
// In linear_f4 the kernel before this one only makes the codes and scales of X
// (`early`): the first weights are fetched while it still runs.
// Of up to 6 rows this kernel makes them itself (FUSED): 8 values a lane, eight
// warps, some 300 cycles a row and K-block of a warp, while the weights arrive.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "f4.h"
#include "gemm_umma.cuh"
#include "group_search.cuh"
#include "quant_f4.cuh"

namespace kb {
namespace {
// Warps: copies of W, MMA issuer, 8 epilogue warps, copies of X.
constexpr int EPI = 8, X_WARP = 2 + EPI, THREADS = 32 * (3 + EPI);
constexpr int SUB = 128 * 128;    // 128 rows of 128 bytes
constexpr int SCALES = 2 * 512;   // of 128 rows and 256 values
constexpr int MAX_STAGES = 8, MAX_WIDTH = 128;
constexpr int TMEM_COLS = 256, SF_COL = 128;  // accumulator, then twice 16 columns of scales

struct F4SkinnyArgs {
  const int32_t* offsets;
  int E, R, N;
  int pitch;             // bytes of a row's codes
  int n_tiles;  // runs of 128 weight rows
  int splits;
  int kps, stages, x_rows;  // K-blocks a stage, stages, rows of X that a stage has room for
  void* Y;
  int64_t ldy;
  const void* bias;
  int early, pdl;
  const void* x;  // FUSED
  int64_t ldx;
  int K, vec_x;   // whether rows of x start on 16-byte boundaries
  WaitCtx ctx;
};

// Boxes of 64, 32 and 16 rows of X.
struct RowMaps {
  CUtensorMap box[3];
};

// FUSED: the epilogue's warps, which have nothing else to do before the end, make
// the codes and scales of X (of the output type) where TMA would place them.
template <typename TO, bool FUSED>
__global__ void __launch_bounds__(THREADS)
    f4_skinny_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmWs,
                     const __grid_constant__ RowMaps tmX, const __grid_constant__ CUtensorMap tmXs,
                     const F4SkinnyArgs g) {
  const bool early = g.early && g.pdl;
  // A kernel that touches memory before its predecessor is done must not let
  // its successor start. The successor of others may start before this CTA has
  // allocated TMEM: beside its shared memory (launch) only another CTA of this
  // kernel fits, and their 256 columns each.
  const bool late = FUSED && !g.offsets;  // nothing is read before the loads
  if (!early && g.pdl) {
    if (!late) pdl_wait();
    pdl_launch_dependents();
  }
  int e, begin, rows;
  if (!nth_share<THREADS, MAX_WIDTH>(g.offsets, g.E, g.R, blockIdx.y, e, begin, rows)) {  // the whole cluster leaves
    if (early) pdl_wait();
    return;
  }

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full, recv_full;
  __shared__ uint32_t tmem_slot;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int S = g.splits, kps = FUSED ? 2 : g.kps, stages = g.stages;  // (FUSED: at most 16 rows)
  const int width = (rows + 15) / 16 * 16;  // columns of the MMA
  // A stage: codes of W and X, scales of W and X, each kps K-blocks.
  const int w_bytes = kps * SUB, x_block = g.x_rows * 128, sf_bytes = w_bytes + kps * x_block;
  const int stage_bytes = sf_bytes + 2 * kps * SCALES;
  float* recv = reinterpret_cast<float*>(smem + stages * stage_bytes);  // [S][128 / S][stride]
  const int stride = width + 4, share = 128 / S;                        // floats of a row; rows this CTA finishes
  const int rank = S > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)(blockIdx.x / S) * 128;
  const WaitCtx& ctx = g.ctx;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], FUSED ? 1 + EPI : 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&recv_full, 1);
    fence_barrier_init();
  }
  __syncwarp();
  // TMEM is not held while another kernel, which may share the SM, still needs some.
  if (late && g.pdl) pdl_wait();
  if (warp == 1) {
    tmem_alloc<1>(&tmem_slot, TMEM_COLS);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  // First half of a cluster barrier: the peers wait for it before they send.
  if (S > 1) cluster_arrive_release();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;

  // This CTA's K-blocks, a multiple of kps but at the end.
  const int total = (g.pitch + 127) / 128;
  const int per = ((total + S - 1) / S + kps - 1) / kps * kps;
  const int kb0 = min(total, rank * per), kb1 = min(total, kb0 + per);
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  bool ok = true;  // of every wait of this warp

  if (FUSED && warp == X_WARP) {
    // (nothing to copy)
  } else if (warp == 0 || warp == X_WARP) {
    // ---------------------------------------- producers: of W (warp 0), of X
    // (the last warp). One warp for both took 1.2 us longer to fill the ring. A stage's
    // bytes are all announced by the first; those of X may land before that.
    const bool of_w = warp == 0;
    const uint32_t block_bytes = FUSED ? SUB + SCALES : SUB + width * 128 + 2 * SCALES;
    const int w_tile = e * g.n_tiles + n0 / 128;
    if (early && !of_w) pdl_wait();
    int stage = 0;
    uint32_t phase = 1;
    for (int kb = kb0; kb < kb1; kb += kps) {
      ok = all_ok(mbar_wait(&empty[stage], phase, ctx, SITE_EMPTY));
      if (!ok) break;
      const int nq = min(kps, kb1 - kb);
      if (elect_one()) {
        if (of_w) mbar_arrive_expect_tx(&full[stage], nq * block_bytes);
        uint8_t* base = smem + stage * stage_bytes;
        uint8_t* dst = base + (of_w ? 0 : w_bytes);
        uint8_t* sf = base + sf_bytes + (of_w ? 0 : kps * SCALES);
        for (int q = 0; q < nq; ++q, sf += SCALES) {
          const int k0 = (kb + q) * 128;  // bytes
          if (of_w) {
            tma_load_3d(dst, &tmW, &full[stage], k0, n0, e);
            tma_load_3d(sf, &tmWs, &full[stage], 0, 2 * (kb + q), w_tile);
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
            tma_load_2d(sf, &tmXs, &full[stage], begin * 8, 2 * (kb + q));
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
    const uint32_t n_bits = (uint32_t)(__shfl_sync(0xffffffffu, width, 0) >> 3) << 17;
    const uint32_t idesc0 = umma_idesc_mxf4(128, 0, 0) | n_bits, idesc2 = umma_idesc_mxf4(128, 0, 2) | n_bits;
    for (int kb = kb0; kb < kb1; kb += kps) {
      ok = all_ok(mbar_wait(&full[stage], phase, ctx, SITE_FULL));
      if (!ok) break;
      tc_fence_after();
      const uint32_t w_addr = ring + stage * stage_bytes, x_addr = w_addr + w_bytes, sf_addr = w_addr + sf_bytes;
      const int nq = min(kps, kb1 - kb);
      if (elect_one()) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          if (q >= nq) break;
          const uint64_t a0 = umma_desc_sw128(w_addr + q * SUB), b0 = umma_desc_sw128(x_addr + q * x_block);
          const int bytes = g.pitch - (kb + q) * 128;  // of codes from here on
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h * 64 >= bytes) break;  // no such run of 128 values
            const uint32_t sf = d_tmem + SF_COL + h * 16;
            const uint32_t tile = sf_addr + q * SCALES + h * 512;
            tmem_cp_scales<1>(sf, umma_desc(tile, 16, 128, 0));
            tmem_cp_scales<1>(sf + 8, umma_desc(tile + kps * SCALES, 16, 128, 0));
            const uint32_t accumulate = h == 0 && q == 0 && kb == kb0 ? 0u : 1u;
            umma_mxf4<1>(d_tmem, a0 + 4 * h, b0 + 4 * h, idesc0, sf, sf + 8, accumulate);
            if (h * 64 + 32 < bytes) umma_mxf4<1>(d_tmem, a0 + 4 * h + 2, b0 + 4 * h + 2, idesc2, sf, sf + 8, 1u);
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
    // Y may be what a kernel before the one that makes X's codes still reads.
    if (early) pdl_wait();
    if constexpr (FUSED) {
      // Rows and K-blocks of a stage in turn, 8 values a lane; four loads ahead.
      const TO* x = static_cast<const TO*>(g.x) + (int64_t)begin * g.ldx;
      const int w = warp - 2, steps = rows * kps;  // of a stage
      int load_kb = kb0, load_i = w;
      auto load = [&] {
        Run<TO, 8> run = {};
        if (load_kb >= kb1 || load_i >= steps) return run;
        const int k = (load_kb + load_i % kps) * 256 + lane * 8;
        const TO* from = x + (int64_t)(load_i / kps) * g.ldx;
        if (g.vec_x && k + 8 <= g.K) {
          run.load(from + k);
        } else {
          float v[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) v[u] = k + u < g.K ? to_float(from[k + u]) : 0.f;
          run.set(v);
        }
        if ((load_i += EPI) >= steps) load_i = w, load_kb += kps;
        return run;
      };
      constexpr int AHEAD = 4;
      Run<TO, 8> next[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) next[u] = load();
      int stage = 0, kb = kb0, i = w;
      uint32_t phase = 1;
      while (kb < kb1) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (kb >= kb1) break;
          if (i == w) ok = all_ok(mbar_wait(&empty[stage], phase, ctx, SITE_EMPTY));
          if (!ok) break;
          uint8_t* base = smem + stage * stage_bytes;
          const Run<TO, 8> run = next[u];
          next[u] = load();
          const EightCodes r = eight_codes(run, lane);
          const int at = i / kps, q = i % kps;  // (of a last stage with less than kps: zeros that nothing reads)
          if (i < steps) {
            *reinterpret_cast<uint32_t*>(base + w_bytes + q * x_block + at * 128 + ((lane / 4 ^ (at & 7)) << 4) +
                                         lane % 4 * 4) = r.codes;
            if (lane % 16 == 0)
              *reinterpret_cast<uint32_t*>(base + sf_bytes + (kps + q) * SCALES + lane / 16 * 512 + at * 16) = r.scales;
          }
          if ((i += EPI) < steps) continue;
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full[stage]);
          __syncwarp();
          i = w;
          kb += kps;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
      }
    }
    if (S > 1) {
      // The barrier completes once every peer's rows have landed.
      if (threadIdx.x == 64) mbar_arrive_expect_tx(&recv_full, (uint32_t)((S - 1) * share * width * 4));
      __syncwarp();
      cluster_wait_acquire();  // second half: the peers' barriers are set up
    }
    const bool some = kb1 > kb0;
    ok = all_ok(!some || mbar_wait(&acc_full, 0, ctx, SITE_TMEM_FULL)) && ok;
    tc_fence_after();
    if (S == 1) {
      const int n = n0 + row;
      const float bias = g.bias && n < g.N ? to_float(static_cast<const TO*>(g.bias)[n]) : 0.f;
      TO* y = static_cast<TO*>(g.Y) + (int64_t)begin * g.ldy + n;
#pragma unroll 1
      for (int c = side * 16; c < width; c += EPI / 4 * 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (!ok || n >= g.N || c + j >= rows) continue;
          y[(int64_t)(c + j) * g.ldy] = from_float<TO>(__uint_as_float(v[j]) + bias);
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
      const float bias = g.bias && n < g.N ? to_float(static_cast<const TO*>(g.bias)[n]) : 0.f;
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
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < 8; ++s) {
            if (s >= S) break;
            const uint32_t v[4] = {part[s].x, part[s].y, part[s].z, part[s].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += __uint_as_float(v[j]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (c + j >= rows) break;
            y[(int64_t)(c + j) * g.ldy] = from_float<TO>(sum[j] + bias);
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
    tmem_dealloc<1>(tmem, TMEM_COLS);
  }
}

template <typename TO, bool FUSED>
int launch(const F4Problem& p) {
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  F4SkinnyArgs g = {};
  if ((rc = wait_ctx(&g.ctx))) return rc;
  g.offsets = p.offsets;
  g.E = (int)p.E, g.R = (int)p.R, g.N = (int)p.N;
  g.pitch = (int)f4_pitch(p.K);
  g.n_tiles = (int)((p.N + 127) / 128);
  g.Y = p.Y, g.ldy = p.ldy, g.bias = p.bias;
  g.pdl = pdl_enabled();
  g.early = p.early;
  if (FUSED) {
    g.x = p.x, g.ldx = p.ldx, g.K = (int)p.K;
    g.vec_x = (reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && p.ldx % 8 == 0;
  }
  CUtensorMap tW, tWs, tXs;
  if ((rc = f4_weight_map(p, &tW)) || (rc = f4_weight_scale_map(p, &tWs))) return rc;
  tXs = tW;  // not used if FUSED
  if (!FUSED && (rc = f4_token_scale_map(p, &tXs))) return rc;
  // The boxes that the shares' widths are made of; of groups, whose sizes the
  // device knows, all.
  int boxes = 64 | 32 | 16;
  if (!p.offsets) {
    const int64_t n = (p.R + MAX_WIDTH - 1) / MAX_WIDTH, share = (p.R + n - 1) / n, last = p.R - (n - 1) * share;
    auto width = [](int64_t rows) { return (int)((rows + 15) / 16 * 16); };
    boxes = width(share) | width(last) | (std::max(width(share), width(last)) == MAX_WIDTH ? 64 : 0);
  }
  RowMaps tX;
  for (int i = 0; i < 3; ++i) {
    tX.box[i] = tXs;  // not used
    if (!FUSED && (boxes & (64 >> i)) && (rc = f4_token_map(p, 64 >> i, &tX.box[i]))) return rc;
  }
  // Once per device and instantiation: the shared-memory opt-in, and how many
  // clusters of 2, 4 and 8 such CTAs the device holds at once (fewer than its
  // SMs would give: a cluster stays within a GPC).
  auto kern = f4_skinny_kernel<TO, FUSED>;
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
  const int64_t tiles = g.n_tiles * shares, blocks = (g.pitch + 127) / 128;
  g.splits = 1;
  while (g.splits < 8 && tiles <= clusters[di][g.splits * 2] && blocks >= g.splits * 8) g.splits *= 2;
  const int width = (int)std::min<int64_t>(MAX_WIDTH, (p.R + 15) / 16 * 16);  // of the widest share there can be
  g.x_rows = width;
  g.kps = width <= 64 ? 2 : 1;
  const int stage = g.kps * (SUB + width * 128 + 2 * SCALES);
  const int recv = g.splits > 1 ? 128 * (width + 4) * 4 : 0;
  // One CTA an SM takes most of the shared memory; with more CTAs than SMs two share it.
  const int budget = (tiles * g.splits > dev->sm_count ? 110 : 220) * 1024 - recv;
  g.stages = std::max(2, std::min(MAX_STAGES, budget / stage));
  // At least a third of an SM's, so that no more than two CTAs (512 columns of TMEM) share one.
  const int smem = std::max(g.stages * stage + recv + 1024, 80 * 1024);
  const int64_t x = (int64_t)g.n_tiles * g.splits;
  if (x > INT32_MAX || shares > 65535) return fail(KEBAB_EINVAL, "gemm_f4: too many tiles");
  PdlLaunch l(dim3((unsigned)x, (unsigned)shares), dim3(THREADS), smem, p.stream, g.splits);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, tW, tWs, tX, tXs, (const F4SkinnyArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "few-rows 4-bit launch");
}
}  // namespace

int launch_f4_skinny(const F4Problem& p) {
  if (p.x) return p.out == KEBAB_F16 ? launch<__half, true>(p) : launch<__nv_bfloat16, true>(p);
  return p.out == KEBAB_F16 ? launch<__half, false>(p) : launch<__nv_bfloat16, false>(p);
}

}  // namespace kb
