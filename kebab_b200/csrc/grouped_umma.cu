// Grouped and 8-bit integer products on the tensor cores: persistent CTA pairs
// (cta_group::2) over the tiles of every group, whatever their sizes.
//
// The MMA's 256 rows are the output's contiguous dimension and its columns the
// other one, so that a lane of TMEM is a column of the row-major result:
//   forward (RC, RR)  rows: n (a W_e panel), columns: up to 256 rows of the
//                     group, contraction: k
//   dw                rows: the contiguous dimension of dW_e, columns: the
//                     other, contraction: the group's rows
// Ragged sizes cost what they are: a forward tile is as wide as its rows need
// (a multiple of 32; N is a field of the instruction descriptor), a group of
// 257 rows gives two tiles of 160 and 97 and not 256 and 1, and no group is
// padded in memory. Which tile belongs to which group is worked out on the
// device, from the offsets, by a prefix sum that every CTA does for itself.
//
// Edges: a forward tile may read past its group's end (the columns are not
// stored; a column does not reach its neighbours). In dw the contraction runs
// over rows, so rows past the group's end have to be zeros in both operands
// (a NaN there would spread): the last 16-row step is cleared in shared memory
// after it has landed, and steps beyond it are not issued.
//
// Ring: 3 stages of two 128-byte K-blocks (64 16-bit or 128 8-bit elements) of
// 128 rows of each operand a CTA; two accumulators of 256 columns, so that the
// epilogue of a tile runs under the next one's MMAs. Warps: TMA producer, MMA
// issuer, 4 epilogue warps, as in gemm_umma.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "gemm_umma.cuh"
#include "grouped.h"

namespace kb {
namespace {

enum : int { MODE_RC = 0, MODE_RR = 1, MODE_DW = 2 };

struct TileArgs {
  const int32_t* offsets;
  int E, R;
  int DA;      // extent of the MMA-row side: N (forward) or dW's contiguous dimension
  int DB;      // dw: the other dimension of dW
  int K;       // forward: contraction length
  int tma_out;
  void* Y;
  int64_t ldy;
  const float* scale;
  const float* w_scale;
  const void* bias;
  int pdl;
  WaitCtx ctx;
};

struct GSmem {
  static constexpr int STAGES = 3, KPS = 2;
  static constexpr int SUB = 128 * 128;  // 128 rows of 128 bytes: one K-block of one operand
  static constexpr int OFF_A = 0;
  static constexpr int OFF_B = OFF_A + STAGES * KPS * SUB;
  static constexpr int OFF_C = OFF_B + STAGES * KPS * SUB;
  static constexpr int C_SUB = 32 * 32 * 2;
  static constexpr int OFF_BAR = OFF_C + 4 * 2 * C_SUB;
  // full, empty, tail_full, tail_done a stage; tmem_full and tmem_empty twice; drain
  static constexpr int NUM_BARS = 4 * STAGES + 5;
  static constexpr int OFF_GROUPS = OFF_BAR + NUM_BARS * 8 + 16;
  static constexpr int bytes(int E) { return OFF_GROUPS + (3 * E + 1) * 4; }
  static constexpr int ALLOC = OFF_GROUPS + (3 * kMaxExperts + 1) * 4 + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget exceeded");
};

// Where each group's tiles start (first[e] .. first[e + 1]), in shared memory.
struct Groups {
  const int* first;  // [E + 1]
  const int* begin;  // [E]
  const int* rows;   // [E]
};

struct Tile {
  int e, a0, b0, width;  // group, first row and column of the tile, its columns (a multiple of 32)
  int begin, rows;       // the group's rows
  int blocks;            // 128-byte K-blocks of the contraction
};

template <int MODE>
__device__ __forceinline__ int tiles_b(const TileArgs& g, int rows) {
  return ((MODE == MODE_DW ? g.DB : rows) + 255) / 256;
}

template <int MODE, int EPB>
__device__ __forceinline__ Tile tile_of(int t, const TileArgs& g, const Groups& gr) {
  Tile x;
  int lo = 0, hi = g.E - 1;  // the last group that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (gr.first[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  x.e = lo;
  x.begin = gr.begin[lo];
  x.rows = gr.rows[lo];
  const int ta = (g.DA + 255) / 256, tb = tiles_b<MODE>(g, x.rows);
  int ma, mb;
  // Eight panels of the row side share the passes over the column side: the
  // 74 pairs then hold about 8 x 9 tiles at a time, near square.
  tile_coords(t - gr.first[lo], ta, tb, 8, ma, mb);
  x.a0 = ma * 256;
  if (MODE == MODE_DW) {
    x.width = 256;
    x.blocks = (x.rows + EPB - 1) / EPB;
  } else {
    x.width = ((x.rows + tb - 1) / tb + 31) / 32 * 32;  // equal shares
    x.blocks = (g.K + EPB - 1) / EPB;
  }
  x.b0 = mb * x.width;
  return x;
}

template <typename TO, bool I8, int MODE>
__global__ void __launch_bounds__(192, 1)
    grouped_umma_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ CUtensorMap tmB16, const __grid_constant__ CUtensorMap tmC,
                        const TileArgs g) {
  using L = GSmem;
  constexpr bool DW = MODE == MODE_DW;
  constexpr bool A_MN = MODE != MODE_RC, B_MN = DW;
  constexpr int EPB = I8 ? 128 : 64;  // elements of the contraction in a K-block
  constexpr int STAGES = L::STAGES, KPS = L::KPS;
  constexpr uint32_t IDESC = (I8 ? umma_idesc_i8(256, 0) : umma_idesc_f16(256, 0, ElemTraits<TO>::kBf16)) |
                             (A_MN ? (1u << 15) : 0u) | (B_MN ? (1u << 16) : 0u);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* tail_full = empty + STAGES;  // dw, in the peer: its own bytes of a group's last stage
  uint64_t* tail_done = tail_full + STAGES;  // dw, in the leader: the peer has cleared its share of it
  uint64_t* tmem_full = tail_done + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* drain = tmem_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + L::NUM_BARS);
  int* s_first = reinterpret_cast<int*>(smem + L::OFF_GROUPS);
  int* s_begin = s_first + g.E + 1;
  int* s_rows = s_begin + g.E;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const WaitCtx& ctx = g.ctx;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    tma_prefetch_desc(&tmC);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail_full[s], 1);
      mbar_init(&tail_done[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 4 * 2);
    }
    mbar_init(drain, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc<2>(tmem_slot, 512);
    tmem_relinquish<2>();
  }
  if (g.pdl) {
    pdl_wait();
    pdl_launch_dependents();
  }
  if (warp == 2) {
    // Prefix sum of the groups' tiles: a lane takes a run of groups.
    const int per = (g.E + 31) / 32, e0 = lane * per, ta = (g.DA + 255) / 256;
    int sum = 0;
    for (int i = 0; i < per && e0 + i < g.E; ++i) {
      int begin, rows;
      group_range(g.offsets, e0 + i, g.R, begin, rows);
      s_begin[e0 + i] = begin;
      s_rows[e0 + i] = rows;
      sum += ta * tiles_b<MODE>(g, rows);
    }
    int at = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, at, d);
      if (lane >= d) at += up;
    }
    if (lane == 31) s_first[g.E] = at;
    at -= sum;
    for (int i = 0; i < per && e0 + i < g.E; ++i) {
      s_first[e0 + i] = at;
      at += ta * tiles_b<MODE>(g, s_rows[e0 + i]);
    }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Groups gr{s_first, s_begin, s_rows};
  const int num_tiles = s_first[g.E];
  const int step = gridDim.x / 2;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      uint32_t issued = 0, parity = 0;  // a bit a stage
      const uint32_t full_leader0 = mapa_shared(smem_u32(&full[0]), 0);
      for (int t = blockIdx.x / 2; ok && t < num_tiles; t += step) {
        const Tile x = tile_of<MODE, EPB>(t, g, gr);
        const int half = x.width / 2;
        const int a0 = x.a0 + (int)rank * 128, b0 = x.b0 + (int)rank * half;
        const uint32_t block_bytes = L::SUB + half * 128;
        for (int kb = 0; kb < x.blocks; kb += KPS) {
          if (!mbar_wait(&empty[stage], phase ^ 1u, ctx, SITE_EMPTY)) {
            ok = false;
            break;
          }
          const int nq = min(KPS, x.blocks - kb);
          // A group's last stage that does not end on a 16-row step: each CTA
          // waits for its own bytes and clears the rows past the end.
          const bool tail = DW && kb + KPS >= x.blocks && (x.rows & 15) != 0;
          uint32_t bar = full_leader0 + stage * 8u;
          if (tail && !leader) {
            mbar_arrive_expect_tx(&tail_full[stage], nq * block_bytes);
            bar = mapa_shared(smem_u32(&tail_full[stage]), rank);
          } else if (leader) {
            mbar_arrive_expect_tx(&full[stage], (tail ? 1 : 2) * nq * block_bytes);
          }
          for (int q = 0; q < nq; ++q) {
            uint8_t* sA = smem + L::OFF_A + (stage * KPS + q) * L::SUB;
            uint8_t* sB = smem + L::OFF_B + (stage * KPS + q) * L::SUB;
            const int k0 = (kb + q) * EPB;
            if constexpr (MODE == MODE_RC) {
              tma_load_3d_pair(sA, &tmA, bar, k0, a0, x.e);
            } else if constexpr (MODE == MODE_RR) {
              tma_load_3d_pair(sA, &tmA, bar, a0, k0, x.e);
              tma_load_3d_pair(sA + 8192, &tmA, bar, a0 + 64, k0, x.e);
            } else {
              tma_load_2d_pair(sA, &tmA, bar, a0, x.begin + k0);
              tma_load_2d_pair(sA + 8192, &tmA, bar, a0 + 64, x.begin + k0);
              tma_load_2d_pair(sB, &tmB, bar, b0, x.begin + k0);
              tma_load_2d_pair(sB + 8192, &tmB, bar, b0 + 64, x.begin + k0);
            }
            if constexpr (!DW) {
              if (half == 128) {
                tma_load_2d_pair(sB, &tmB, bar, k0, x.begin + b0);
              } else {
                for (int r = 0; r < half; r += 16) tma_load_2d_pair(sB + r * 128, &tmB16, bar, k0, x.begin + b0 + r);
              }
            }
          }
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && leader) {
        // Abort: let the copies still in flight land before the CTA exits.
        WaitCtx drain_ctx{ctx.status, 50000000ull};
        for (int s = 0; s < STAGES; ++s)
          if (issued >> s & 1u) mbar_wait(&full[s], parity >> s & 1u, drain_ctx, SITE_DRAIN);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------ MMA issuer (leader); in dw the
    // whole warp of both CTAs clears the rows past a group's end.
    if (DW || (leader && lane == 0)) {
      int stage = 0;
      uint32_t phase = 0, tail_parity = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true, any_issued = false;
      const uint32_t tail_done_leader0 = mapa_shared(smem_u32(&tail_done[0]), 0);
      for (int t = blockIdx.x / 2; ok && t < num_tiles; t += step) {
        const Tile x = tile_of<MODE, EPB>(t, g, gr);
        if (x.blocks == 0) continue;  // dw of a group without rows
        if (leader) {
          ok = mbar_wait(&tmem_empty[acc], acc_phase ^ 1u, ctx, SITE_TMEM_EMPTY);
          if constexpr (DW) ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * 256);
        const uint32_t idesc = IDESC | (uint32_t)(x.width >> 3) << 17;
        for (int kb = 0; kb < x.blocks; kb += KPS) {
          const int left = DW ? x.rows - kb * EPB : 0;  // dw: rows of the group in this stage and later
          const bool tail = DW && kb + KPS >= x.blocks && (x.rows & 15) != 0;
          if (leader) {
            ok = mbar_wait(&full[stage], phase, ctx, SITE_FULL);
          } else if (DW && tail) {
            ok = mbar_wait(&tail_full[stage], tail_parity >> stage & 1u, ctx, SITE_FULL);
          }
          if constexpr (DW) {
            ok = __all_sync(0xffffffffu, ok);
            if (ok && tail) {
              // Rows left .. the end of its 16-row step, in the two boxes of
              // 64 columns of each operand (128-byte rows; the swizzle stays
              // within a row).
              const int q = left / EPB, r = left % EPB, n = (16 - (r & 15)) * 8;
              uint8_t* sA = smem + L::OFF_A + (stage * KPS + q) * L::SUB + r * 128;
              uint8_t* sB = smem + L::OFF_B + (stage * KPS + q) * L::SUB + r * 128;
              for (int i = lane; i < n; i += 32) {
                const uint4 zero = make_uint4(0, 0, 0, 0);
                *reinterpret_cast<uint4*>(sA + i * 16) = zero;
                *reinterpret_cast<uint4*>(sA + 8192 + i * 16) = zero;
                *reinterpret_cast<uint4*>(sB + i * 16) = zero;
                *reinterpret_cast<uint4*>(sB + 8192 + i * 16) = zero;
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (!leader) {
                if (lane == 0) mbar_arrive_cluster(tail_done_leader0 + stage * 8u);
              } else {
                ok = mbar_wait_cluster(&tail_done[stage], tail_parity >> stage & 1u, ctx, SITE_FULL);
                ok = __all_sync(0xffffffffu, ok);
              }
              tail_parity ^= 1u << stage;
            }
          }
          if (!ok) break;
          if (leader && (!DW || lane == 0)) {
            tc_fence_after();
            const uint32_t a_addr = smem_u32(smem + L::OFF_A + stage * KPS * L::SUB);
            const uint32_t b_addr = smem_u32(smem + L::OFF_B + stage * KPS * L::SUB);
            const int nq = min(KPS, x.blocks - kb);
#pragma unroll
            for (int q = 0; q < KPS; ++q) {
              if (q >= nq) break;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (DW && (q * 4 + k) * 16 >= left) break;
                const uint64_t ad = operand_desc<A_MN>(a_addr + q * L::SUB, k);
                const uint64_t bd = operand_desc<B_MN>(b_addr + q * L::SUB, k);
                const uint32_t accumulate = (kb | q | k) != 0 ? 1u : 0u;
                if constexpr (I8) umma_i8<2>(d_tmem, ad, bd, idesc, accumulate);
                else umma_f16_cg2(d_tmem, ad, bd, idesc, accumulate);
              }
            }
            any_issued = true;
            umma_commit_cg2_mc(&empty[stage], 0x3);
          }
          if constexpr (DW) __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (leader && (!DW || lane == 0)) umma_commit_cg2_mc(&tmem_full[acc], 0x3);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok && any_issued) {
        // Abort: wait for the MMAs already issued before TMEM is freed.
        umma_commit_cg2_mc(drain, 0x1);
        WaitCtx drain_ctx{ctx.status, 50000000ull};
        mbar_wait(drain, 0, drain_ctx, SITE_DRAIN);
      }
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    TO* stage_c = reinterpret_cast<TO*>(smem + L::OFF_C + (warp - 2) * 2 * L::C_SUB);
    const uint32_t tmem_empty_leader0 = mapa_shared(smem_u32(&tmem_empty[0]), 0);
    int acc = 0;
    uint32_t acc_phase = 0;
    int sub = 0;
    for (int t = blockIdx.x / 2; t < num_tiles; t += step) {
      const Tile x = tile_of<MODE, EPB>(t, g, gr);
      const int a_warp = x.a0 + (int)rank * 128 + q * 32;  // this warp's first row of the tile
      const int a = a_warp + lane;
      const int limit = DW ? g.DB : x.rows;  // columns end here
      const int chunks = x.width / 32;
      float sw = 0.f, bias = 0.f;
      if constexpr (I8) {
        if (a < g.DA) {
          sw = g.w_scale[(int64_t)x.e * g.DA + a];
          if (g.bias) bias = (float)static_cast<const TO*>(g.bias)[a];
        }
      }
      const bool some = x.blocks != 0;
      if (some && !mbar_wait(&tmem_full[acc], acc_phase, ctx, SITE_TMEM_FULL)) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * 256);
#pragma unroll 1
      for (int c = 0; c < chunks; ++c) {
        uint32_t v[32];
        if (some) {
          tmem_ld_32x32b_x32(t_row + (uint32_t)(c * 32), v);
          tmem_ld_wait();
          if (c == chunks - 1) {
            // Accumulator fully read: hand it back to the MMA issuer.
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tmem_empty_leader0 + (uint32_t)acc * 8u);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = 0u;
        }
        const int b = x.b0 + c * 32;  // this chunk's first column
        if (a_warp >= g.DA || b >= limit) continue;
        if constexpr (I8) {
          const float sx = b + lane < limit ? g.scale[x.begin + b + lane] : 0.f;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j] = __float_as_uint((float)(int)v[j] * (sw * __shfl_sync(0xffffffffu, sx, j)) + bias);
        }
        if (g.tma_out && (DW || b + 32 <= limit)) {
          TO* buf = stage_c + (sub & 1) * (32 * 32);
          if (lane == 0) tma_store_wait_read<1>();  // the store that used `buf` has read it
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 32; ++j) buf[j * 32 + lane] = ElemTraits<TO>::cvt(__uint_as_float(v[j]));
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if constexpr (DW) tma_store_3d(&tmC, buf, a_warp, b, x.e);
            else tma_store_2d(&tmC, buf, a_warp, x.begin + b);
            tma_store_commit();
          }
          ++sub;
        } else if (a < g.DA) {
          // The group ends inside the chunk (the next rows are another
          // group's), or TMA cannot address Y: 64 bytes a warp and column.
          TO* out = static_cast<TO*>(g.Y) + (DW ? (int64_t)x.e * g.DB + b : (int64_t)x.begin + b) * g.ldy + a;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (b + j < limit) out[j * g.ldy] = ElemTraits<TO>::cvt(__uint_as_float(v[j]));
        }
      }
      if (some) {
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    // The CTA may exit once its last stores have read their staging buffers.
    if (lane == 0) tma_store_wait_read<0>();
    __syncwarp();
  }

  // ------------------------------------------------------------- teardown
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

// Tensor map of a stack of row-major matrices (rows x cols, row pitch ld,
// matrix pitch `stride`, in elements of es bytes) with a box of box_rows rows
// of box_cols elements.
int map3(CUtensorMap* m, const void* base, int type, int es, int64_t n, int64_t rows, int64_t cols, int64_t ld,
         int64_t stride, int box_rows, int box_cols, int swizzle) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)n};
  const uint64_t strides[2] = {(uint64_t)(ld * es), (uint64_t)((n > 1 ? stride : ld * rows) * es)};
  const uint32_t box[3] = {(uint32_t)box_cols, (uint32_t)box_rows, 1};
  return make_tmap(m, base, type, 3, dims, strides, box, swizzle);
}
int map2(CUtensorMap* m, const void* base, int type, int es, int64_t rows, int64_t cols, int64_t ld, int box_rows,
         int box_cols, int swizzle) {
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)(ld * es)};
  const uint32_t box[2] = {(uint32_t)box_cols, (uint32_t)box_rows};
  return make_tmap(m, base, type, 2, dims, strides, box, swizzle);
}

template <typename TO, bool I8, int MODE>
int launch(const GroupedProblem& p) {
  constexpr bool DW = MODE == MODE_DW;
  constexpr int EPB = I8 ? 128 : 64, ES = I8 ? 1 : 2;
  const int type = I8 ? TMAP_U8 : p.in;
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  TileArgs g = {};
  if ((rc = wait_ctx(&g.ctx))) return rc;
  g.offsets = p.offsets;
  g.E = (int)p.E;
  g.R = (int)p.R;
  g.K = (int)p.K;
  g.Y = p.Y;
  g.scale = p.scale;
  g.w_scale = p.w_scale;
  g.bias = p.bias;
  g.pdl = pdl_enabled() ? 1 : 0;
  CUtensorMap tA, tB, tB16, tC;
  int64_t tiles;
  if constexpr (!DW) {
    g.DA = (int)p.N;
    g.ldy = p.ldy;
    if (MODE == MODE_RC) rc = map3(&tA, p.W, type, ES, p.E, p.N, p.K, p.ldw, p.w_stride, 128, EPB, 128);
    else rc = map3(&tA, p.W, type, ES, p.E, p.K, p.N, p.ldw, p.w_stride, 64, 64, 128);
    if (rc || (rc = map2(&tB, p.X, type, ES, p.R, p.K, p.ldx, 128, EPB, 128)) ||
        (rc = map2(&tB16, p.X, type, ES, p.R, p.K, p.ldx, 16, EPB, 128)))
      return rc;
    tiles = (p.N + 255) / 256 * (p.R / 256 + std::min(p.E, p.R));  // at most
  } else {
    // The contiguous dimension of dW is X's (RC) or dY's (RR) columns.
    const void* a = p.kn ? p.W : p.X;
    const void* b = p.kn ? p.X : p.W;
    const int64_t lda = p.kn ? p.ldw : p.ldx, ldb = p.kn ? p.ldx : p.ldw;
    g.DA = (int)(p.kn ? p.N : p.K);
    g.DB = (int)(p.kn ? p.K : p.N);
    g.ldy = g.DA;
    if ((rc = map2(&tA, a, type, ES, p.R, g.DA, lda, 64, 64, 128)) ||
        (rc = map2(&tB, b, type, ES, p.R, g.DB, ldb, 64, 64, 128)))
      return rc;
    tB16 = tB;
    tiles = p.E * ((g.DA + 255) / 256) * ((g.DB + 255) / 256);
  }
  if (tiles > INT32_MAX / 2) return fail(KEBAB_EINVAL, "grouped product: too many tiles");
  g.tma_out = (reinterpret_cast<uintptr_t>(p.Y) & 15u) == 0 && g.ldy % 8 == 0;
  if (!g.tma_out) tC = tA;  // not used
  else if (DW) rc = map3(&tC, p.Y, p.out, 2, p.E, g.DB, g.DA, g.ldy, g.ldy * g.DB, 32, 32, 0);
  else rc = map2(&tC, p.Y, p.out, 2, p.R, p.N, p.ldy, 32, 32, 0);
  if (rc) return rc;

  auto kern = grouped_umma_kernel<TO, I8, MODE>;
  const int smem = GSmem::bytes(g.E) + 1024;
  // Once per device and instantiation: the shared-memory opt-in and how many pairs fit.
  static std::once_flag once[64];
  static cudaError_t err[64];
  static int max_pairs[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, GSmem::ALLOC);
    max_pairs[di] = dev->sm_count / 2;
    if (err[di] != cudaSuccess) return;
    PdlLaunch q(dim3(2 * max_pairs[di]), dim3(192), GSmem::ALLOC, nullptr, 2);
    q.cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &q.cfg) == cudaSuccess && n > 0) max_pairs[di] = std::min(n, max_pairs[di]);
    (void)cudaGetLastError();
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  const int pairs = (int)std::min<int64_t>(tiles, max_pairs[di]);
  PdlLaunch l(dim3(2 * pairs), dim3(192), smem, p.stream, 2);
  const cudaError_t e = cudaLaunchKernelEx(&l.cfg, kern, tA, tB, tB16, tC, g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "grouped tcgen05 launch");
}

template <typename TO>
int launch_type(const GroupedProblem& p) {
  if (p.in == IN_I8) return launch<TO, true, MODE_RC>(p);
  if (p.dw) return launch<TO, false, MODE_DW>(p);
  return p.kn ? launch<TO, false, MODE_RR>(p) : launch<TO, false, MODE_RC>(p);
}
}  // namespace

int launch_grouped_umma(const GroupedProblem& p) {
  return p.out == KEBAB_F16 ? launch_type<__half>(p) : launch_type<__nv_bfloat16>(p);
}

// TMA takes 16-byte aligned bases and pitches of multiples of 16 bytes.
bool grouped_tma_ok(const GroupedProblem& p) {
  const int64_t es = p.in == IN_I8 ? 1 : 2;
  const bool w_ok = (reinterpret_cast<uintptr_t>(p.W) & 15u) == 0 && p.ldw * es % 16 == 0 &&
                    (p.dw || p.E == 1 || p.w_stride * es % 16 == 0);
  return w_ok && (reinterpret_cast<uintptr_t>(p.X) & 15u) == 0 && p.ldx * es % 16 == 0;
}

}  // namespace kb
