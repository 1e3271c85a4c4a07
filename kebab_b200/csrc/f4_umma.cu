// 4-bit floating-point products on the tensor cores: persistent CTA pairs
// (cta_group::2) over the tiles of every group, whatever their sizes.
//
// The MMA's rows are weight rows n, so that a lane of TMEM is a column of the
// row-major result, and its columns are rows of the group. A tile is a panel of
// 256 rows by up to 240 columns. Two accumulators of 240 columns take turns, so
// that 8 epilogue warps read one tile while the next is multiplied; the other 32
// of TMEM's 512 columns hold scales.
//
// A K-block is 256 values: 128 bytes of codes a row, and two runs of 128 values
// whose scales (512 bytes for 128 rows, as they are stored) the issuer copies
// into TMEM before the MMAs that use them. Copies and MMAs of one thread execute
// in order, so that two places in turn suffice. Token scales are stored so that
// a run of 128 rows may begin anywhere (include/kebab/f4.h): the copies of a tile
// that starts at any row of a group start on 16 bytes.
//
// Ragged sizes cost what they are: a tile is as wide as its rows need (a
// multiple of 16; equal shares of a group), and no group is padded in memory. A
// tile may read past its group's end: the columns are not stored, and a column
// does not reach its neighbours.
//
// Copies: as few as there can be (the panel's codes, its scales, the columns'
// codes, at most two of the columns' scales a K-block; of ten smaller ones, 1 %
// more). 4093 x 28672 x 8192 takes 295 us after a pause, 6.5 PFLOP/s (3.9 times the
// 16-bit library product's rate), and 320 in a row, at the clock that the power
// leaves. Panels of 512 rows, two MMAs to a stage's columns, copy a third less and
// took 324: what they save is not what bounds it, and their halves had to wait for
// one another's accumulators (8 matrices of 14336 x 4096, 4093 rows: 131 against
// 104). 32 matrices of 4096 x 4096 and 1021 rows, bound by the weights: 55 us with
// the quantisation, 5.1 TB/s.
//
// Ring: 6 stages of 34 KB a CTA. Warps: TMA producer, MMA issuer, 8 epilogue
// warps, and one that works out the tiles ahead of them.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>

#include "f4.h"
#include "gemm_umma.cuh"
#include "vec.cuh"

namespace kb {
namespace {

constexpr int EPILOGUE = 8, THREADS = 32 * (EPILOGUE + 3);
constexpr int CAP = 240;             // columns of a tile, at most
constexpr int SUB = 128 * 128;       // 128 rows of 128 bytes of codes
constexpr int B_BYTES = CAP / 2 * 128;
constexpr int SCALES = 2 * 512;      // of 128 rows and 256 values
// A stage: codes of the panel and the columns, scales of the panel and the columns.
constexpr int OFF_SFA = SUB + B_BYTES, OFF_SFB = OFF_SFA + SCALES, STAGE_BYTES = OFF_SFB + 2 * SCALES;
constexpr int STAGES = 6, TILES = 4;
constexpr int SF_COL = 2 * CAP;      // twice 16 columns: 8 of the columns' scales, 4 of the rows'
constexpr int RUN = 32;              // columns that an epilogue warp stores at a time
constexpr int OFF_C = STAGES * STAGE_BYTES;
constexpr int OFF_BAR = OFF_C + EPILOGUE * RUN * 32 * 2;
constexpr int NUM_BARS = 2 * STAGES + 4 + 2 * TILES;
constexpr int OFF_TILES = (OFF_BAR + NUM_BARS * 8 + 8 + 15) / 16 * 16;  // after the TMEM address, abort
constexpr int OFF_TABLE = OFF_TILES + TILES * 32;
constexpr int smem_bytes(int E) { return OFF_TABLE + (E + 1) * 4 + 1024; }
static_assert(smem_bytes(kMaxExperts) <= 232448, "shared memory budget exceeded");

struct F4Args {
  const int32_t* offsets;
  int E, R, N;
  int pitch;             // bytes of a row's codes
  int n_tiles;           // runs of 128 weight rows
  int vec_out;           // rows of Y on 16-byte boundaries
  void* Y;
  int64_t ldy;
  const void* bias;
  int pdl;
  WaitCtx ctx;
};

// Boxes of rows of X: the least that holds a CTA's half of a tile's columns.
constexpr int BOXES = 5;
struct ColumnMaps {
  CUtensorMap box[BOXES];
};
__host__ __device__ constexpr int box_rows(int i) { return i == 0 ? 120 : i == 1 ? 112 : i == 2 ? 96 : i == 3 ? 64 : 32; }

// Group i has the column blocks first[i] .. first[i + 1] - 1, each of `panels` tiles.
struct Table {
  const int* first;
  int panels, cap;
};

struct alignas(16) Tile {
  int e, a0, b0, width;  // group (-1: no more tiles), first row and column of the tile, its columns (a multiple of 16)
  int begin, rows;       // the group's rows
};

// Columns of a group's tiles: equal shares of at most `cap`, in runs of 16, the wider ones first.
struct Widths {
  int count, narrow, wider;  // `wider` of the tiles have 16 columns more
  __device__ __forceinline__ Widths(int rows, int cap) {
    const int runs = (rows + 15) / 16;
    count = (rows + cap - 1) / cap;
    const int per = count > 1 ? runs / count : runs;
    wider = runs - per * count;
    narrow = per * 16;
  }
};

// Tile `local` of panels x blocks: eight panels share the passes over the
// columns, so that the pairs hold about 8 x 9 tiles at a time.
__device__ __forceinline__ void raster(int local, int panels, int blocks, int& pa, int& cb) {
  const int group = local / (8 * blocks), in_group = local - group * 8 * blocks;
  const int height = min(8, panels - group * 8);
  cb = in_group / height;
  pa = group * 8 + in_group - cb * height;
}

__device__ __forceinline__ Tile tile_of(int64_t t, const F4Args& g, const Table& tab) {
  Tile x;
  int lo = 0, hi = g.E - 1;  // the last group that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((int64_t)tab.first[mid] * tab.panels <= t) lo = mid;
    else hi = mid - 1;
  }
  x.e = lo;
  group_range(g.offsets, x.e, g.R, x.begin, x.rows);
  const Widths w(x.rows, tab.cap);
  int pa, cb;
  raster((int)(t - (int64_t)tab.first[lo] * tab.panels), tab.panels, w.count, pa, cb);
  x.width = w.narrow + (cb < w.wider ? 16 : 0);
  x.b0 = cb * w.narrow + min(cb, w.wider) * 16;
  x.a0 = pa * 256;
  return x;
}

// The same from lane 0, for code of a whole warp.
__device__ __forceinline__ Tile uniform(const Tile& x) {
  auto u = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  return {u(x.e), u(x.a0), u(x.b0), u(x.width), u(x.begin), u(x.rows)};
}

// Block-wide sums of three values a thread.
__device__ __forceinline__ void block_sums(int (&v)[3], int (*sums)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) v[i] = __reduce_add_sync(0xffffffffu, v[i]);
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) sums[threadIdx.x >> 5][i] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = 0;
    for (int w = 0; w < THREADS / 32; ++w) v[i] += sums[w][i];
  }
  __syncthreads();
}

// Makes the table, by all threads of the CTA.
__device__ __forceinline__ Table make_table(const F4Args& g, int pairs, int* first) {
  __shared__ int sums[THREADS / 32][3];
  __shared__ int totals[THREADS / 32];
  const int panels = (g.N + 255) / 256;
  // The widest tile of 240, 192 or 128 columns, by the waves over the pairs and
  // the rows that a tile's K-block copies (256 of the panel and its columns). (Of
  // a cost that counts the columns more, 64 + width, 4096 x 14336 x 4093 took 103 us,
  // not 84; five widths to choose from gave nothing.)
  int c[3] = {0, 0, 0};
  for (int i = threadIdx.x; i < g.E; i += THREADS) {
    int begin, rows;
    group_range(g.offsets, i, g.R, begin, rows);
    c[0] += (rows + CAP - 1) / CAP;
    c[1] += (rows + 191) / 192;
    c[2] += (rows + 127) / 128;
  }
  block_sums(c, sums);
  Table tab;
  tab.cap = CAP;
  int total = c[0];
  auto cost = [&](int blocks, int width) { return ((int64_t)blocks * panels + pairs - 1) / pairs * (256 + width); };
  if (cost(c[1], 192) < cost(total, tab.cap)) tab.cap = 192, total = c[1];
  if (cost(c[2], 128) < cost(total, tab.cap)) tab.cap = 128, total = c[2];
  // Sums over the groups before each, a run of groups a thread.
  const int per = (g.E + THREADS - 1) / THREADS, i0 = threadIdx.x * per;
  int mine = 0;
  for (int i = i0; i < min(g.E, i0 + per); ++i) {
    int begin, rows;
    group_range(g.offsets, i, g.R, begin, rows);
    mine += (rows + tab.cap - 1) / tab.cap;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int at = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, at, d);
    if (lane >= d) at += up;
  }
  if (lane == 31) totals[warp] = at;
  __syncthreads();
  at -= mine;
  for (int w = 0; w < warp; ++w) at += totals[w];
  for (int i = i0; i < min(g.E, i0 + per); ++i) {
    int begin, rows;
    group_range(g.offsets, i, g.R, begin, rows);
    first[i] = at;
    at += (rows + tab.cap - 1) / tab.cap;
  }
  if (threadIdx.x == 0) first[g.E] = total;
  tab.first = first;
  tab.panels = panels;
  return tab;
}

template <typename TO>
__global__ void __launch_bounds__(THREADS, 1)
    f4_umma_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmWs,
                   const __grid_constant__ ColumnMaps tmX, const __grid_constant__ CUtensorMap tmXs,
                   const __grid_constant__ CUtensorMap tmY, const F4Args g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* tmem_full = empty + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* tile_full = tmem_empty + 2;
  uint64_t* tile_empty = tile_full + TILES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + NUM_BARS);
  uint32_t* s_abort = tmem_slot + 1;  // some wait of the pair ran out
  Tile* s_tiles = reinterpret_cast<Tile*>(smem + OFF_TILES);
  int* s_first = reinterpret_cast<int*>(smem + OFF_TABLE);

  // A warp takes one path; the producer and the issuer run with all lanes, one
  // of which is elected at each copy or MMA, so that addresses and descriptors
  // stay in uniform registers.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const WaitCtx& ctx = g.ctx;

  cluster_arrive_release();  // this CTA has started
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmWs);
    tma_prefetch_desc(&tmXs);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], EPILOGUE * 2);
    }
    for (int a = 0; a < TILES; ++a) {
      mbar_init(&tile_full[a], 1);
      mbar_init(&tile_empty[a], EPILOGUE + 1 + (leader ? 1 : 0));  // the warps that read descriptions
    }
    *s_abort = 0;
    fence_barrier_init();
  }
  __syncwarp();
  // The pair allocates together: not before the other CTA has started.
  cluster_wait_acquire();
  if (warp == 1) {
    tmem_alloc<2>(tmem_slot, 512);
    tmem_relinquish<2>();
  }
  __syncwarp();
  cluster_arrive_release();  // the pair's barriers; the other half is below
  if (g.pdl) {
    pdl_wait();
    pdl_launch_dependents();
  }
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  const Table tab = make_table(g, pairs, s_first);
  tc_fence_before();
  __syncthreads();
  cluster_wait_acquire();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int blocks = (g.pitch + 127) / 128;  // K-blocks
  // The i-th tile of this pair, for a whole warp; e is -1 after the last, and -2
  // where the wait for it ran out.
  auto next_tile = [&](int i) {
    const int at = i % TILES;
    Tile x;
    if (__all_sync(0xffffffffu, mbar_wait(&tile_full[at], i / TILES & 1, ctx, SITE_TILE))) x = uniform(s_tiles[at]);
    else x.e = -2;
    __syncwarp();
    if (lane == 0) mbar_arrive(&tile_empty[at]);
    return x;
  };
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  bool ok = true;  // of every wait of this warp

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0;
    const uint32_t full_leader0 = mapa_shared(smem_u32(&full[0]), 0);
    for (int i = 0; ok; ++i) {
      const Tile x = next_tile(i);
      if (x.e < 0) {
        ok = x.e == -1;
        break;
      }
      const int half = x.width / 2, atoms = x.width > 128 ? 2 : 1;
      const int a0 = x.a0 + (int)rank * 128, row0 = x.begin + x.b0, b0 = row0 + (int)rank * half;
      const int w_tile = x.e * g.n_tiles + a0 / 128;  // (rows past N have no scales of their own: any, for zeros)
      int box = BOXES - 1;
#pragma unroll
      for (int i = BOXES - 2; i >= 0; --i)
        if (half > box_rows(i + 1)) box = i;
      const CUtensorMap* columns = &tmX.box[box];
      const uint32_t bytes = 2 * (SUB + SCALES + box_rows(box) * 128 + atoms * SCALES);
      for (int kb = 0; kb < blocks; ++kb) {
        ok = all_ok(mbar_wait(&empty[stage], phase ^ 1u, ctx, SITE_EMPTY));
        if (!ok) break;
        const uint32_t bar = full_leader0 + stage * 8u;
        uint8_t* sA = smem + stage * STAGE_BYTES;
        if (elect_one()) {
          if (leader) mbar_arrive_expect_tx(&full[stage], bytes);
          tma_load_3d_pair(sA, &tmW, bar, kb * 128, a0, x.e);
          tma_load_3d_pair(sA + OFF_SFA, &tmWs, bar, 0, 2 * kb, w_tile);
          tma_load_2d_pair(sA + SUB, columns, bar, kb * 128, b0);
          tma_load_2d_pair(sA + OFF_SFB, &tmXs, bar, row0 * 8, 2 * kb);
          if (atoms == 2) tma_load_2d_pair(sA + OFF_SFB + SCALES, &tmXs, bar, (row0 + 128) * 8, 2 * kb);
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------ MMA issuer (leader)
    if (leader) {
      int stage = 0;
      uint32_t phase = 0;
      const uint32_t ring = smem_u32(smem);
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
      for (int i = 0; ok; ++i) {
        const Tile x = next_tile(i);
        if (x.e < 0) {
          ok = x.e == -1;
          break;
        }
        const uint32_t slot = i & 1, d_tmem = tmem_u + slot * CAP;
        const uint32_t n_bits = (uint32_t)(x.width >> 3) << 17;
        const uint32_t idesc0 = umma_idesc_mxf4(256, 0, 0) | n_bits, idesc2 = umma_idesc_mxf4(256, 0, 2) | n_bits;
        ok = all_ok(mbar_wait(&tmem_empty[slot], (i >> 1 & 1) ^ 1u, ctx, SITE_TMEM_EMPTY));
        if (!ok) break;
        tc_fence_after();
        for (int kb = 0; kb < blocks; ++kb) {
          ok = all_ok(mbar_wait(&full[stage], phase, ctx, SITE_FULL));
          if (!ok) break;
          tc_fence_after();
          const uint32_t base = ring + stage * STAGE_BYTES;
          const uint64_t a0 = umma_desc_sw128(base), b0 = umma_desc_sw128(base + SUB);
          const uint64_t sfa0 = umma_desc(base + OFF_SFA, 16, 128, 0), sfb0 = umma_desc(base + OFF_SFB, 16, 128, 0);
          const int bytes = g.pitch - kb * 128;  // of codes from here on
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (h * 64 >= bytes) break;  // no such run of 128 values
              const uint32_t sfb = tmem_u + SF_COL + h * 16, sfa = sfb + 8;
              tmem_cp_scales<2>(sfb, sfb0 + h * 32);  // 512 bytes on
              if (x.width > 128) tmem_cp_scales<2>(sfb + 4, sfb0 + 64 + h * 32);
              tmem_cp_scales<2>(sfa, sfa0 + h * 32);
              umma_mxf4<2>(d_tmem, a0 + 4 * h, b0 + 4 * h, idesc0, sfa, sfb, h == 0 && kb == 0 ? 0u : 1u);
              if (h * 64 + 32 < bytes) umma_mxf4<2>(d_tmem, a0 + 4 * h + 2, b0 + 4 * h + 2, idesc2, sfa, sfb, 1u);
            }
            umma_commit_cg2_mc(&empty[stage], 0x3);
            if (kb + 1 == blocks) umma_commit_cg2_mc(&tmem_full[slot], 0x3);
          }
          __syncwarp();
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == EPILOGUE + 2) {
    // ------------------------------------------------------- tiles, in order
    const int64_t num_tiles = (int64_t)s_first[g.E] * tab.panels;
    for (int i = 0;; ++i) {
      // Back and forth over the pairs.
      const int64_t t = (int64_t)i * pairs + ((i & 1) ? pairs - 1 - pair : pair);
      Tile x;
      x.e = -1;
      if (t < num_tiles) x = tile_of(t, g, tab);
      const int at = i % TILES;
      ok = all_ok(mbar_wait(&tile_empty[at], (i / TILES & 1) ^ 1u, ctx, SITE_TILE));
      if (!ok) break;
      if (lane == 0) {
        s_tiles[at] = x;
        mbar_arrive(&tile_full[at]);
      }
      __syncwarp();
      if (x.e < 0) break;
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3;           // TMEM lane quarter this warp may access
    const int side = (warp - 2) / 4;  // which half of a tile's columns it takes
    uint32_t* stage_c = reinterpret_cast<uint32_t*>(smem + OFF_C + (warp - 2) * RUN * 32 * 2);  // [RUN / 2 pairs][32]
    const uint32_t tmem_empty_leader0 = mapa_shared(smem_u32(&tmem_empty[0]), 0);
    const uint32_t t_quarter = tmem_base + ((uint32_t)(q * 32) << 16);
    for (int i = 0; ok; ++i) {
      const Tile x = next_tile(i);
      if (x.e < 0) {
        ok = x.e == -1;
        break;
      }
      const int cols = x.width / 2;  // of this warp, a multiple of 8
      const int d0 = side * cols;    // its first column in the tile
      const uint32_t slot = i & 1;
      const int a_warp = x.a0 + (int)rank * 128 + q * 32;  // this warp's first row
      const float bias =
          g.bias && a_warp + lane < g.N ? to_float(static_cast<const TO*>(g.bias)[a_warp + lane]) : 0.f;
      ok = all_ok(mbar_wait(&tmem_full[slot], i >> 1 & 1, ctx, SITE_TMEM_FULL));
      if (!ok) break;
      tc_fence_after();
      // Columns RUN c + 2 j and the next of this thread's row, as outputs (a
      // last run is read whole; what is past it is not used).
      uint32_t out[4][RUN / 2];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c * RUN >= cols) break;
        uint32_t v[RUN];
        tmem_ld_32x32b_x32(t_quarter + slot * CAP + (uint32_t)(d0 + c * RUN), v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < RUN / 2; ++j)
          out[c][j] = pack2(TO(), __uint_as_float(v[2 * j]) + bias, __uint_as_float(v[2 * j + 1]) + bias);
      }
      // This warp's share read: hand it back to the MMA issuer.
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(tmem_empty_leader0 + slot * 8u);
      if (a_warp >= g.N) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int b = x.b0 + d0 + c * RUN;
        const int n = min(min(RUN, cols - c * RUN), x.rows - b);  // columns to store
        if (n <= 0) break;
        uint16_t* y = static_cast<uint16_t*>(g.Y) + ((int64_t)x.begin + b) * g.ldy + a_warp;
        if (g.vec_out && n == RUN) {
          // Half a run at a time by TMA, staged in two buffers in turn.
          uint16_t* b16 = reinterpret_cast<uint16_t*>(stage_c);
#pragma unroll
          for (int u = 0; u < 2; ++u, b16 += RUN / 2 * 32) {
            if (lane == 0) tma_store_wait_read<1>();  // the store that used this buffer has read it
            __syncwarp();
#pragma unroll
            for (int j = 0; j < RUN / 4; ++j) {
              const uint32_t two = out[c][u * (RUN / 4) + j];
              b16[(2 * j) * 32 + lane] = (uint16_t)(two & 0xFFFFu);
              b16[(2 * j + 1) * 32 + lane] = (uint16_t)(two >> 16);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_2d(&tmY, b16, a_warp, x.begin + b + u * (RUN / 2));
              tma_store_commit();
            }
          }
        } else if (g.vec_out) {
          if (lane == 0) tma_store_wait_read<0>();
          // Transposed through shared memory as pairs of columns: a lane reads 8
          // rows of a pair and stores 16 bytes of each column.
          __syncwarp();  // the run before has been read
#pragma unroll
          for (int j = 0; j < RUN / 2; ++j) stage_c[j * 32 + lane] = out[c][j];
          __syncwarp();
          const int a = lane % 4 * 8;
#pragma unroll
          for (int u = 0; u < RUN / 16; ++u) {
            const int two = u * 8 + lane / 4;
            const uint4 l = *reinterpret_cast<const uint4*>(stage_c + two * 32 + a);
            const uint4 h = *reinterpret_cast<const uint4*>(stage_c + two * 32 + a + 4);
            uint16_t* to = y + (2 * two) * g.ldy + a;
            if (a_warp + a < g.N) {
              if (2 * two < n)
                *reinterpret_cast<uint4*>(to) =
                    make_uint4(__byte_perm(l.x, l.y, 0x5410), __byte_perm(l.z, l.w, 0x5410),
                               __byte_perm(h.x, h.y, 0x5410), __byte_perm(h.z, h.w, 0x5410));
              if (2 * two + 1 < n)
                *reinterpret_cast<uint4*>(to + g.ldy) =
                    make_uint4(__byte_perm(l.x, l.y, 0x7632), __byte_perm(l.z, l.w, 0x7632),
                               __byte_perm(h.x, h.y, 0x7632), __byte_perm(h.z, h.w, 0x7632));
            }
          }
        } else if (a_warp + lane < g.N) {
          // Rows of Y on odd boundaries: 64 bytes a column and warp.
          y += lane;
#pragma unroll
          for (int j = 0; j < RUN / 2; ++j) {
            if (2 * j < n) y[(2 * j) * g.ldy] = (uint16_t)(out[c][j] & 0xFFFFu);
            if (2 * j + 1 < n) y[(2 * j + 1) * g.ldy] = (uint16_t)(out[c][j] >> 16);
          }
        }
      }
    }
    // The CTA may exit once its last stores have read their staging buffers.
    if (lane == 0) tma_store_wait_read<0>();
  }

  // ------------------------------------------------------------- teardown
  // A wait of either CTA ran out: both stay until what is in flight between them
  // (copies, the pair's MMAs and their arrivals) has ended.
  if (!ok && lane < 2) store_cluster(mapa_shared(smem_u32(s_abort), lane), 1);
  __syncwarp();
  tc_fence_before();
  cluster_sync();
  if (*s_abort) settle();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<2>(tmem_base, 512);
  }
}

template <typename TO>
int launch(const F4Problem& p) {
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev))) return rc;
  F4Args g = {};
  if ((rc = wait_ctx(&g.ctx))) return rc;
  g.offsets = p.offsets;
  g.E = (int)p.E, g.R = (int)p.R, g.N = (int)p.N;
  g.pitch = (int)f4_pitch(p.K);
  g.n_tiles = (int)((p.N + 127) / 128);
  g.Y = p.Y, g.ldy = p.ldy, g.bias = p.bias;
  g.pdl = pdl_enabled() ? 1 : 0;
  ColumnMaps tX;
  CUtensorMap tW, tWs, tXs;
  if ((rc = f4_weight_map(p, &tW)) || (rc = f4_weight_scale_map(p, &tWs))) return rc;
  for (int i = 0; i < BOXES; ++i)
    if ((rc = f4_token_map(p, box_rows(i), &tX.box[i]))) return rc;
  if ((rc = f4_token_scale_map(p, &tXs))) return rc;
  const int64_t tiles = (p.N + 255) / 256 * (p.R / 128 + std::min(p.E, p.R));  // at most
  if (tiles > INT32_MAX / 2) return fail(KEBAB_EINVAL, "gemm_f4: too many tiles");
  // Whole runs of 8 (N too: a run stays within its row).
  CUtensorMap tY = tXs;  // not used unless vec_out
  g.vec_out = (reinterpret_cast<uintptr_t>(p.Y) & 15u) == 0 && g.ldy % 8 == 0 && g.N % 8 == 0;
  if (g.vec_out) {
    const uint64_t dims[2] = {(uint64_t)p.N, (uint64_t)p.R}, strides[1] = {(uint64_t)p.ldy * 2};
    const uint32_t box[2] = {32, RUN / 2};
    if ((rc = make_tmap(&tY, p.Y, p.out, 2, dims, strides, box, 0))) return rc;
  }
  auto kern = f4_umma_kernel<TO>;
  const int smem = smem_bytes(g.E);
  // Once per device and instantiation: the shared-memory opt-in and how many pairs fit.
  static std::once_flag once[64];
  static cudaError_t err[64];
  static int max_pairs[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    constexpr int most = smem_bytes(kMaxExperts);
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    max_pairs[di] = dev->sm_count / 2;
    if (err[di] != cudaSuccess) return;
    PdlLaunch q(dim3(2 * max_pairs[di]), dim3(THREADS), most, nullptr, 2);
    q.cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &q.cfg) == cudaSuccess && n > 0)
      max_pairs[di] = std::min(n, max_pairs[di]);
    (void)cudaGetLastError();
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  const int pairs = (int)std::min<int64_t>(tiles, max_pairs[di]);
  PdlLaunch ln(dim3(2 * pairs), dim3(THREADS), smem, p.stream, 2);
  const cudaError_t e = cudaLaunchKernelEx(&ln.cfg, kern, tW, tWs, tX, tXs, tY, (const F4Args)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "4-bit tcgen05 launch");
}
}  // namespace

int launch_f4_umma(const F4Problem& p) {
  return p.out == KEBAB_F16 ? launch<__half>(p) : launch<__nv_bfloat16>(p);
}

}  // namespace kb
