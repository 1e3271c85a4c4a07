// Grouped and 8-bit integer products on the tensor cores: persistent CTA pairs
// (cta_group::2) over the tiles of every group, whatever their sizes.
//
// The MMA's rows are the output's contiguous dimension and its columns the
// other one, so that a lane of TMEM is a column of the row-major result:
//   forward (RC, RR)  rows: n (a W_e panel), columns: up to 256 rows of the
//                     group, contraction: k
//   dw                rows: the contiguous dimension of dW_e, columns: the
//                     other, contraction: the group's rows
// A tile is a panel of 512 rows (two MMAs of 256 that share the staged columns)
// or, where that would leave the pairs few tiles each, of 256. Its halves take
// turns on two accumulators of up to 256 columns. With 512-row panels both are
// in use at once, so the second half runs one K-block behind the first: each
// accumulator then has two K-blocks' MMAs of the other half (1024 cycles)
// between its last MMA and the next tile's first, in which 8 epilogue warps read
// it into registers (as pairs of outputs) and hand it back; they store
// afterwards. One half at a time, in a loop: unrolled over both, the epilogue
// was bound by fetching its instructions (dw of 352 rows over 108 experts, 2552
// x 2648: 1000 us against 656). Tiles of 8 K-blocks or more store by TMA, whose
// pace leaves the operands' copies alone: 32768 x 8192 x 4096 over 8 groups 1757
// us against 1810 with stores from registers, 24831 x 7112 x 776 277 against 284,
// dw of 32 groups of 512 rows, 4096 x 2048, 240 against 246. Shorter ones store
// from registers (dw of 43 groups of 95 rows, 4040 x 1272, 165 us against 181 by
// TMA).
//
// Ragged sizes cost what they are: a forward tile is as wide as its rows need
// (a multiple of 32; N is a field of the instruction descriptor), a group of
// 514 rows gives tiles of 192, 192 and 160 columns and not 256, 256 and 32, and
// no group is padded in memory. Which tile belongs to which group is worked out
// on the device: every CTA sorts the groups by their tiles' cost (widest, or in
// dw longest, first) and sums them up for itself, and the pairs take the tiles
// in turn, back and forth, which leaves their loads within a tile of each other.
// A group's tiles stay together, so that its weights are read once: with the
// last, narrower tiles of all groups at the end, 16381 x 4096 x 2048 over 14
// groups took 252 us and 464 MB from memory, and takes 243 and 322.
//
// Edges: a forward tile may read past its group's end (the columns are not
// stored; a column does not reach its neighbours). In dw the contraction runs
// over rows, so rows past the group's end have to be zeros in both operands
// (a NaN there would spread): the last 16-row step is cleared in shared memory
// after it has landed, and steps beyond it are not issued.
//
// Ring: 4 stages of 48 KB a CTA, each one 128-byte K-block (64 16-bit or 128
// 8-bit elements) of a 512-row panel and its columns, or two K-blocks of a
// 256-row panel where no tile is wider than 128 columns (few rows: bound by the
// weights' bytes, and 256 contiguous bytes a weight row and stage are fetched
// faster than 128); else 6 stages of 32 KB. Warps: TMA producer, MMA issuer, 8
// or (dw) 16 epilogue warps, and one that works out the tiles ahead of them (finding a
// tile's place takes about 2000 cycles, as long as 16 MMAs).
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
  int vec_out;  // rows of Y on 16-byte boundaries
  void* Y;
  int64_t ldy;
  const float* scale;
  const float* w_scale;
  const void* bias;
  int pdl;
  int sort;
  WaitCtx ctx;
};

// Epilogue warps: a set of 8 that takes every half in turn, or (dw) one for each
// accumulator. dw's contraction is short and its outputs many, so that what the
// epilogue takes to store a half would delay its reading of the next: 16384 x
// 4096 x 2048, burst, 1024 rows a group 204 us against 222 with one set, 256 rows
// 378 against 405. The forward tiles are longer, and the registers that a thread
// then has too few: 32768 x 8192 x 4096 over 8 groups 1808 us with one, 1853 with
// two.
template <int MODE>
struct Warps {
  static constexpr int SETS = MODE == MODE_DW ? 2 : 1;
  static constexpr int EPILOGUE = 8 * SETS;
  static constexpr int TAIL = MODE == MODE_DW ? 1 : 0;        // the one that writes zeros
  static constexpr int THREADS = 32 * (EPILOGUE + TAIL + 3);  // and producer, issuer, tiles
};
// Tiles are sorted by cost where that can pay: from 2048 rows (a product of
// fewer takes about as long as its weights' bytes in any order), and up to 512
// groups (the ranks take groups^2 / 352 (dw 640) comparisons a thread).
constexpr int SORT_ROWS = 2048, SORT_LIMIT = 512;

template <int SETS>
struct GSmem {
  static constexpr int SUB = 128 * 128;  // 128 rows of 128 bytes: one K-block of one operand
  static constexpr int RING = 12 * SUB;
  static constexpr int MAX_STAGES = 6;
  static constexpr int OFF_C = RING;
  static constexpr int RUN = 32 / SETS;  // columns that an epilogue warp stores at a time
  static constexpr int C_SUB = RUN * 32 * 2 + 128 * 4;  // its: a run of columns of 32 values, 128 scales
  static constexpr int OFF_BAR = OFF_C + 8 * SETS * C_SUB;
  // full, empty, tail_full, tail_done a stage; tmem_full and tmem_empty twice
  static constexpr int TILES = 4;  // descriptions of tiles in flight: full and empty each
  static constexpr int NUM_BARS = 4 * MAX_STAGES + 4 + 2 * TILES;
  static constexpr int OFF_TILES = (OFF_BAR + NUM_BARS * 8 + 8 + 15) / 16 * 16;  // after the TMEM address, abort
  static constexpr int OFF_TABLE = OFF_TILES + TILES * 32;
  // first[E + 1] (int), entry[E] (uint16, sorted only)
  static constexpr int bytes(int E, bool sorted) {
    return OFF_TABLE + (E + 1) * 4 + (sorted ? E * 2 : 0) + 1024;
  }
  static constexpr int ALLOC =
      OFF_TABLE + std::max((kMaxExperts + 1) * 4, (SORT_LIMIT + 1) * 4 + SORT_LIMIT * 2) + 1024;
  static_assert(ALLOC <= 232448, "shared memory budget exceeded");
};

// a / b for 0 <= a, 0 < b. Below 2^22 by a float quotient, put right by one
// step: every role divides a few times a tile, on its critical path.
__device__ __forceinline__ int divide(int a, int b) {
  if (a >= 1 << 22) return a / b;
  int q = (int)__fdividef((float)a, (float)b);
  const int r = a - q * b;
  if (r < 0) --q;
  else if (r >= b) ++q;
  return q;
}

// The tiles in the order in which they are dealt out. Group entry[i] (unsorted:
// group i) has the column blocks first[i] .. first[i + 1] - 1, each of `panels`
// tiles.
struct Table {
  const int* first;
  const uint16_t* entry;
  bool sorted;
  int panels;             // tiles along the MMA-row side
  int nsub;               // 256-row halves of a panel
  int kps;                // K-blocks a stage
  int cap;                // columns that a tile may have
};

struct alignas(16) Tile {
  int e, a0, b0, width;  // group (-1: no more tiles), first row and column of the tile, its columns (a multiple of 32)
  int nsub;              // halves of the panel that exist here
  int begin, rows;       // the group's rows
  int blocks;            // 128-byte K-blocks of the contraction
};

// Columns of a group's tiles: equal shares of at most `cap`, in runs of 32, the wider ones first.
struct Widths {
  int count, narrow, wider;  // `wider` of the tiles have 32 columns more
  __device__ __forceinline__ Widths(int rows, int cap) {
    const int runs = (rows + 31) / 32;
    count = (rows + cap - 1) / cap;
    const int per = count > 1 ? divide(runs, count) : runs;
    wider = runs - per * count;
    narrow = per * 32;
  }
  __device__ __forceinline__ int widest() const { return narrow + (wider > 0 ? 32 : 0); }
};

// Tile `local` of panels x blocks: eight panels share the passes over the
// columns, so that the 74 pairs hold about 8 x 9 tiles at a time.
__device__ __forceinline__ void raster(int local, int panels, int blocks, int& pa, int& cb) {
  if (blocks == 1) {
    pa = local;
    cb = 0;
  } else {
    const int group = divide(local, 8 * blocks), in_group = local - group * 8 * blocks;
    const int height = min(8, panels - group * 8);
    cb = divide(in_group, height);
    pa = group * 8 + in_group - cb * height;
  }
}

template <int MODE, int EPB>
__device__ __forceinline__ Tile tile_of(int t, const TileArgs& g, const Table& tab) {
  Tile x;
  int lo = 0, hi = g.E - 1;  // the last group that starts at or before t
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first[mid] * tab.panels <= t) lo = mid;
    else hi = mid - 1;
  }
  const int local = t - tab.first[lo] * tab.panels;
  x.e = tab.sorted ? tab.entry[lo] : lo;
  group_range(g.offsets, x.e, g.R, x.begin, x.rows);
  int pa, cb;
  if (MODE == MODE_DW) {
    raster(local, tab.panels, (g.DB + 255) / 256, pa, cb);
    x.width = 256;
    x.b0 = cb * 256;
    x.blocks = (x.rows + EPB - 1) / EPB;
  } else {
    const Widths w(x.rows, tab.cap);
    raster(local, tab.panels, w.count, pa, cb);
    x.width = w.narrow + (cb < w.wider ? 32 : 0);
    x.b0 = cb * w.narrow + min(cb, w.wider) * 32;
    x.blocks = (g.K + EPB - 1) / EPB;
  }
  x.a0 = pa * 256 * tab.nsub;
  x.nsub = min(tab.nsub, (g.DA - x.a0 + 255) / 256);
  return x;
}

// The same from lane 0, for code of a whole warp.
__device__ __forceinline__ Tile uniform(const Tile& x) {
  auto u = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
  return {u(x.e), u(x.a0), u(x.b0), u(x.width), u(x.nsub), u(x.begin), u(x.rows), u(x.blocks)};
}

// Block-wide sum of one value a thread before this thread's; `total` of all.
template <int THREADS>
__device__ __forceinline__ int scan_before(int v, int* sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int at = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, at, d);
    if (lane >= d) at += up;
  }
  if (lane == 31) sums[warp] = at;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    total += s;
  }
  __syncthreads();
  return before + at - v;
}

// Makes the table, by all threads of the CTA. `scratch`: 3 ints a group and 40.
template <int MODE, bool I8>
__device__ __forceinline__ Table make_table(const TileArgs& g, int pairs, int* first, uint16_t* entry, int* scratch) {
  constexpr bool DW = MODE == MODE_DW;
  constexpr int THREADS = Warps<MODE>::THREADS;
  // 512-row panels from this many 256-row tiles a pair (0: never). Measured
  // under the power cap, us: forward 16381 x 4096 x 2048 over 14 uneven groups
  // (15 tiles a pair) 245 against 252; dw with 7 tiles a pair (4 groups of 8192
  // rows) 430 against 477: a 256-row dw tile needs four copies a K-block, whose
  // issue is as long as its MMAs. 8-bit: 4093 x 28672 x 8192 735 against 682
  // (the epilogue, which scales every sum, stands between two tiles' MMAs).
  constexpr int WIDE_FROM = I8 ? 0 : DW ? 4 : 8;
  int* sums = scratch;  // [32]
  int* cost = scratch + 32;
  const int tb = (g.DB + 255) / 256;
  const bool sorted = g.sort;
  const int n = g.E;
  int wide = 0;  // some tile of more than 128 columns
  int total = 0;
  int cap = 256;
  if (!sorted) {
    // The widest tile of 256, 192 or 128 columns, by the waves over the pairs and
    // the rows that a tile's K-block copies (256 of the panel and its columns,
    // which take as long as its MMAs or longer). 128 also keeps two K-blocks a
    // stage. 1267 rows over 3 groups, 3320 x 5224: 76 us with 256 (78 tiles on 74
    // pairs), 68 so. Of 65536 rows or more (more groups than are sorted) it is 256.
    if (!DW && g.R < 65536) {
      int c256 = 0, c192 = 0, c128 = 0;
      for (int i0 = 0; i0 < n; i0 += THREADS) {
        int begin, rows = 0, two, one;
        if (i0 + (int)threadIdx.x < n) group_range(g.offsets, i0 + threadIdx.x, g.R, begin, rows);
        scan_before<THREADS>((rows + 255) / 256 << 16 | (rows + 191) / 192, sums, two);
        scan_before<THREADS>((rows + 127) / 128, sums, one);
        c256 += two >> 16;
        c192 += two & 0xffff;
        c128 += one;
      }
      const int panels = (g.DA + 255) / 256;
      auto cost = [&](int blocks, int width) {
        return ((int64_t)blocks * panels + pairs - 1) / pairs * (256 + width);
      };
      if (cost(c192, 192) < cost(c256, 256)) cap = 192;
      if (cost(c128, 128) <= min(cost(c192, 192), cost(c256, 256))) cap = 128;
    }
    for (int i0 = 0; i0 < n; i0 += THREADS) {
      const int i = i0 + threadIdx.x;
      int b = 0;
      if (i < n) {
        int begin, rows;
        group_range(g.offsets, i, g.R, begin, rows);
        b = DW ? tb : (rows + cap - 1) / cap;
        wide |= DW || (cap > 128 && rows > 128);
      }
      int all;
      const int at = total + scan_before<THREADS>(b, sums, all);
      if (i < n) first[i] = at;
      total += all;
    }
    wide = __syncthreads_or(wide);
  } else {
    int* blocks = cost + (n + 3) / 4 * 4;  // column blocks of the group
    int* by_rank = blocks + n;
    for (int i = threadIdx.x; i < (n + 3) / 4 * 4; i += THREADS) {
      int c = -1, b = 0;
      if (i < n) {
        int begin, rows;
        group_range(g.offsets, i, g.R, begin, rows);
        if (DW) {
          c = rows;
          b = tb;
        } else {
          const Widths w(rows, 256);
          c = w.widest();
          b = w.count;
        }
        wide |= DW || c > 128;
        blocks[i] = b;
      }
      cost[i] = c;
    }
    wide = __syncthreads_or(wide);
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const int c = cost[i];
      int rank = 0;
      for (int j = 0; j < n; j += 4) {
        const int4 o = *reinterpret_cast<const int4*>(cost + j);
        rank += (o.x > c || (o.x == c && j < i)) + (o.y > c || (o.y == c && j + 1 < i)) +
                (o.z > c || (o.z == c && j + 2 < i)) + (o.w > c || (o.w == c && j + 3 < i));
      }
      entry[rank] = (uint16_t)i;
      by_rank[rank] = blocks[i];
    }
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += THREADS) {
      const int i = i0 + threadIdx.x;
      int all;
      const int at = total + scan_before<THREADS>(i < n ? by_rank[i] : 0, sums, all);
      if (i < n) first[i] = at;
      total += all;
    }
  }
  if (threadIdx.x == 0) first[n] = total;
  Table tab;
  tab.first = first;
  tab.entry = entry;
  tab.sorted = sorted;
  const int p256 = (g.DA + 255) / 256;
  tab.nsub = WIDE_FROM > 0 && (int64_t)total * p256 >= (int64_t)WIDE_FROM * pairs ? 2 : 1;
  tab.panels = tab.nsub == 2 ? (g.DA + 511) / 512 : p256;
  tab.kps = tab.nsub == 1 && !wide ? 2 : 1;
  tab.cap = cap;
  return tab;
}

// Forward: the rows of X in boxes of 64, 32 and 16, for shares of a tile's
// columns under 128.
struct ColumnMaps {
  CUtensorMap box[3];
};

template <typename TO, bool I8, int MODE>
__global__ void __launch_bounds__(Warps<MODE>::THREADS, 1)
    grouped_umma_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                        const __grid_constant__ ColumnMaps tmBs, const __grid_constant__ CUtensorMap tmC,
                        const TileArgs g) {
  using W = Warps<MODE>;
  using L = GSmem<W::SETS>;
  constexpr bool DW = MODE == MODE_DW;
  constexpr bool A_MN = MODE != MODE_RC, B_MN = DW;
  constexpr int PACED_FROM = 8;  // K-blocks of a tile from which its stores go by TMA
  constexpr int EPB = I8 ? 128 : 64;  // elements of the contraction in a K-block
  constexpr int STAGES = L::MAX_STAGES;
  constexpr uint32_t IDESC = (I8 ? umma_idesc_i8(256, 0) : umma_idesc_f16(256, 0, ElemTraits<TO>::kBf16)) |
                             (A_MN ? (1u << 15) : 0u) | (B_MN ? (1u << 16) : 0u);

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  uint64_t* tail_full = empty + STAGES;  // dw: this CTA's bytes of a group's last stage, where it is to be cleared
  uint64_t* tail_done = tail_full + STAGES;  // dw, in the leader: both CTAs have cleared their shares of it
  uint64_t* tmem_full = tail_done + STAGES;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* tile_full = tmem_empty + 2;
  uint64_t* tile_empty = tile_full + L::TILES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full + L::NUM_BARS);
  uint32_t* s_abort = tmem_slot + 1;  // some wait of the pair ran out
  Tile* s_tiles = reinterpret_cast<Tile*>(smem + L::OFF_TILES);
  int* s_first = reinterpret_cast<int*>(smem + L::OFF_TABLE);
  uint16_t* s_entry = reinterpret_cast<uint16_t*>(s_first + g.E + 1);

  // The shuffle tells the compiler that a warp takes one path. The producer and
  // the issuer run with all lanes, one of which is elected at each copy or MMA,
  // so that addresses and descriptors stay in uniform registers: a branch on
  // the lane around the whole loop cost about 100 cycles an MMA to issue, of
  // the 128 that a 256 x 256 x 16 takes.
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const WaitCtx& ctx = g.ctx;

  cluster_arrive_release();  // this CTA has started
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
      mbar_init(&tail_full[s], 1);
      mbar_init(&tail_done[s], 2);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], 8 * 2);
    }
    for (int a = 0; a < L::TILES; ++a) {
      mbar_init(&tile_full[a], 1);
      mbar_init(&tile_empty[a], W::EPILOGUE + W::TAIL + 1 + (leader ? 1 : 0));  // the warps that read descriptions
    }
    *s_abort = 0;
    fence_barrier_init();
  }
  __syncwarp();
  // The pair allocates together: not before the other CTA has started. With
  // kernels of several streams on the SMs a pair that did hung in it.
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
  const Table tab = make_table<MODE, I8>(g, pairs, s_first, s_entry, reinterpret_cast<int*>(smem));
  // The table's scratch is in the ring: order it before the copies into it.
  fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  cluster_wait_acquire();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int kps = tab.kps;
  // A stage: the panel's K-blocks (or halves), then the columns'.
  const int stages = tab.nsub + kps == 3 ? 4 : 6;
  const int a_bytes = tab.nsub * kps * L::SUB, stage_bytes = a_bytes + L::SUB;
  // The i-th tile of this pair, for a whole warp; e is -1 after the last, and -2
  // where the wait for it ran out.
  auto next_tile = [&](int i) {
    const int at = i % L::TILES;
    Tile x;
    if (__all_sync(0xffffffffu, mbar_wait(&tile_full[at], i / L::TILES & 1, ctx, SITE_TILE))) x = uniform(s_tiles[at]);
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
    const uint32_t tail_mine0 = mapa_shared(smem_u32(&tail_full[0]), rank);
    for (int i = 0; ok; ++i) {
      const Tile x = next_tile(i);
      if (x.e < 0) {
        ok = x.e == -1;
        break;
      }
      const int half = x.width / 2;
      const int a0 = x.a0 + (int)rank * 128, b0 = x.b0 + (int)rank * half;
      const uint32_t block_bytes = x.nsub * L::SUB + half * 128;
      const bool has_tail = DW && (x.rows & 15) != 0, early = has_tail && x.blocks > 1;
      for (int j = 0; j < x.blocks; j += kps) {
        // The tail's K-block comes before the one that precedes it, which gives
        // the time to clear it.
        const int kb = early && j >= x.blocks - 2 ? 2 * x.blocks - 3 - j : j;
        ok = all_ok(mbar_wait(&empty[stage], phase ^ 1u, ctx, SITE_EMPTY));
        if (!ok) break;
        // A group's last stage that does not end on a 16-row step: each CTA
        // waits for its own bytes and clears the rows past the end (`full` only
        // moves on).
        const bool tail = has_tail && kb + 1 == x.blocks;
        const int nq = min(kps, x.blocks - kb);
        const uint32_t bar = (tail ? tail_mine0 : full_leader0) + stage * 8u;
        uint8_t* sA = smem + stage * stage_bytes;
        uint8_t* sB = sA + a_bytes;
        if (elect_one()) {
          if (tail) mbar_arrive_expect_tx(&tail_full[stage], block_bytes);
          if (leader && tail) mbar_arrive(&full[stage]);
          else if (leader) mbar_arrive_expect_tx(&full[stage], 2 * nq * block_bytes);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q >= nq) break;
            const int k0 = (kb + q) * EPB;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (s >= x.nsub) break;
              uint8_t* dst = sA + (q + s) * L::SUB;
              const int as = a0 + s * 256;
              if constexpr (MODE == MODE_RC) {
                tma_load_3d_pair(dst, &tmA, bar, k0, as, x.e);
              } else if constexpr (MODE == MODE_RR) {
                tma_load_3d_pair(dst, &tmA, bar, as, k0, x.e);
                tma_load_3d_pair(dst + 8192, &tmA, bar, as + 64, k0, x.e);
              } else {
                tma_load_2d_pair(dst, &tmA, bar, as, x.begin + k0);
                tma_load_2d_pair(dst + 8192, &tmA, bar, as + 64, x.begin + k0);
              }
            }
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (q >= nq) break;
            const int k0 = (kb + q) * EPB;
            uint8_t* dst = sB + q * half * 128;
            if constexpr (DW) {
              tma_load_2d_pair(dst, &tmB, bar, b0, x.begin + k0);
              tma_load_2d_pair(dst + 8192, &tmB, bar, b0 + 64, x.begin + k0);
            } else if (half == 128) {
              tma_load_2d_pair(dst, &tmB, bar, k0, x.begin + b0);
            } else {
              int r = 0;
#pragma unroll
              for (int m = 0; m < 3; ++m) {
                if (half & (64 >> m)) {
                  tma_load_2d_pair(dst + r * 128, &tmBs.box[m], bar, k0, x.begin + b0 + r);
                  r += 64 >> m;
                }
              }
            }
          }
        }
        __syncwarp();
        if (++stage == stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------ MMA issuer (leader)
    if (leader) {
      int stage = 0;
      uint32_t phase = 0, tail_parity = 0;
      uint32_t halves = 0;  // accumulators used so far: slot = bit 0, phase = bit 1
      const uint32_t ring = smem_u32(smem);
      const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem_base, 0);
      // The MMAs of half `s` over the stage `at`, whose first K-block is kb;
      // `left`: dw's rows of the group from there on.
      auto issue = [&](const Tile& x, uint32_t idesc, int s, int at, int kb, bool last, int left) {
        const uint32_t slot = (halves + s) & 1u;
        if (kb == 0) {
          if (!all_ok(mbar_wait(&tmem_empty[slot], ((halves + s) >> 1 & 1u) ^ 1u, ctx, SITE_TMEM_EMPTY))) return false;
          tc_fence_after();
        }
        const uint32_t a_addr = ring + at * stage_bytes + s * L::SUB, b_addr = ring + at * stage_bytes + a_bytes;
        const uint32_t d_tmem = tmem_u + slot * 256;
        const uint64_t a0 = operand_desc<A_MN>(a_addr, 0), b0 = operand_desc<B_MN>(b_addr, 0);
        const uint64_t a1 = operand_desc<A_MN>(a_addr + L::SUB, 0);
        const uint64_t b1 = operand_desc<B_MN>(b_addr + x.width / 2 * 128, 0);
        const int nq = min(kps, x.blocks - kb);
        const int steps = DW ? min(4, (left + 15) / 16) : 4;  // of 32 bytes (dw: 16 rows) a K-block
        if (elect_one()) {
          // Addresses in 16 bytes: 32 bytes a step along rows, 16 rows of 128 bytes across them.
          if (!DW || steps == 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t ad = a0 + k * (A_MN ? 128 : 2), bd = b0 + k * (B_MN ? 128 : 2);
              const uint32_t accumulate = k == 0 && kb == 0 ? 0u : 1u;
              if constexpr (I8) umma_i8<2>(d_tmem, ad, bd, idesc, accumulate);
              else umma_f16_cg2(d_tmem, ad, bd, idesc, accumulate);
            }
          } else if constexpr (DW) {
            for (int k = 0; k < steps; ++k)
              umma_f16_cg2(d_tmem, a0 + k * 128, b0 + k * 128, idesc, k == 0 && kb == 0 ? 0u : 1u);
          }
          if (!DW && nq == 2) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t ad = a1 + k * (A_MN ? 128 : 2), bd = b1 + k * (B_MN ? 128 : 2);
              if constexpr (I8) umma_i8<2>(d_tmem, ad, bd, idesc, 1u);
              else umma_f16_cg2(d_tmem, ad, bd, idesc, 1u);
            }
          }
          if (s + 1 == x.nsub) umma_commit_cg2_mc(&empty[at], 0x3);  // the stage's last reader
          if (last) umma_commit_cg2_mc(&tmem_full[slot], 0x3);
        }
        __syncwarp();
        return true;
      };
      for (int i = 0; ok; ++i) {
        const Tile x = next_tile(i);
        if (x.e < 0) {
          ok = x.e == -1;
          break;
        }
        const uint32_t idesc = IDESC | (uint32_t)(x.width >> 3) << 17;
        const bool has_tail = DW && (x.rows & 15) != 0, early = has_tail && x.blocks > 1;
        int before = 0;  // the stage of the K-block before
        for (int kb = 0; kb < x.blocks; kb += kps) {
          const int left = DW ? x.rows - kb * EPB : 0;  // dw: rows of the group in this stage and later
          // Of a group with a tail, the last two K-blocks' stages are the other way round.
          int at = stage;
          uint32_t ph = phase;
          if (early && kb == x.blocks - 2 && ++at == stages) {
            at = 0;
            ph ^= 1u;
          }
          if (early && kb == x.blocks - 1) at = stage == 0 ? stages - 1 : stage - 1;
          if (has_tail && kb + 1 == x.blocks) {
            ok = mbar_wait_cluster(&tail_done[at], tail_parity >> at & 1u, ctx, SITE_FULL);
            tail_parity ^= 1u << at;
          } else {
            ok = mbar_wait(&full[at], ph, ctx, SITE_FULL);
          }
          ok = all_ok(ok);
          if (!ok) break;
          tc_fence_after();
          const bool last = kb + kps >= x.blocks;
          ok = issue(x, idesc, 0, at, kb, last, left);
          if (ok && x.nsub == 2 && kb > 0) ok = issue(x, idesc, 1, before, kb - 1, false, EPB);
          if (ok && x.nsub == 2 && last) ok = issue(x, idesc, 1, at, kb, true, left);
          if (!ok) break;
          before = at;
          __syncwarp();
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (x.blocks) halves += x.nsub;
      }
    }
  } else if (warp == W::EPILOGUE + 2) {
    // ------------------------------------------------------- tiles, in order
    const int num_tiles = s_first[g.E] * tab.panels;
    for (int i = 0;; ++i) {
      // Back and forth over the pairs. (64 bits: groups that overlap, as offsets
      // that fall make them, can have up to 2^31 tiles.)
      const int64_t t = (int64_t)i * pairs + ((i & 1) ? pairs - 1 - pair : pair);
      Tile x;
      x.e = -1;
      if (t < num_tiles) x = tile_of<MODE, EPB>((int)t, g, tab);
      const int at = i % L::TILES;
      ok = all_ok(mbar_wait(&tile_empty[at], (i / L::TILES & 1) ^ 1u, ctx, SITE_TILE));
      if (!ok) break;
      if (lane == 0) {
        s_tiles[at] = x;
        mbar_arrive(&tile_full[at]);
      }
      __syncwarp();
      if (x.e < 0) break;
    }
  } else if (DW && warp == W::EPILOGUE + 3) {
    // --------------------------------------- zeros past the ends of dw's groups
    // (by the issuer itself, between two tiles' MMAs, it took 1.3 us a tile)
    int stage = 0;
    uint32_t tail_parity = 0;
    const uint32_t tail_done_leader0 = mapa_shared(smem_u32(&tail_done[0]), 0);
    for (int i = 0;; ++i) {
      const Tile x = next_tile(i);
      if (x.e < 0) {
        ok = x.e == -1;
        break;
      }
      if (x.blocks == 0) {
        // A group without rows: the whole tile, each CTA every other column, 512
        // contiguous bytes a step (108 experts of 2552 x 2648, all but one empty:
        // 306 us, 680 from the epilogue, whose warps write 64 bytes at a time).
        const int b0 = x.b0 + (int)rank, columns = (min(x.b0 + x.width, g.DB) - b0 + 1) / 2;
        const int end = min(x.a0 + x.nsub * 256, g.DA);
        uint16_t* y = static_cast<uint16_t*>(g.Y) + ((int64_t)x.e * g.DB + b0) * g.ldy;
        if (g.vec_out) {
          const int a = x.a0 + lane * 8;
          const bool one = a < end, two = a + 256 < end;
          y += a;
#pragma unroll 8
          for (int c = 0; c < columns; ++c, y += 2 * g.ldy) {
            if (one) *reinterpret_cast<uint4*>(y) = make_uint4(0, 0, 0, 0);
            if (two) *reinterpret_cast<uint4*>(y + 256) = make_uint4(0, 0, 0, 0);
          }
        } else {
          for (int c = 0; c < columns; ++c, y += 2 * g.ldy)
            for (int a = x.a0 + lane; a < end; a += 32) y[a] = 0;
        }
      } else if ((x.rows & 15) != 0) {
        const int at = (stage + max(x.blocks - 2, 0)) % stages;
        ok = all_ok(mbar_wait(&tail_full[at], tail_parity >> at & 1u, ctx, SITE_FULL));
        if (!ok) break;
        // Rows left .. the end of its 16-row step, in every box of 64 columns
        // (128-byte rows; the swizzle stays within a row).
        uint8_t* sA = smem + at * stage_bytes;
        uint8_t* sB = sA + a_bytes;
        const int left = x.rows - (x.blocks - 1) * EPB;
        const int n = (16 - (left & 15)) * 8;
        for (int c = lane; c < n; c += 32) {
          const int to = left * 128 + c * 16;
          const uint4 zero = make_uint4(0, 0, 0, 0);
          for (int box = 0; box < 2 * x.nsub; ++box) *reinterpret_cast<uint4*>(sA + box * 8192 + to) = zero;
          for (int box = 0; box < 2; ++box) *reinterpret_cast<uint4*>(sB + box * 8192 + to) = zero;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tail_done_leader0 + at * 8u);
        __syncwarp();
        tail_parity ^= 1u << at;
      }
      stage = (stage + x.blocks) % stages;
    }
  } else {
    // -------------------------------------------------------------- epilogue
    const int q = warp & 3;             // TMEM lane quarter this warp may access
    const int side = (warp - 2) / 4 % 2;  // which half of a tile's columns it takes
    const uint32_t set = (warp - 2) / 8;  // of two sets, the accumulator it reads
    constexpr int RUN = L::RUN;
    // [RUN / 2 pairs][32 values]
    uint32_t* stage_c = reinterpret_cast<uint32_t*>(smem + L::OFF_C + (warp - 2) * L::C_SUB);
    float* s_scale = reinterpret_cast<float*>(stage_c + RUN / 2 * 32);
    const uint32_t tmem_empty_leader0 = mapa_shared(smem_u32(&tmem_empty[0]), 0);
    const uint32_t t_quarter = tmem_base + ((uint32_t)(q * 32) << 16);
    uint32_t halves = 0;
    for (int i = 0; ok; ++i) {
      const Tile x = next_tile(i);
      if (x.e < 0) {
        ok = x.e == -1;
        break;
      }
      const int limit = DW ? g.DB : x.rows;  // columns end here
      const int cols = x.width / 2;          // of this warp, a multiple of 16
      const int d0 = side * cols;            // its first column in the tile
      if (DW && x.blocks == 0) continue;  // zeros, by another warp
      if constexpr (I8) {
        __syncwarp();
        for (int c = lane; c < cols; c += 32) {
          const int b = x.b0 + d0 + c;
          s_scale[c] = b < limit ? g.scale[x.begin + b] : 0.f;
        }
        __syncwarp();
      }
#pragma unroll 1
      for (int s = 0; s < x.nsub; ++s) {
        const uint32_t slot = halves & 1u, use = halves >> 1;
        ++halves;
        if (W::SETS == 2 && slot != set) continue;
        const int a_warp = x.a0 + s * 256 + (int)rank * 128 + q * 32;  // this warp's first row of the half
        float sw = 0.f, bias = 0.f;
        if constexpr (I8) {
          const int a = a_warp + lane;
          if (a < g.DA) {
            sw = g.w_scale[(int64_t)x.e * g.DA + a];
            if (g.bias) bias = (float)static_cast<const TO*>(g.bias)[a];
          }
        }
        ok = all_ok(mbar_wait(&tmem_full[slot], use & 1u, ctx, SITE_TMEM_FULL));
        if (!ok) break;
        tc_fence_after();
        // Columns RUN c + 2 j and the next of this thread's row, as outputs (an odd
        // last run of 16 is read as 32; what is past it is not used).
        uint32_t out[128 / RUN][RUN / 2];
#pragma unroll
        for (int c = 0; c < 128 / RUN; ++c) {
          if (c * RUN >= cols) break;
          uint32_t v[RUN];
          const uint32_t at = t_quarter + slot * 256 + (uint32_t)(d0 + c * RUN);
          if constexpr (RUN == 32) tmem_ld_32x32b_x32(at, v);
          else tmem_ld_32x32b_x16(at, v);
          tmem_ld_wait();
          if constexpr (I8) {
#pragma unroll
            for (int j = 0; j < RUN; ++j) v[j] = __float_as_uint((float)(int)v[j] * (sw * s_scale[c * RUN + j]) + bias);
          }
#pragma unroll
          for (int j = 0; j < RUN / 2; ++j)
            out[c][j] = pack2(TO(), __uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
        }
        // This warp's share read: hand it back to the MMA issuer.
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(tmem_empty_leader0 + slot * 8u);
        if (a_warp >= g.DA) continue;
#pragma unroll
        for (int c = 0; c < 128 / RUN; ++c) {
          const int b = x.b0 + d0 + c * RUN;
          const int n = min(min(RUN, cols - c * RUN), limit - b);  // columns to store
          if (n <= 0) break;
          uint16_t* y = static_cast<uint16_t*>(g.Y) +
                        (DW ? (int64_t)x.e * g.DB + b : (int64_t)x.begin + b) * g.ldy + a_warp;
          if (g.vec_out && x.blocks >= PACED_FROM && n == RUN) {
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
                if constexpr (DW) tma_store_3d(&tmC, b16, a_warp, b + u * (RUN / 2), x.e);
                else tma_store_2d(&tmC, b16, a_warp, x.begin + b + u * (RUN / 2));
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
              const int pair = u * 8 + lane / 4;
              const uint4 l = *reinterpret_cast<const uint4*>(stage_c + pair * 32 + a);
              const uint4 h = *reinterpret_cast<const uint4*>(stage_c + pair * 32 + a + 4);
              uint16_t* to = y + (2 * pair) * g.ldy + a;
              if (a_warp + a < g.DA) {
                if (2 * pair < n)
                  *reinterpret_cast<uint4*>(to) =
                      make_uint4(__byte_perm(l.x, l.y, 0x5410), __byte_perm(l.z, l.w, 0x5410),
                                 __byte_perm(h.x, h.y, 0x5410), __byte_perm(h.z, h.w, 0x5410));
                if (2 * pair + 1 < n)
                  *reinterpret_cast<uint4*>(to + g.ldy) =
                      make_uint4(__byte_perm(l.x, l.y, 0x7632), __byte_perm(l.z, l.w, 0x7632),
                                 __byte_perm(h.x, h.y, 0x7632), __byte_perm(h.z, h.w, 0x7632));
              }
            }
          } else if (a_warp + lane < g.DA) {
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
  using W = Warps<MODE>;
  using L = GSmem<W::SETS>;
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
  g.sort = p.R >= SORT_ROWS && p.E <= SORT_LIMIT;
  CUtensorMap tA, tB;
  ColumnMaps tBs;
  int64_t tiles;
  if constexpr (!DW) {
    g.DA = (int)p.N;
    g.ldy = p.ldy;
    if (MODE == MODE_RC) rc = map3(&tA, p.W, type, ES, p.E, p.N, p.K, p.ldw, p.w_stride, 128, EPB, 128);
    else rc = map3(&tA, p.W, type, ES, p.E, p.K, p.N, p.ldw, p.w_stride, 64, 64, 128);
    if (rc || (rc = map2(&tB, p.X, type, ES, p.R, p.K, p.ldx, 128, EPB, 128)) ||
        (rc = map2(&tBs.box[0], p.X, type, ES, p.R, p.K, p.ldx, 64, EPB, 128)) ||
        (rc = map2(&tBs.box[1], p.X, type, ES, p.R, p.K, p.ldx, 32, EPB, 128)) ||
        (rc = map2(&tBs.box[2], p.X, type, ES, p.R, p.K, p.ldx, 16, EPB, 128)))
      return rc;
    tiles = (p.N + 255) / 256 * (p.R / 128 + std::min(p.E, p.R));  // at most
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
    tBs = {{tB, tB, tB}};  // not used
    tiles = p.E * ((g.DA + 255) / 256) * ((g.DB + 255) / 256);
  }
  if (tiles > INT32_MAX / 2) return fail(KEBAB_EINVAL, "grouped product: too many tiles");
  // Whole runs of 8 (DA too: a run stays within its row).
  CUtensorMap tC = tA;  // not used unless vec_out
  g.vec_out = (reinterpret_cast<uintptr_t>(p.Y) & 15u) == 0 && g.ldy % 8 == 0 && g.DA % 8 == 0;
  if (g.vec_out) {
    if (DW) rc = map3(&tC, p.Y, p.out, 2, p.E, g.DB, g.DA, g.ldy, g.ldy * g.DB, L::RUN / 2, 32, 0);
    else rc = map2(&tC, p.Y, p.out, 2, p.R, p.N, p.ldy, L::RUN / 2, 32, 0);
    if (rc) return rc;
  }

  auto kern = grouped_umma_kernel<TO, I8, MODE>;
  const int smem = L::bytes(g.E, g.sort);
  // Once per device and instantiation: the shared-memory opt-in and how many pairs fit.
  static std::once_flag once[64];
  static cudaError_t err[64];
  static int max_pairs[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::ALLOC);
    max_pairs[di] = dev->sm_count / 2;
    if (err[di] != cudaSuccess) return;
    PdlLaunch q(dim3(2 * max_pairs[di]), dim3(W::THREADS), L::ALLOC, nullptr, 2);
    q.cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &q.cfg) == cudaSuccess && n > 0)
      max_pairs[di] = std::min(n, max_pairs[di]);
    (void)cudaGetLastError();
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  const int pairs = (int)std::min<int64_t>(tiles, max_pairs[di]);
  PdlLaunch ln(dim3(2 * pairs), dim3(W::THREADS), smem, p.stream, 2);
  const cudaError_t e = cudaLaunchKernelEx(&ln.cfg, kern, tA, tB, tBs, tC, g);
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
