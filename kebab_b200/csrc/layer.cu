// A mixture-of-experts feed-forward layer for up to 16 tokens, in two launches.
//
// The first computes the router's logits (a block an expert; for 8-bit experts
// also the codes of the tokens) and clears what the second counts in. The second
// is one CTA an SM, all resident (a cooperative launch): every CTA finds the
// top-k choices by itself, takes an equal share of the hidden values of all
// chosen experts (a gate row and an up row each), meets the others at a grid
// barrier, and takes an equal share of the rows of the chosen experts' second
// matrices. A choice's outputs go to the workspace, weighted; whoever completes
// a block of 32 outputs adds them up, in the order of the choices, so that the
// results do not depend on who comes first.
//
// Bound by the chosen experts' bytes, and by latency for few of them. Weights
// come by TMA in K-blocks of 128 bytes a row, through a ring of some 200 KB, as
// the row side of tcgen05.mma (up to 128 rows; rows that the CTA does not own
// are not loaded, and what the MMA reads in their place ends in rows that are
// not used). The tokens, or the hidden values of the tokens that chose the
// expert, are the columns, 8 or 16. A warp of its own copies the columns: at the grid
// barrier only it waits, while the second matrices' rows arrive in the ring.
// 1 token, 8 experts of H 2048 and D 1024 in BF16: 31 us (3.3 TB/s; 8 of them are
// the logits and the second kernel's start, which cooperative launches do not
// overlap); 13 tokens, 6 of 64 experts each, D 1272, F16: 165 us (4.4 TB/s); 5
// tokens, 2 of 8 experts each, H 4096, D 8192, BF16: 225 us (5.5 TB/s).
//
// A token takes the products of its own experts only, from columns of its own:
// what other experts or tokens hold (infinities, NaN) does not reach it.
//
// For 16-bit weights the hidden values enter the second product as a sum of
// 16-bit numbers, each with columns of its own. BF16 has FP32's range: its values are split as
// they are made, into three numbers of 8 bits, which are all of FP32's 24. F16 ones
// are scaled by the power of two that brings the largest of a choice's values to
// [2^13, 2^14), and are sums of two numbers (22 bits, or 2^-38 of that largest; a
// rounding that F16 outputs, of 11 bits, do not show). For 8-bit weights they are
// codes of the largest value / 127. The largest is found with atomic maxima, which
// do not depend on their order; it is known at the grid barrier, after which every
// CTA converts its share, and all meet once more.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "gemm_umma.cuh"
#include "grouped.h"
#include "kebab/layer.h"
#include "quant_i8.cuh"

namespace kb {
namespace {

constexpr int MAX_TOKENS = KEBAB_FEW_TOKENS, MAX_K = 32;
// Warps: copies of weights, MMA issuer, copies of columns, copies of weights,
// four for the epilogue.
constexpr int THREADS = 256, EPI_WARP = 4;
constexpr int ROWS = 128;                 // weight rows of a pass
constexpr int MAX_SLOTS = 16, MAX_UNITS = 8;
// K-blocks of 16-bit values that the MMA sums before the epilogue adds the sum to
// the others. Each of the MMA's additions (4 a K-block) cuts off bits, always
// towards zero: of 5 tokens, H 4096 and D 8192 in one run 0.75 % of the BF16
// outputs were rounded otherwise than the exact ones, in runs of 16 0.16 %, of 8
// 0.08 %, and in FP32 throughout 0.04 %. (172.9, 174.1 and 175.3 us; with two sets
// of accumulators, so that the MMA waits for the end of the pass before, 176.3.)
constexpr int CHUNK = 8, SETS = 4;        // sets of accumulators, in turn
constexpr int TAIL = 128 * 128;           // what an MMA may read past the ring: the tables lie there
constexpr int RING = 200 * 1024;
constexpr int SLOT = 40 * 1024;           // bytes of a slot, about
constexpr int BLOCK = 32;                 // outputs that are added up together
constexpr int COUNTING = 2048;            // comparisons of keys a choice, at most, to choose by counting

struct LayerArgs {
  const void* x;
  int64_t ldx;
  const void* w_in;
  const void* w_out;
  const float* in_scale;
  const float* out_scale;
  void* y;
  int64_t ldy;
  int T, E, k, H, D;
  int renormalize;
  int tma_w, tma_x;  // whether TMA can address the weights, x
  int vec_x;         // whether rows of x start on 16-byte boundaries
  const float* router;
  // The workspace.
  float* logits;      // [T][E]
  float* hidden;      // [T k][D] by expert and token, not BF16
  uint8_t* operand;   // [parts][T k][d_bytes]: the numbers that add up to the values; or their codes
  int d_bytes;
  uint32_t* top;      // [T k]: bits of the largest |hidden|, not BF16
  float* out;         // [T k][out_pitch]: weighted outputs of the choices
  int out_pitch;
  uint32_t* done;     // [ceil(H / BLOCK)]: rows of the block that are in `out`
  float* x_scale;     // [T], 8-bit
  int8_t* x_codes;    // [T][x_pitch], 8-bit
  int x_pitch;
  uint32_t* arrived;  // [2]: CTAs at the grid barriers
  int pdl;
  WaitCtx ctx;
};

// Boxes of 8, 16, .. 64 weight rows: a copy costs about 100 cycles of a warp
// whatever its height, and a pass has any height.
struct RowBoxes {
  CUtensorMap box[8];
};

// ------------------------------------------------------------------- logits

template <typename T>
__global__ void __launch_bounds__(256) layer_logits_kernel(const LayerArgs g) {
  __shared__ float part[8][MAX_TOKENS];
  __shared__ uint32_t tops[8];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(g.x);
  if (blockIdx.x >= g.E) {
    // Codes of a token, nearest to 127 x / amax, ties to even. Of 16-bit values
    // the product is exact and the quotient distinguishes ties from others. (Both
    // by 2^-8 for rows that the product by 127 would bring beyond FP32.)
    const int t = blockIdx.x - g.E;
    x += t * g.ldx;
    uint32_t top = 0;
    for (int h = threadIdx.x; h < g.H; h += 256) top = max(top, abs_bits(to_float(x[h])));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, tops[w]);
    const RowScale s = row_scale(top);
    const float down = __uint_as_float(top) > 0x1p100f ? 0x1p-8f : 1.f, amax = __uint_as_float(top) * down;
    int8_t* q = g.x_codes + (int64_t)t * g.x_pitch;
    for (int h = threadIdx.x; h < g.x_pitch; h += 256)
      q[h] = h < g.H && s.inv != 0.f ? (int8_t)__float2int_rn(to_float(x[h]) * down * 127.f / amax) : 0;
    if (threadIdx.x == 0) g.x_scale[t] = s.scale;
    return;
  }
  const int e = blockIdx.x;
  if (e == 0) {
    for (int i = threadIdx.x; i < g.T * g.k; i += 256) g.top[i] = 0;
    for (int i = threadIdx.x; i < (g.H + BLOCK - 1) / BLOCK; i += 256) g.done[i] = 0;
    if (threadIdx.x < 2) g.arrived[threadIdx.x] = 0;
  }
  const float* r = g.router + (int64_t)e * g.H;
  float sum[MAX_TOKENS];
#pragma unroll
  for (int t = 0; t < MAX_TOKENS; ++t) sum[t] = 0.f;
  // Eight values a step on any boundary, so that the order of the sum is the same.
  const bool vec_r = (reinterpret_cast<uintptr_t>(r) & 15u) == 0;
  for (int h = threadIdx.x * 8; h < g.H; h += 256 * 8) {
    const bool whole = h + 8 <= g.H;
    float w[8], v[8];
    if (whole && vec_r) {
      load_row<8>(r + h, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = h + i < g.H ? r[h + i] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < MAX_TOKENS; ++t) {
      if (t >= g.T) break;
      const T* row = x + t * g.ldx;
      if (whole && g.vec_x) {
        load_row<8>(row + h, v);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = h + i < g.H ? to_float(row[h + i]) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[t] += v[i] * w[i];
    }
  }
#pragma unroll
  for (int t = 0; t < MAX_TOKENS; ++t) {
    if (t >= g.T) break;
#pragma unroll
    for (int d = 16; d; d >>= 1) sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], d);
    if (lane == 0) part[warp][t] = sum[t];
  }
  __syncthreads();
  if (threadIdx.x < g.T) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += part[w][threadIdx.x];
    g.logits[threadIdx.x * g.E + e] = v;
  }
}

// -------------------------------------------------------------------- layer

// How many operands a hidden value makes.
template <typename TX, bool I8>
constexpr int parts_of() {
  return I8 ? 1 : std::is_same<TX, __nv_bfloat16>::value ? 3 : 2;
}
// Whether hidden values are stored as numbers of the weights' type: BF16 has
// FP32's range, F16 needs a scale that is known only when all of them are.
template <typename TX, bool I8>
constexpr bool is_split() {
  return !I8 && std::is_same<TX, __nv_bfloat16>::value;
}

// The top-k choices of the tokens, as kebab_route.
__device__ __forceinline__ uint32_t order_key(float x) {
  x += 0.f;  // -0 becomes +0: they are equal
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// By one warp, choice after choice; `keys`: the token's E words in shared memory.
__device__ __forceinline__ void choose(const LayerArgs& g, int* experts, uint32_t* keys) {
  const int lane = threadIdx.x & 31;
  // The lane's largest key (ties: the lower expert).
  uint32_t top = 0;
  int e_top = 0;
  auto scan = [&] {
    top = 0;
#pragma unroll 1
    for (int e = lane; e < g.E; e += 32) {
      const uint32_t key = keys[e];
      if (key > top) top = key, e_top = e;
    }
  };
  scan();
#pragma unroll 1
  for (int j = 0; j < g.k; ++j) {
    const uint32_t all = __reduce_max_sync(0xffffffffu, top);
    const int e = (int)__reduce_min_sync(0xffffffffu, top == all ? (unsigned)e_top : 0xffffffffu);
    if (lane == 0) experts[j] = e;
    if (top == all && e_top == e) {  // the lane that had it
      keys[e] = 0;
      scan();
    }
    __syncwarp();
  }
}

// All tokens' choices at once by the whole block: an expert's place is how many
// stand before it (larger keys, or as large ones of lower experts). `parts`
// neighbouring lanes share an expert's comparisons.
__device__ __forceinline__ void choose_by_counting(const LayerArgs& g, int* experts, const uint32_t* keys) {
  const int items = g.T * g.E;
  int parts = 1;
  while (parts < 32 && items * parts * 2 <= THREADS) parts *= 2;
  const int part = threadIdx.x % parts;
#pragma unroll 1
  for (int i0 = 0; i0 < items; i0 += THREADS / parts) {
    const int i = min(i0 + (int)threadIdx.x / parts, items - 1);
    const int t = i / g.E, e = i - t * g.E;
    const uint32_t* row = keys + t * g.E;
    const uint32_t key = row[e];
    int before = 0;
#pragma unroll 4
    for (int o = part; o < g.E; o += parts) {
      const uint32_t other = row[o];
      before += o < e ? other >= key : other > key;
    }
    for (int d = 1; d < parts; d *= 2) before += __shfl_xor_sync(0xffffffffu, before, d);
    if (before < g.k) experts[t * g.k + before] = e;
  }
}

// 2^n by which a choice's values are multiplied, for the bits of the largest
// (0 or not finite: 1), and its inverse.
__device__ __forceinline__ float power_for(uint32_t top, float& inverse) {
  const int e = (int)(top >> 23) - 127;
  const int n = top == 0 || e == 128 ? 0 : max(min(13 - e, 126), -126);
  inverse = __uint_as_float((uint32_t)(127 - n) << 23);
  return __uint_as_float((uint32_t)(127 + n) << 23);
}

// Shared memory past the ring: barriers, and tables of the choices.
struct LayerSmem {
  static constexpr int OFF_BAR = RING;
  static constexpr int OFF_TABLES = OFF_BAR + (2 * MAX_SLOTS + 2 * SETS) * 8 + 32;
  // weights by place, weights, scales (float), places, chosen experts (int), [T k]; who chose an expert,
  // places before it (uint16, [T k] and one); the same of all (int [E])
  static __host__ __device__ constexpr int tables(int n, int E) { return OFF_TABLES + n * 20 + (n + 1) * 4 + E * 4; }
  // The first product's rows, whose threads are the gate rows' or the up rows'.
  static constexpr int EXCHANGE = ROWS * (MAX_TOKENS + 1) * 4;
  static constexpr int bytes(int T, int k, int E) {
    const int n = T * k;
    const int end = tables(n, E) + EXCHANGE;
    return (end > RING + TAIL ? end : RING + TAIL) + 1024;  // and the alignment
  }
};
static_assert(LayerSmem::bytes(MAX_TOKENS, MAX_K, kMaxExperts) <= 232448, "shared memory budget exceeded");

// The passes of a CTA: its share [at, end) of active x per rows, cut at the
// experts' ends and then in equal parts of at most `most`. Where the CTAs divide
// among the experts with at most an eighth of them left over, no share crosses
// from one expert to the next, which costs a pass more: 2 experts of 4096 x 2048
// 49 us, 43 without such shares, 8 98 and 94; from an eighth on what is left over
// costs as much (26 experts, 0.12 of the CTAs: 248 and 249 us).
// Made by whole warps; the shuffles tell the compiler that a warp's lanes have
// the same values.
struct Passes {
  int at, end, per, most;
  int a, first, rows;  // the expert (by its place among the chosen), the first row, rows
  int left;            // rows of the segment after this pass
  __device__ __forceinline__ Passes(int active, int per_expert, int most) : per(per_expert), most(most), rows(0), left(0) {
    const int ctas = gridDim.x, cta = blockIdx.x, each = ctas / active;
    if (each * active * 8 >= ctas * 7) {
      const int before = cta / each * per, i = cta % each, share = per / each, more = per % each;
      at = cta < each * active ? before + share * i + min(i, more) : 0;
      end = cta < each * active ? at + share + (i < more) : 0;
    } else {
      const int total = active * per, share = total / ctas, more = total % ctas;
      at = share * cta + min(cta, more);
      end = at + share + (cta < more);
    }
  }
  __device__ __forceinline__ bool next() {
    if (left > 0) {
      first += rows;
    } else {
      if (at >= end) return false;
      a = at / per;
      first = at - a * per;
      left = min(per - first, end - at);
      at += left;
    }
    const int passes = (left + most - 1) / most;
    rows = (left + passes - 1) / passes;
    rows = min(left, (rows + 7) / 8 * 8);  // whole boxes but for the last
    left -= rows;
    a = __shfl_sync(0xffffffffu, a, 0);
    first = __shfl_sync(0xffffffffu, first, 0);
    rows = __shfl_sync(0xffffffffu, rows, 0);
    return true;
  }
};

// One of the two products: rows of the first come in pairs, a gate row and an up
// row; its columns are the tokens, those of the second the hidden values of the
// expert's tokens, in `PARTS` operands.
template <bool UP, int PARTS>
struct Product {
  static constexpr bool kUp = UP;
  static constexpr int MATRICES = UP ? 2 : 1, MOST = ROWS / MATRICES;
  static constexpr int OPERANDS = UP ? 1 : PARTS;
  // Columns of the MMA, a multiple of 16, of operands of `box` each.
  static __device__ __forceinline__ int columns(int box) { return (OPERANDS * box + 15) / 16 * 16; }
};

// How a pass lies in the ring: units of `bytes` (the matrices' rows, r8 each, then
// the columns), `units` K-blocks to a slot.
struct Layout {
  int r8, bytes, units;
  template <typename P>
  __device__ __forceinline__ Layout(P, int rows, int box, int slot) {
    r8 = (rows + 7) / 8 * 8;
    bytes = (P::MATRICES * r8 + P::columns(box)) * 128;
    units = min(MAX_UNITS, slot / bytes);
  }
};

template <typename TX, bool I8>
__global__ void __launch_bounds__(THREADS, 1)
    layer_kernel(const __grid_constant__ RowBoxes tmIn, const __grid_constant__ RowBoxes tmOut,
                 const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmH, const LayerArgs g) {
  constexpr int ES = I8 ? 1 : 2;              // bytes of a weight
  constexpr int EPB = 128 / ES;               // values of a K-block
  constexpr int PARTS = parts_of<TX, I8>();
  constexpr int SET_COLS = PARTS == 3 ? 64 : 32, TMEM_COLS = SETS * SET_COLS;
  constexpr bool SPLIT = is_split<TX, I8>();  // made in the first product's epilogue
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + LayerSmem::OFF_BAR);
  uint64_t* empty = full + MAX_SLOTS;
  uint64_t* acc_full = empty + MAX_SLOTS;
  uint64_t* acc_empty = acc_full + SETS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + SETS);
  int* s_count = reinterpret_cast<int*>(tmem_slot + 1);  // chosen experts
  int* s_last = s_count + 1;                             // of the blocks of a pass, which it completed (bits)
  const int choices = g.T * g.k;
  float* s_factor = reinterpret_cast<float*>(smem + LayerSmem::OFF_TABLES);  // by place: the choice's weight
  float* s_weight = s_factor + choices;                                      // [T][k]
  float* s_scale = s_weight + choices;                                       // by place
  int* s_place = reinterpret_cast<int*>(s_scale + choices);                  // [T][k], at first the expert
  int* s_active = s_place + choices;                                         // chosen experts, ascending
  uint16_t* s_who = reinterpret_cast<uint16_t*>(s_active + choices);         // of each, the tokens that chose it (bits)
  uint16_t* s_base = s_who + choices;                                        // of each, the place of its first choice
  uint32_t* s_chose = reinterpret_cast<uint32_t*>(s_base + choices + 2);     // [E]: the tokens that chose it (bits)
  float* s_rows = reinterpret_cast<float*>(smem + LayerSmem::tables(choices, g.E));  // [ROWS][MAX_TOKENS + 1]
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const WaitCtx& ctx = g.ctx;

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_SLOTS; ++s) {
      mbar_init(&full[s], 3);  // the copying warps
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SETS; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 4);
    }
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc<1>(tmem_slot, TMEM_COLS);
    tmem_relinquish<1>();
  }
  // The tensor maps, whichever boxes the passes will need.
  if (warp == 2 && lane < 18) {
    const CUtensorMap* tm = lane < 8 ? &tmIn.box[lane] : lane < 16 ? &tmOut.box[lane - 8] : lane == 16 ? &tmX : &tmH;
    if (lane == 17 || (lane == 16 ? g.tma_x : g.tma_w)) tma_prefetch_desc(tm);
  }
  for (int i = threadIdx.x; i < g.E; i += THREADS) s_chose[i] = 0;
  if (g.pdl) pdl_wait();
  __syncthreads();
  // Keys of the logits, in the ring. Choice after choice costs each one's latency,
  // counting the comparisons of all pairs of experts (a whole call of 1 token, 64
  // experts: of 16 choices 18.2 us against 16.2, of 8 16.0 against 15.2, of 2 15.1
  // against 15.4; 256 experts, 8 choices: 19.3 against 21.2; 16 tokens, 128
  // experts, 8 choices: 33.5 against 50.0).
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);
  for (int i = threadIdx.x; i < g.T * g.E; i += THREADS) keys[i] = order_key(__ldcg(g.logits + i));
  __syncthreads();
  const bool counting = g.k >= 4 && g.T * g.E * g.E <= COUNTING * g.k;
  if (counting) {
    choose_by_counting(g, s_place, keys);
    __syncthreads();
  }
  for (int t = warp; t < g.T; t += THREADS / 32) {
    if (!counting) {
      // The softmax's sum needs the keys that `choose` takes away.
      choose(g, s_place + t * g.k, keys + t * g.E);
      __syncwarp();
    }
    const bool mine = lane < g.k;
    const int e = mine ? s_place[t * g.k + lane] : 0;
    const float* logits = g.logits + t * g.E;
    const float v = mine ? __ldcg(logits + e) + 0.f : 0.f;
    const float highest = __shfl_sync(0xffffffffu, v, 0);
    // All logits -inf: nothing to weigh.
    const float p = mine && highest != -INFINITY ? expf(v - highest) : 0.f;
    float sum = p;
    if (!g.renormalize) {
      sum = 0.f;
#pragma unroll 1
      for (int i = lane; i < g.E; i += 32) sum += expf(__ldcg(logits + i) - highest);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (mine) {
      s_weight[t * g.k + lane] = p / (highest == -INFINITY ? 1.f : sum);
      atomicOr(&s_chose[e], 1u << t);
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0, before = 0;
    for (int e0 = 0; e0 < g.E; e0 += 32) {
      const uint32_t who = e0 + lane < g.E ? s_chose[e0 + lane] : 0u;
      const uint32_t mask = __ballot_sync(0xffffffffu, who != 0);
      if (mask == 0) continue;
      int sum = __popc(who);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (who) {
        const int a = n + __popc(mask & ((1u << lane) - 1u));
        s_active[a] = e0 + lane;
        s_who[a] = (uint16_t)who;
        s_base[a] = (uint16_t)(before + sum - __popc(who));
        s_chose[e0 + lane] = (who & 0xffffu) | (uint32_t)(before + sum - __popc(who)) << 16;
      }
      n += __popc(mask);
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) *s_count = n;
    __syncwarp();
    for (int i = lane; i < choices; i += 32) {
      const uint32_t chose = s_chose[s_place[i]];  // and the place of the expert's first choice
      const int place = (int)(chose >> 16) + __popc(chose & 0xffffu & ((1u << (i / g.k)) - 1u));
      s_place[i] = place;
      s_factor[place] = s_weight[i];
    }
  }
  fence_proxy_async_smem();  // the keys' reads and writes before the copies into the ring
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int active = __shfl_sync(0xffffffffu, *s_count, 0);

  const int box = g.T <= 8 ? 8 : 16;  // columns of an operand
  // The ring's slots, by the longest pass that there can be.
  using Up = Product<true, PARTS>;
  using Down = Product<false, PARTS>;
  auto longest = [&](auto product, int per) {
    using P = decltype(product);
    const int each = gridDim.x / active;  // CTAs of an expert (Passes)
    const int rows = each ? (per + each - 1) / each : (active * per + (int)gridDim.x - 1) / (int)gridDim.x;
    const int share = min(P::MOST, rows);
    return (P::MATRICES * ((share + 7) / 8 * 8) + P::columns(box)) * 128;
  };
  const int unit_bytes = max(longest(Up(), g.D), longest(Down(), g.H));
  const int slot_bytes = unit_bytes * max(1, min(MAX_UNITS, SLOT / unit_bytes));
  const int slots = min(MAX_SLOTS, RING / slot_bytes);
  // The first pass: here, once for all warps. (The second product's are worked out
  // by each warp while it has time.)
  Passes first_up(active, g.D, Up::MOST);
  const bool any_up = first_up.next();
  const int up_blocks = (g.H + EPB - 1) / EPB, down_blocks = (g.D + EPB - 1) / EPB;
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  bool ok = true;
  int slot = 0;
  uint32_t phase = 0;
  auto advance = [&] {
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  };
  // A wait for all CTAs, by one thread; what they wrote before they arrived is
  // visible after it.
  auto wait_for_all = [&](const uint32_t* count) {
    const uint64_t t0 = globaltimer();
    for (uint32_t it = 1;; ++it) {
      uint32_t n;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(count) : "memory");
      if (n >= gridDim.x) return true;
      if ((it & 63u) == 0u) {
        if (aborted(ctx.status)) return false;
        if (globaltimer() - t0 > ctx.timeout_ns) {
          record_error(ctx.status, DEV_TIMEOUT, SITE_GRID);
          return false;
        }
      }
    }
  };
  // 128 bytes of rows on any boundary, value by value, as TMA would place them:
  // `rows` rows of `cols` values at a pitch (in values), from value k0 on; zeros
  // past the ends. By a whole warp.
  auto copy_rows = [&](uint8_t* dst, const void* src, int64_t pitch, int rows, int r8, int k0, int cols) {
    for (int i = lane; i < r8 * EPB; i += 32) {
      const int r = i / EPB, c = i % EPB, b = c * ES;
      const bool is = r < rows && k0 + c < cols;
      uint8_t* to = dst + r * 128 + ((b >> 4 ^ (r & 7)) << 4) + (b & 15);
      if constexpr (I8) *to = is ? static_cast<const uint8_t*>(src)[r * pitch + k0 + c] : 0;
      else *reinterpret_cast<uint16_t*>(to) = is ? static_cast<const uint16_t*>(src)[r * pitch + k0 + c] : 0;
    }
  };

  if (warp == 0 || warp == 3) {
    // -------------------------------------------------- copies of weights
    // Of the first product one warp copies the gate rows, the other the up rows;
    // of the second every other K-block. The loops run with all lanes, so that
    // addresses stay in uniform registers.
    const int which = warp == 0 ? 0 : 1;
    // Weights are read once: they leave L2 first, and the rest (hidden values, the
    // kernel's own instructions) stays (13 tokens 177 -> 166 us, 1 token 31.6 -> 30.3).
    const uint64_t policy = l2_policy_evict_first();
    auto copy = [&](auto product, Passes p, bool more, const RowBoxes& tm, const void* w, int per, int cols, int blocks) {
      using P = decltype(product);
      for (; ok && more; more = p.next()) {
        const Layout l(product, p.rows, box, slot_bytes);
        const int e = __shfl_sync(0xffffffffu, s_active[p.a], 0);
        const int row = P::kUp ? which * per + p.first : p.first;
        const int low = min(l.r8, 64), high = l.r8 - low;
        for (int kb = 0; kb < blocks; kb += l.units) {
          ok = all_ok(mbar_wait(&empty[slot], phase ^ 1u, ctx, SITE_EMPTY));
          if (!ok) break;
          const int n = min(l.units, blocks - kb);
          const int q0 = P::kUp ? 0 : which, step = P::kUp ? 1 : 2;
          const int mine = P::kUp ? n : (n - which + 1) / 2;
          uint8_t* dst = smem + slot * slot_bytes + (P::kUp ? which * l.r8 * 128 : which * l.bytes);
          if (g.tma_w) {
            if (elect_one()) mbar_arrive_expect_tx(&full[slot], mine * l.r8 * 128);
            __syncwarp();
            for (int q = q0; q < n; q += step, dst += step * l.bytes) {
              const int k0 = (kb + q) * EPB;
              if (elect_one()) {
                tma_load_3d_hint(dst, &tm.box[low / 8 - 1], &full[slot], k0, row, e, policy);
                if (high) tma_load_3d_hint(dst + 64 * 128, &tm.box[high / 8 - 1], &full[slot], k0, row + 64, e, policy);
              }
              __syncwarp();
            }
          } else {
            const int64_t from = ((int64_t)e * P::MATRICES * per + row) * cols * ES;
            for (int q = q0; q < n; q += step, dst += step * l.bytes)
              copy_rows(dst, static_cast<const uint8_t*>(w) + from, cols, p.rows, l.r8, (kb + q) * EPB, cols);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            __syncwarp();
          }
          advance();
        }
      }
    };
    copy(Up(), first_up, any_up, tmIn, g.w_in, g.D, g.H, up_blocks);
    Passes first_down(active, g.H, Down::MOST);
    const bool any_down = first_down.next();
    copy(Down(), first_down, any_down, tmOut, g.w_out, g.H, g.D, down_blocks);
  } else if (warp == 2) {
    // -------------------------------------------------- copies of columns
    bool met = false;  // past the grid barrier
    auto copy = [&](auto product, Passes p, bool more, int blocks) {
      using P = decltype(product);
      for (; ok && more; more = p.next()) {
        const Layout l(product, p.rows, box, slot_bytes);
        const int base = __shfl_sync(0xffffffffu, (int)s_base[p.a], 0);
        for (int kb = 0; kb < blocks; kb += l.units) {
          ok = all_ok(mbar_wait(&empty[slot], phase ^ 1u, ctx, SITE_EMPTY));
          if (!P::kUp && ok && !met) {
            // The hidden values of all CTAs, which wrote them as other memory than
            // TMA's. (Waited for here, with all of the way to the first copy done:
            // between the products it cost 2.8 us more, for instructions that are
            // fetched from a memory that is busy with the weights.)
            if (lane == 0) ok = wait_for_all(g.arrived + (SPLIT ? 0 : 1));
            ok = all_ok(ok);
            fence_proxy_async_global();
            __syncwarp();
            met = true;
          }
          if (!ok) break;
          const int n = min(l.units, blocks - kb);
          uint8_t* dst = smem + slot * slot_bytes + P::MATRICES * l.r8 * 128;
          if (P::kUp && !g.tma_x) {
            for (int q = 0; q < n; ++q, dst += l.bytes)
              copy_rows(dst, g.x, g.ldx, g.T, box, (kb + q) * EPB, g.H);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            __syncwarp();
          } else {
            if (elect_one()) mbar_arrive_expect_tx(&full[slot], n * P::OPERANDS * box * 128);
            __syncwarp();
            for (int q = 0; q < n; ++q, dst += l.bytes) {
              const int k0 = (kb + q) * EPB;
              if (elect_one()) {
                if constexpr (P::kUp) tma_load_2d(dst, &tmX, &full[slot], k0, 0);
                else tma_load_3d(dst, &tmH, &full[slot], k0, base, 0);
              }
              __syncwarp();
            }
          }
          advance();
        }
      }
    };
    copy(Up(), first_up, any_up, up_blocks);
    Passes first_down(active, g.H, Down::MOST);
    const bool any_down = first_down.next();
    copy(Down(), first_down, any_down, down_blocks);
  } else if (warp == 1) {
    // --------------------------------------------------------- MMA issuer
    const uint32_t ring = smem_u32(smem), d0 = __shfl_sync(0xffffffffu, tmem, 0);
    uint32_t run = 0;  // of CHUNK K-blocks
    auto multiply = [&](auto product, Passes p, bool more, int blocks) {
      using P = decltype(product);
      const uint32_t idesc = (I8 ? umma_idesc_i8(128, 0) : umma_idesc_f16(128, 0, ElemTraits<TX>::kBf16)) |
                             (uint32_t)(P::columns(box) >> 3) << 17;
      for (; ok && more; more = p.next()) {
        const Layout l(product, p.rows, box, slot_bytes);
        uint32_t set = 0;
        for (int kb = 0; ok && kb < blocks; kb += l.units) {
          ok = all_ok(mbar_wait(&full[slot], phase, ctx, SITE_FULL));
          if (!ok) break;
          tc_fence_after();
          const int n = min(l.units, blocks - kb);
          const uint32_t base = ring + slot * slot_bytes;
          for (int q = 0; q < n; ++q) {
            const uint64_t a = umma_desc_sw128(base + q * l.bytes);
            const uint64_t b = umma_desc_sw128(base + q * l.bytes + P::MATRICES * l.r8 * 128);
            const bool begins = I8 ? kb + q == 0 : (kb + q) % CHUNK == 0;
            const uint32_t first = begins ? 0u : 1u;
            if (begins) {
              if (kb + q > 0 && elect_one()) umma_commit_cg1(&acc_full[set]);
              __syncwarp();
              set = run % SETS;
              ok = all_ok(mbar_wait(&acc_empty[set], (run / SETS & 1u) ^ 1u, ctx, SITE_TMEM_EMPTY));
              if (!ok) break;
              tc_fence_after();
              ++run;
            }
            const uint32_t d_tmem = d0 + set * SET_COLS;
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if constexpr (I8) umma_i8<1>(d_tmem, a + k * 2, b + k * 2, idesc, k == 0 ? first : 1u);
                else umma_f16_cg1(d_tmem, a + k * 2, b + k * 2, idesc, k == 0 ? first : 1u);
              }
            }
            __syncwarp();
          }
          if (elect_one()) {
            umma_commit_cg1(&empty[slot]);
            if (kb + l.units >= blocks) umma_commit_cg1(&acc_full[set]);
          }
          __syncwarp();
          advance();
        }
      }
    };
    multiply(Up(), first_up, any_up, up_blocks);
    Passes first_down(active, g.H, Down::MOST);
    const bool any_down = first_down.next();
    multiply(Down(), first_down, any_down, down_blocks);
  } else if (warp >= EPI_WARP) {
    // ----------------------------------------------------------- epilogue
    const int et = threadIdx.x - 32 * EPI_WARP;  // the thread's row of a pass
    const uint32_t quarter = tmem + ((uint32_t)(warp % 4 * 32) << 16);
    auto meet = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    auto number = [](uint32_t v) {
      if constexpr (I8) return (float)(int)v;
      else return __uint_as_float(v);
    };
    // Arrival at a grid barrier, after all that the CTA's threads wrote.
    auto arrive = [&](uint32_t* count) {
      fence_proxy_async_global();
      meet();
      if (et == 0) asm volatile("fence.acq_rel.gpu;\n\tred.relaxed.gpu.global.add.u32 [%0], 1;" ::"l"(count) : "memory");
    };
    uint32_t run = 0;
    // The sums of a pass for the first `n` columns, its runs of K-blocks one after the other.
    float sum[MAX_TOKENS];
    auto take = [&](auto product, int blocks, int n) {
      constexpr int OPERANDS = decltype(product)::OPERANDS;
      const int runs = I8 ? 1 : (blocks + CHUNK - 1) / CHUNK;
#pragma unroll 1
      for (int i = 0; i < runs; ++i, ++run) {
        const uint32_t set = run % SETS;
        uint32_t v[32], v3[16];
        if (ok) ok = all_ok(mbar_wait(&acc_full[set], run / SETS & 1u, ctx, SITE_TMEM_FULL));
        tc_fence_after();
        tmem_ld_32x32b_x32(quarter + set * SET_COLS, v);
        if (OPERANDS == 3 && box == 16) tmem_ld_32x32b_x16(quarter + set * SET_COLS + 32, v3);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&acc_empty[set]);
#pragma unroll
        for (int c = 0; c < MAX_TOKENS; ++c) {
          if (c >= n) break;
          float o = number(v[c]);
          if constexpr (OPERANDS == 2) o += number(box == 16 ? v[16 + c] : v[8 + c % 8]);
          if constexpr (OPERANDS == 3)
            o += box == 16 ? number(v3[c]) + number(v[16 + c]) : number(v[16 + c % 8]) + number(v[8 + c % 8]);
          sum[c] = i == 0 ? o : sum[c] + o;
        }
      }
    };

    // Hidden values: silu(gate) * up.
    {
      Passes p = first_up;
      for (bool more = any_up; more; more = p.next()) {
        const int i = p.first + et, r8 = (p.rows + 7) / 8 * 8;
        const bool mine = et < p.rows;
        float gate_scale = 1.f, up_scale = 1.f;
        if constexpr (I8) {
          const float* scale = g.in_scale + (int64_t)s_active[p.a] * 2 * g.D + i;
          gate_scale = mine ? scale[0] : 0.f;
          up_scale = mine ? scale[g.D] : 0.f;
        }
        const uint32_t who = s_who[p.a];
        int place = s_base[p.a];
        take(Up(), up_blocks, g.T);
        // The up rows are the threads from r8 on. Through shared memory, and then
        // token by token in a loop: unrolled, one token's values took 4 us, for
        // the instructions that are fetched on the way.
        meet();  // what was there has been read
#pragma unroll
        for (int t = 0; t < MAX_TOKENS; ++t)
          if (who >> t & 1u) s_rows[et * (MAX_TOKENS + 1) + t] = sum[t];
        meet();
        if (warp - EPI_WARP > (p.rows - 1) / 32) continue;
#pragma unroll 1
        for (uint32_t rest = who; rest; rest &= rest - 1) {
          const int t = __ffs(rest) - 1;
          float gate = mine ? s_rows[et * (MAX_TOKENS + 1) + t] : 0.f;
          float value = mine ? s_rows[(et + r8) * (MAX_TOKENS + 1) + t] : 0.f;
          if constexpr (I8) {
            const float s = g.x_scale[t];
            gate *= s * gate_scale;
            value *= s * up_scale;
          }
          const float h = gate / (1.f + expf(-gate)) * value;
          if constexpr (SPLIT) {
            if (mine && ok) {
              // Cut after eight bits, not rounded: what is left is exact, and the largest
              // values stay finite. Of an infinity or a NaN nothing is left.
              uint8_t* to = g.operand + (int64_t)place * g.d_bytes + (int64_t)i * 2;
              const bool finite = abs_bits(h) < 0x7f800000u;
              float rest = h;
#pragma unroll
              for (int part = 0; part < PARTS; ++part, to += (int64_t)choices * g.d_bytes) {
                const float cut = finite ? __uint_as_float(__float_as_uint(rest) & 0xffff0000u) : rest;
                *reinterpret_cast<TX*>(to) = from_float<TX>(cut);
                rest = finite ? rest - cut : 0.f;
              }
            }
          } else {
            if (mine && ok) g.hidden[(int64_t)place * g.D + i] = h;
            const uint32_t top = __reduce_max_sync(0xffffffffu, mine ? abs_bits(h) : 0u);
            if (lane == 0) atomicMax(g.top + place, top);
          }
          ++place;
        }
      }
    }
    arrive(g.arrived);
    if constexpr (!SPLIT) {
      // The largest values are known: this CTA's share in the operands' form.
      bool here = true;
      if (et == 0) here = wait_for_all(g.arrived);
      ok = all_ok(here && ok);  // of the whole warp, which goes on together
      __threadfence();
      meet();
      for (int i = et; i < choices; i += 128) {
        float inverse;
        const uint32_t top = __ldcg(g.top + i);
        if constexpr (I8) {
          const RowScale code = row_scale(top);
          s_scale[i] = code.inv;
          inverse = code.scale;
        } else {
          s_scale[i] = power_for(top, inverse);
        }
        s_factor[i] *= inverse;
      }
      meet();
      Passes p(active, g.D, 1 << 30);  // the expert's part of the share at once
      while (p.next()) {
        const int base = s_base[p.a], values = __popc((uint32_t)s_who[p.a]) * p.rows;
        // Eight loads in flight a thread: one by one, they took 10 us of 13 tokens
        // of 6 choices, 1272 values each.
        for (int i0 = et; i0 < values; i0 += 8 * 128) {
          float h[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * 128, c = i / p.rows;
            if (i < values) h[u] = __ldcg(g.hidden + (int64_t)(base + c) * g.D + p.first + i - c * p.rows);
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const int i = i0 + u * 128, c = i / p.rows, at = p.first + i - c * p.rows;
            if (i >= values) break;
            const float scale = s_scale[base + c];
            uint8_t* to = g.operand + (int64_t)(base + c) * g.d_bytes;
            if constexpr (I8) {
              to[at] = scale == 0.f ? 0 : (uint8_t)(code_bits(h[u], scale) & 0xffu);
            } else {
              const float x = h[u] * scale;
              const TX hi = from_float<TX>(x);
              reinterpret_cast<TX*>(to)[at] = hi;
              reinterpret_cast<TX*>(to + (int64_t)choices * g.d_bytes)[at] = from_float<TX>(isinf(x) ? 0.f : x - to_float(hi));
            }
          }
        }
      }
      arrive(g.arrived + 1);
    }

    // Outputs of the choices, and sums of the blocks that they complete.
    Passes p(active, g.H, Down::MOST);
    while (p.next()) {
      const int r = p.first + et, n = __popc((uint32_t)s_who[p.a]), base = s_base[p.a];
      const bool mine = et < p.rows;
      float scale = 1.f;
      if constexpr (I8) scale = mine ? g.out_scale[(int64_t)s_active[p.a] * g.H + r] : 0.f;
      take(Down(), down_blocks, n);
#pragma unroll
      for (int c = 0; c < MAX_TOKENS; ++c) {
        if (c >= n) break;
        if (mine) g.out[(int64_t)(base + c) * g.out_pitch + r] = s_factor[base + c] * scale * sum[c];
      }
      __threadfence();
      meet();
      // The pass's rows lie in at most 5 blocks.
      const int b0 = p.first / BLOCK, b1 = (p.first + p.rows - 1) / BLOCK;
      if (et == 0) *s_last = 0;
      meet();
      if (et <= b1 - b0) {
        const int b = b0 + et, begin = b * BLOCK, end = min(begin + BLOCK, g.H);
        const uint32_t rows = min(end, p.first + p.rows) - max(begin, p.first);
        const uint32_t all = (uint32_t)active * (uint32_t)(end - begin);
        if (atomicAdd(g.done + b, rows) + rows == all) atomicOr(s_last, 1 << et);
      }
      __threadfence();
      meet();
      // Eight threads a block and token, four outputs each.
      const int last = *s_last, blocks = __popc((uint32_t)last);
      for (int i = et / 8; i < blocks * g.T; i += 16) {
        const int t = i % g.T;
        uint32_t rest = (uint32_t)last;
        for (int skip = i / g.T; skip; --skip) rest &= rest - 1;
        const int o = (b0 + __ffs(rest) - 1) * BLOCK + et % 8 * 4;
        if (o >= g.H) continue;
        const int* place = s_place + t * g.k;
        float4 all = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
        for (int j0 = 0; j0 < g.k; j0 += 8) {
          float4 u[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j0 + j < g.k) u[j] = __ldcg(reinterpret_cast<const float4*>(g.out + (int64_t)place[j0 + j] * g.out_pitch + o));
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j0 + j < g.k) all.x += u[j].x, all.y += u[j].y, all.z += u[j].z, all.w += u[j].w;
        }
        const float f[4] = {all.x, all.y, all.z, all.w};
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (ok && o + u < g.H) static_cast<TX*>(g.y)[t * g.ldy + o + u] = from_float<TX>(f[u]);
      }
    }
  }
  // A wait ran out: what is in flight has to land before the CTA leaves.
  __syncwarp();
  tc_fence_before();
  if (__syncthreads_or(!ok)) settle();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem, TMEM_COLS);
  }
}

// ---------------------------------------------------------------- host side

constexpr int64_t kMaxWidth = 1 << 20;  // of H and D: the rows of 512 choices are counted in 32 bits

struct Sizes {
  int64_t T, E, k, H, D;
};

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

// Of T tokens: logits, hidden values, operands, their largest, outputs, blocks' counts, scales, barriers, codes.
struct Workspace {
  int64_t logits, hidden, operand, top, out, done, x_scale, arrived, x_codes, end;
  explicit Workspace(const Sizes& s) {
    int64_t at = 0;
    auto take = [&](int64_t n) {
      const int64_t here = at;
      at += up16(n);
      return here;
    };
    const int64_t n = s.T * s.k;
    logits = take(s.T * s.E * 4);
    hidden = take(n * s.D * 4);
    operand = take(3 * n * up16(2 * s.D));
    top = take(n * 4);
    out = take(n * up16(s.H) * 4);
    done = take((s.H + BLOCK - 1) / BLOCK * 4);
    x_scale = take(64);
    arrived = take(8);
    x_codes = take(s.T * up16(s.H));
    end = at;
  }
};
int64_t bytes(const Sizes& s) { return Workspace(s).end; }

int check(const char* what, int dtype, const void* x, int64_t ldx, const void* router, const void* w_in,
          const void* w_out, const void* y, int64_t ldy, const Sizes& s, void* ws, int64_t ws_bytes) {
  const std::string w = what;
  if (dtype != KEBAB_F16 && dtype != KEBAB_BF16) return fail(KEBAB_ENOTSUP, w + ": only F16 and BF16 are implemented");
  if (s.T < 0 || s.T > KEBAB_FEW_TOKENS)
    return fail(KEBAB_EINVAL, w + ": " + std::to_string(s.T) + " tokens are not in 0.." + std::to_string(KEBAB_FEW_TOKENS));
  if (s.E < 1 || s.E > kMaxExperts)
    return fail(KEBAB_EINVAL, w + ": number of experts " + std::to_string(s.E) + " is not in 1.." + std::to_string(kMaxExperts));
  if (s.k < 1 || s.k > MAX_K || s.k > s.E)
    return fail(KEBAB_EINVAL, w + ": k = " + std::to_string(s.k) + " is not in 1..min(E, 32)");
  if (s.H <= 0 || s.D <= 0 || s.H > kMaxWidth || s.D > kMaxWidth)
    return fail(KEBAB_EINVAL, w + ": invalid dimensions H=" + std::to_string(s.H) + " D=" + std::to_string(s.D));
  if (ldx < s.H || ldy < s.H) return fail(KEBAB_EINVAL, w + ": a row pitch is below the row length");
  if (s.T == 0) return KEBAB_OK;
  if (!x || !router || !w_in || !w_out || !y) return fail(KEBAB_EINVAL, w + ": null pointer");
  if (!ws || ws_bytes < bytes(s) || (reinterpret_cast<uintptr_t>(ws) & 15u))
    return fail(KEBAB_EINVAL, w + ": the workspace is null, too small or not 16-byte aligned");
  return KEBAB_OK;
}

// Boxes of a stack of matrices' rows.
int row_boxes(RowBoxes* m, const void* base, int type, int es, int64_t n, int64_t rows, int64_t cols) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)n};
  const uint64_t strides[2] = {(uint64_t)(cols * es), (uint64_t)(rows * cols * es)};
  for (int i = 0; i < 8; ++i) {
    const uint32_t box[3] = {(uint32_t)(128 / es), 8u * (i + 1), 1};
    const int rc = make_tmap(&m->box[i], base, type, 3, dims, strides, box, 128);
    if (rc) return rc;
  }
  return KEBAB_OK;
}

template <typename TX, bool I8>
int launch(int dtype, LayerArgs& g, cudaStream_t stream) {
  constexpr int ES = I8 ? 1 : 2;
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev)) || (rc = wait_ctx(&g.ctx))) return rc;
  g.pdl = pdl_enabled();
  const int type = I8 ? TMAP_U8 : dtype;
  RowBoxes in = {}, out = {};
  CUtensorMap tx = {}, th = {};
  if (g.tma_w && ((rc = row_boxes(&in, g.w_in, type, ES, g.E, 2 * (int64_t)g.D, g.H)) ||
                  (rc = row_boxes(&out, g.w_out, type, ES, g.E, g.H, g.D))))
    return rc;
  const uint32_t columns = g.T <= 8 ? 8 : 16;
  if (g.tma_x) {
    const uint64_t dims[2] = {(uint64_t)(I8 ? g.x_pitch : g.H), (uint64_t)g.T};
    const uint64_t strides[1] = {(uint64_t)(I8 ? g.x_pitch : g.ldx * 2)};
    const uint32_t box[2] = {128 / ES, columns};
    if ((rc = make_tmap(&tx, I8 ? (const void*)g.x_codes : g.x, type, 2, dims, strides, box, 128))) return rc;
  }
  {
    const uint64_t n = (uint64_t)g.T * g.k;
    const uint64_t dims[3] = {(uint64_t)g.D, n, (uint64_t)parts_of<TX, I8>()}, strides[2] = {(uint64_t)g.d_bytes, n * g.d_bytes};
    const uint32_t box[3] = {128 / ES, columns, (uint32_t)parts_of<TX, I8>()};
    if ((rc = make_tmap(&th, g.operand, type, 3, dims, strides, box, 128))) return rc;
  }
  auto kern = layer_kernel<TX, I8>;
  static std::once_flag once[64];
  static cudaError_t err[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   LayerSmem::bytes(MAX_TOKENS, MAX_K, kMaxExperts));
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  PdlLaunch first(dim3((unsigned)(g.E + (I8 ? g.T : 0))), dim3(256), 0, stream);
  cudaError_t e = cudaLaunchKernelEx(&first.cfg, layer_logits_kernel<TX>, (const LayerArgs)g);
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer: logits launch");
  PdlLaunch l(dim3((unsigned)dev->sm_count), dim3(THREADS), LayerSmem::bytes(g.T, g.k, g.E), stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  if (l.cfg.numAttrs) attr[1] = l.attr[0];
  l.cfg.attrs = attr;
  ++l.cfg.numAttrs;
  e = cudaLaunchKernelEx(&l.cfg, kern, in, out, tx, th, (const LayerArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "expert_layer launch");
}

template <bool I8>
int run(int dtype, LayerArgs g, const Sizes& s, void* ws, kebab_stream_t stream) {
  constexpr int ES = I8 ? 1 : 2;
  g.T = (int)s.T, g.E = (int)s.E, g.k = (int)s.k, g.H = (int)s.H, g.D = (int)s.D;
  const Workspace w(s);
  uint8_t* at = static_cast<uint8_t*>(ws);
  g.logits = reinterpret_cast<float*>(at + w.logits);
  g.hidden = reinterpret_cast<float*>(at + w.hidden);
  g.operand = at + w.operand;
  g.d_bytes = (int)up16(s.D * ES);
  g.top = reinterpret_cast<uint32_t*>(at + w.top);
  g.out = reinterpret_cast<float*>(at + w.out);
  g.out_pitch = (int)up16(s.H);
  g.done = reinterpret_cast<uint32_t*>(at + w.done);
  g.x_scale = reinterpret_cast<float*>(at + w.x_scale);
  g.arrived = reinterpret_cast<uint32_t*>(at + w.arrived);
  g.x_codes = reinterpret_cast<int8_t*>(at + w.x_codes);
  g.x_pitch = (int)up16(s.H);
  auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  g.tma_w = on16(g.w_in) && on16(g.w_out) && s.H * ES % 16 == 0 && s.D * ES % 16 == 0;
  g.vec_x = on16(g.x) && g.ldx % 8 == 0;
  g.tma_x = I8 || g.vec_x;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == KEBAB_F16 ? launch<__half, I8>(dtype, g, st) : launch<__nv_bfloat16, I8>(dtype, g, st);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int64_t kebab_expert_layer_workspace(int64_t T, int64_t E, int k, int64_t H, int64_t D) {
  if (T < 0 || T > KEBAB_FEW_TOKENS || E < 1 || E > kMaxExperts || k < 1 || k > MAX_K || H <= 0 || D <= 0 ||
      H > kMaxWidth || D > kMaxWidth)
    return -KEBAB_EINVAL;
  return bytes({T, E, k, H, D});
}

int kebab_expert_layer(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const void* w_in,
                       const void* w_out, void* y, int64_t ldy, int64_t T, int64_t E, int k, int renormalize,
                       int64_t H, int64_t D, void* workspace, int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const Sizes s = {T, E, k, H, D};
    const int rc = check("expert_layer", dtype, x, ldx, router, w_in, w_out, y, ldy, s, workspace, workspace_bytes);
    if (rc || T == 0) return rc;
    LayerArgs g = {};
    g.x = x, g.ldx = ldx, g.router = router, g.w_in = w_in, g.w_out = w_out, g.y = y, g.ldy = ldy;
    g.renormalize = renormalize;
    return run<false>(dtype, g, s, workspace, stream);
  });
}

int kebab_expert_layer_i8(kebab_dtype dtype, const void* x, int64_t ldx, const float* router, const int8_t* w_in,
                          const float* in_scale, const int8_t* w_out, const float* out_scale, void* y, int64_t ldy,
                          int64_t T, int64_t E, int k, int renormalize, int64_t H, int64_t D, void* workspace,
                          int64_t workspace_bytes, kebab_stream_t stream) {
  return guarded([&] {
    const Sizes s = {T, E, k, H, D};
    const int rc = check("expert_layer_i8", dtype, x, ldx, router, w_in, w_out, y, ldy, s, workspace, workspace_bytes);
    if (rc || T == 0) return rc;
    if (H > 131072 || D > 131072)
      return fail(KEBAB_EINVAL, "expert_layer_i8: H or D above 131072 could overflow the 32-bit sums");
    if (!in_scale || !out_scale) return fail(KEBAB_EINVAL, "expert_layer_i8: null pointer");
    LayerArgs g = {};
    g.x = x, g.ldx = ldx, g.router = router, g.w_in = w_in, g.in_scale = in_scale, g.w_out = w_out;
    g.out_scale = out_scale, g.y = y, g.ldy = ldy, g.renormalize = renormalize;
    return run<true>(dtype, g, s, workspace, stream);
  });
}

}  // extern "C"
