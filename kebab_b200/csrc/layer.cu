// A mixture-of-experts feed-forward layer for up to 16 tokens, in two launches.
//
// The first computes the router's logits (a block an expert; for 8-bit experts
// also the codes of the tokens) and clears what the second counts in. The second
// is one CTA an SM, all resident (a cooperative launch): every CTA finds the
// top-k choices by itself, takes an equal share of the hidden values of all
// chosen experts (a gate row and an up row each), meets the others at a grid
// barrier, and takes an equal share of the layer's outputs, over all chosen
// experts. So the sum over a token's experts needs no further exchange, and the
// results do not depend on who comes first.
//
// Bound by the chosen experts' bytes, and by latency for few of them. One warp
// copies the CTA's weights, which are contiguous rows, through a ring of 32 KB
// stages; it does not wait at the grid barrier, so that the second product's
// weights arrive meanwhile. Eight warps multiply on the tensor cores (mma.sync,
// 16 weight rows by 8 tokens: the tokens are so few that this takes a tenth of
// the time that the bytes take, and unlike a tile of 128 rows it lets the CTAs
// share the rows evenly). They split the row's length in steps of 64 bytes:
// lane (g, c) of a warp reads the 16 bytes c of the step from rows g and g + 8,
// which are the operand registers of two MMAs if the tokens' values are read in
// the same order, since a sum over k may take its terms in any.
//
// An expert's rows are multiplied with the tokens that chose it and added onto
// those only: what other experts hold (infinities, NaN) does not reach a token.
//
// For 16-bit weights the hidden values enter the second product as the sum of
// two 16-bit numbers (at least 16 bits of them); F16 ones scaled by the power of
// two that brings the largest of a choice's values to [2^13, 2^14). For 8-bit
// weights they are codes of that largest value / 127. The largest is found with
// atomic maxima, which do not depend on their order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <mutex>
#include <string>
#include <type_traits>

#include "grouped.h"
#include "kebab/layer.h"
#include "quant_i8.cuh"

namespace kb {
namespace {

constexpr int MAX_TOKENS = KEBAB_FEW_TOKENS, MAX_K = 32;
constexpr int WARPS = 8, THREADS = 32 * (WARPS + 1);  // and the copying one
constexpr int CHUNK = 2048;                           // bytes of a row in a stage, at most
constexpr int STAGE = 16 * (CHUNK + 64);
constexpr int STEPS = CHUNK / 64 / WARPS;             // steps of a chunk that a warp takes, at most
constexpr int MT = 4;                                 // 16-row tiles of a pass
constexpr int RED = 68;                               // floats from one token's partial sums (64 rows) to the next's

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
  int fast;   // weight rows on 16-byte boundaries: copied by the bulk engine
  int vec_x;  // rows of x (or of its codes) on 16-byte boundaries
  const float* router;
  // The workspace.
  float* logits;      // [T][E]
  void* hidden;       // [T k][d_pitch] floats, or twice as many of the weights' type: the rounded values, the rest
  int d_pitch;
  uint32_t* top;      // [T k]: bits of the largest |hidden|
  float* x_scale;     // [T], 8-bit
  int8_t* x_codes;    // [T][x_pitch], 8-bit
  int x_pitch;
  uint32_t* arrived;  // CTAs at the grid barrier
  int pdl;
  WaitCtx ctx;
};

// ------------------------------------------------------------------- logits

template <typename T>
__global__ void __launch_bounds__(256) layer_logits_kernel(const LayerArgs g, int split) {
  __shared__ float part[8][MAX_TOKENS];
  __shared__ uint32_t tops[8];
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(g.x);
  if (blockIdx.x >= g.E) {
    // Codes of a token, nearest to 127 x / amax, ties to even. Of 16-bit values
    // the product is exact and the quotient distinguishes ties from others.
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
    const float amax = __uint_as_float(top);
    int8_t* q = g.x_codes + (int64_t)t * g.x_pitch;
    for (int h = threadIdx.x; h < g.x_pitch; h += 256)
      q[h] = h < g.H && s.inv != 0.f ? (int8_t)__float2int_rn(to_float(x[h]) * 127.f / amax) : 0;
    if (threadIdx.x == 0) g.x_scale[t] = s.scale;
    return;
  }
  const int e = blockIdx.x;
  if (e == 0) {
    for (int i = threadIdx.x; i < g.T * g.k; i += 256) {
      g.top[i] = 0;
      // The hidden values' rows are filled up with zeros (as floats or as pairs).
      float* row = static_cast<float*>(g.hidden) + (int64_t)i * g.d_pitch;
      if (split) {
        T* hi = reinterpret_cast<T*>(row);
        for (int d = g.D; d < g.d_pitch; ++d) hi[d] = hi[g.d_pitch + d] = from_float<T>(0.f);
      } else {
        for (int d = g.D; d < g.d_pitch; ++d) row[d] = 0.f;
      }
    }
    if (threadIdx.x == 0) *g.arrived = 0;
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

template <typename T, bool I8>
struct Mma;
template <>
struct Mma<__half, false> {
  using Acc = float;
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <>
struct Mma<__nv_bfloat16, false> {
  using Acc = float;
  static __device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};
template <typename T>
struct Mma<T, true> {
  using Acc = int;
  static __device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Whether hidden values are stored as two numbers of the weights' type: BF16 has
// FP32's range, F16 needs a scale that is known only when all of them are.
template <typename TX, bool I8>
constexpr bool is_split() {
  return !I8 && std::is_same<TX, __nv_bfloat16>::value;
}

// How rows of `bytes` lie in the ring: chunks of equal size (a multiple of 64
// bytes), tiles of 16 rows at a pitch, `units` tiles to a stage.
struct Shape {
  int64_t bytes;
  int chunks, chunk, pitch, unit, units;
  __device__ __forceinline__ Shape(int64_t row, bool fast) {
    bytes = row;
    chunks = (int)((row + CHUNK - 1) / CHUNK);
    chunk = (int)((row + 64 * (int64_t)chunks - 1) / (64 * (int64_t)chunks)) * 64;
    // Short rows are copied together, as they lie. Others one by one, to an odd
    // multiple of 64 bytes, so that the warps read two rows without a conflict.
    pitch = fast && row < 512 ? (int)row : chunk + (chunk % 128 == 0 ? 64 : 0);
    unit = 16 * pitch;
    units = STAGE / unit;
  }
  __device__ __forceinline__ bool together() const { return pitch == bytes; }
  __device__ __forceinline__ int length(int c) const { return (int)min((int64_t)chunk, bytes - (int64_t)c * chunk); }
};

// Shared memory: the ring, the warps' partial sums, barriers, and tables of the
// choices: weights, scales, factors (float [T k]), experts [T k], the chosen
// experts in ascending order [T k], who chose them ([T k][T]: 32 t + j), how many
// did (bytes [T k]), flags (bytes [E]).
template <int NT>
struct LayerSmem {
  static constexpr int STAGES = NT == 1 ? 6 : 5;
  static constexpr int OFF_RED = STAGES * STAGE;
  static constexpr int OFF_BAR = OFF_RED + WARPS * NT * 8 * RED * 4;
  static constexpr int OFF_TABLES = OFF_BAR + 2 * STAGES * 8 + 16;
  static constexpr int bytes(int T, int k, int E) {
    const int n = T * k;
    return OFF_TABLES + n * 20 + n * T * 2 + n + E + 128;  // and the alignment
  }
  static constexpr int MOST = bytes(NT * 8, MAX_K, kMaxExperts);
  static_assert(MOST <= 232448, "shared memory budget exceeded");
};

// The top-k choices of token t by one warp: as kebab_route.
__device__ __forceinline__ uint32_t order_key(float x) {
  x += 0.f;  // -0 becomes +0: they are equal
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);  // NaN's key gives a NaN
}
__device__ void choose(const LayerArgs& g, int t, float* weights, int* experts) {
  constexpr int V = kMaxExperts / 32;
  const int lane = threadIdx.x & 31;
  uint32_t key[V];
#pragma unroll
  for (int u = 0; u < V; ++u) {
    if (u * 32 >= g.E) break;
    const int e = u * 32 + lane;
    key[u] = e < g.E ? order_key(__ldcg(g.logits + t * g.E + e)) : 0u;
  }
  float highest = 0.f, sum = 0.f, mine = 0.f;
  for (int j = 0; j < g.k; ++j) {
    uint32_t top = 0;
    int e = 0;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      if (u * 32 >= g.E) break;
      if (key[u] > top) top = key[u], e = u * 32 + lane;
    }
    const uint32_t all = __reduce_max_sync(0xffffffffu, top);
    e = (int)__reduce_min_sync(0xffffffffu, top == all ? (unsigned)e : 0xffffffffu);
    const float v = key_value(all);
    if (j == 0) {
      highest = v;
      if (!g.renormalize) {
#pragma unroll
        for (int u = 0; u < V; ++u) {
          if (u * 32 >= g.E) break;
          if (u * 32 + lane < g.E) sum += expf(key_value(key[u]) - highest);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      }
    }
    const float p = highest == -INFINITY ? 0.f : expf(v - highest);  // all logits -inf: nothing to weigh
    if (g.renormalize) sum += p;
    if (lane == j) mine = p;
    if (lane == 0) experts[j] = e;
#pragma unroll
    for (int u = 0; u < V; ++u) {
      if (u * 32 >= g.E) break;
      if (e == u * 32 + lane) key[u] = 0;
    }
  }
  if (lane < g.k) weights[lane] = mine / (highest == -INFINITY ? 1.f : sum);
}

// 2^n by which a choice's values are multiplied, for the bits of the largest
// (0 or not finite: 1), and its inverse.
__device__ __forceinline__ float power_for(uint32_t top, float& inverse) {
  const int e = (int)(top >> 23) - 127;
  const int n = top == 0 || e == 128 ? 0 : max(min(13 - e, 126), -126);
  inverse = __uint_as_float((uint32_t)(127 - n) << 23);
  return __uint_as_float((uint32_t)(127 + n) << 23);
}

template <typename TX, bool I8, int NT>
__global__ void __launch_bounds__(THREADS, 1) layer_kernel(const LayerArgs g) {
  using M = Mma<TX, I8>;
  using Acc = typename M::Acc;
  using L = LayerSmem<NT>;
  constexpr int STAGES = L::STAGES;
  constexpr int ES = I8 ? 1 : 2;       // bytes of a weight
  constexpr int PIECE = 16 / ES;       // values of 16 bytes
  constexpr int PARTS = I8 ? 1 : 2;    // operands that a hidden value makes
  constexpr bool SPLIT = is_split<TX, I8>();
  constexpr int RAW = I8 ? 4 : 2;      // registers of 16 bytes that hold a piece's hidden values as they are stored
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((128u - (smem_u32(smem_raw) & 127u)) & 127u);
  uint32_t* red = reinterpret_cast<uint32_t*>(smem + L::OFF_RED);  // [WARPS][NT * 8][RED]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  int* s_count = reinterpret_cast<int*>(empty + STAGES);  // chosen experts; whether the grid barrier failed
  const int choices = g.T * g.k;
  float* s_weight = reinterpret_cast<float*>(smem + L::OFF_TABLES);
  float* s_scale = s_weight + choices;
  float* s_factor = s_scale + choices;
  int* s_expert = reinterpret_cast<int*>(s_factor + choices);
  int* s_active = s_expert + choices;
  uint16_t* s_who = reinterpret_cast<uint16_t*>(s_active + choices);
  uint8_t* s_many = reinterpret_cast<uint8_t*>(s_who + choices * g.T);
  uint8_t* s_flag = s_many + choices;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const WaitCtx& ctx = g.ctx;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], WARPS);
    }
    fence_barrier_init();
    s_count[1] = 0;
  }
  for (int i = threadIdx.x; i < g.E; i += THREADS) s_flag[i] = 0;
  if (g.pdl) pdl_wait();
  __syncthreads();
  if (warp < WARPS) {
    for (int t = warp; t < g.T; t += WARPS) {
      choose(g, t, s_weight + t * g.k, s_expert + t * g.k);
      __syncwarp();
      if (lane < g.k) s_flag[s_expert[t * g.k + lane]] = 1;
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int e0 = 0; e0 < g.E; e0 += 32) {
      const bool is = e0 + lane < g.E && s_flag[e0 + lane];
      const uint32_t mask = __ballot_sync(0xffffffffu, is);
      if (is) s_active[n + __popc(mask & ((1u << lane) - 1u))] = e0 + lane;
      n += __popc(mask);
    }
    if (lane == 0) s_count[0] = n;
  }
  __syncthreads();
  const int active = s_count[0];
  for (int a = threadIdx.x; a < active; a += THREADS) {
    const int e = s_active[a];
    int n = 0;
    for (int t = 0; t < g.T; ++t)
      for (int j = 0; j < g.k; ++j)
        if (s_expert[t * g.k + j] == e) s_who[a * g.T + n++] = (uint16_t)(32 * t + j);
    s_many[a] = (uint8_t)n;
  }
  __syncthreads();

  const int cta = blockIdx.x, ctas = gridDim.x;
  // This CTA's share of the hidden values (counted over the chosen experts) and of the outputs.
  const int64_t total = (int64_t)active * g.D, p0 = total * cta / ctas, p1 = total * (cta + 1) / ctas;
  const int n0 = (int)((int64_t)g.H * cta / ctas), n1 = (int)((int64_t)g.H * (cta + 1) / ctas);
  const Shape up((int64_t)g.H * ES, g.fast), down((int64_t)g.D * ES, g.fast);
  constexpr int PAIRS = 8 * MT, ROWS = 16 * MT;  // hidden values, outputs of a pass
  auto all_ok = [](bool ok) { return __all_sync(0xffffffffu, ok) != 0; };
  bool ok = true;
  int stage = 0;
  uint32_t phase = 0;
  auto advance = [&] {
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1u;
    }
  };

  if (warp == WARPS) {
    // ------------------------------------------------------------- copies
    int left = 0;  // tiles that the stage has room for
    // Chunk c of the rows src .. of a tile: `rows` of them, or (second) 8 places
    // further on as many from `second`.
    auto tile = [&](const Shape& s, const uint8_t* src, const uint8_t* second, int rows, int c) {
      if (left == 0) {
        ok = all_ok(mbar_wait(&empty[stage], phase ^ 1u, ctx, SITE_EMPTY));
        if (!ok) return;
        left = s.units;
      }
      uint8_t* dst = smem + stage * STAGE + (s.units - left) * s.unit;
      const int len = s.length(c), copies = second ? 2 * rows : rows;
      const int64_t at = (int64_t)c * s.chunk;
      if (g.fast) {
        if (lane == 0) mbar_expect_tx(&full[stage], copies * len);
        __syncwarp();
        if (s.together()) {
          if (lane == 0) bulk_load(dst, src, rows * len, &full[stage]);
          if (lane == 1 && second) bulk_load(dst + 8 * s.pitch, second, rows * len, &full[stage]);
        } else if (second ? (lane & 7) < rows && lane < 16 : lane < rows) {
          const uint8_t* from = second && lane >= 8 ? second + (lane - 8) * s.bytes : src + lane * s.bytes;
          bulk_load(dst + lane * s.pitch, from + at, len, &full[stage]);
        }
      } else {
        // Rows on any boundary, value by value, filled up with zeros to 16 bytes.
        const int n = len / ES, padded = (n + PIECE - 1) / PIECE * PIECE;
        for (int r = 0; r < copies; ++r) {
          const bool is_second = r >= rows;
          const uint8_t* from = (is_second ? second + (r - rows) * s.bytes : src + r * s.bytes) + at;
          uint8_t* to = dst + (is_second ? 8 + r - rows : r) * s.pitch;
          for (int i = lane; i < padded; i += 32) {
            if constexpr (I8) to[i] = i < n ? from[i] : 0;
            else reinterpret_cast<uint16_t*>(to)[i] = i < n ? reinterpret_cast<const uint16_t*>(from)[i] : 0;
          }
        }
      }
      __syncwarp();
      if (--left == 0) {
        if (lane == 0) mbar_arrive(&full[stage]);
        __syncwarp();
        advance();
      }
    };
    auto finish = [&] {
      if (left > 0) {
        if (lane == 0) mbar_arrive(&full[stage]);
        __syncwarp();
        advance();
        left = 0;
      }
    };
    const uint8_t* w_in = static_cast<const uint8_t*>(g.w_in);
    const uint8_t* w_out = static_cast<const uint8_t*>(g.w_out);
    for (int64_t p = p0; p < p1 && ok;) {
      const int a = (int)(p / g.D), i0 = (int)(p - (int64_t)a * g.D);
      const int n = (int)min((int64_t)min(PAIRS, g.D - i0), p1 - p);
      const uint8_t* gate = w_in + ((int64_t)s_active[a] * 2 * g.D + i0) * up.bytes;
      for (int c = 0; c < up.chunks && ok; ++c)
        for (int m = 0; m < n && ok; m += 8)
          tile(up, gate + m * up.bytes, gate + ((int64_t)g.D + m) * up.bytes, min(8, n - m), c);
      p += n;
    }
    if (ok) finish();
    for (int r0 = n0; r0 < n1 && ok; r0 += ROWS) {
      const int n = min(ROWS, n1 - r0);
      for (int a = 0; a < active && ok; ++a) {
        const uint8_t* w = w_out + ((int64_t)s_active[a] * g.H + r0) * down.bytes;
        for (int c = 0; c < down.chunks && ok; ++c)
          for (int m = 0; m < n && ok; m += 16) tile(down, w + m * down.bytes, nullptr, min(16, n - m), c);
      }
    }
    if (ok) finish();
  } else {
    // ----------------------------------------------------------- products
    // The columns of an MMA are the tokens that chose the expert. More than 8
    // are rare; they take a second MMA, whose operands are not loaded ahead.
    const int gq = lane >> 2, cq = lane & 3;
    using One = std::integral_constant<int, 1>;
    using All = std::integral_constant<int, PARTS>;
    int left = 0;
    const uint8_t* at = nullptr;
    Acc acc[MT][NT][4];
    uint32_t b[STEPS][NT][PARTS][4];
    auto clear = [&] {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][n][i] = 0;
    };
    auto release = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      advance();
      left = 0;
    };
    // The next tile, with the first `parts` operands of every value, in two
    // chains of MMAs.
    auto multiply = [&](const Shape& s, int len, bool wide, auto parts, Acc (&d)[NT][4]) {
      if (left == 0) {
        if (ok) ok = all_ok(mbar_wait(&full[stage], phase, ctx, SITE_FULL));
        left = s.units;
        at = smem + stage * STAGE;
      } else {
        at += s.unit;
      }
      constexpr bool TWO = decltype(parts)::value == 2;
      const uint8_t* row = at + gq * s.pitch + cq * 16;
      Acc f[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[n][i] = 0;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int off = (warp + i * WARPS) * 64;
        if (off >= len) break;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        if (off + cq * 16 < len) {  // past the end of the row there may be anything
          lo = *reinterpret_cast<const uint4*>(row + off);
          hi = *reinterpret_cast<const uint4*>(row + 8 * s.pitch + off);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (n > 0 && !wide) break;
          M::mma(d[n], lo.x, hi.x, lo.y, hi.y, b[i][n][0][0], b[i][n][0][1]);
          if constexpr (TWO) M::mma(f[n], lo.x, hi.x, lo.y, hi.y, b[i][n][PARTS - 1][0], b[i][n][PARTS - 1][1]);
          M::mma(TWO ? d[n] : f[n], lo.z, hi.z, lo.w, hi.w, b[i][n][0][2], b[i][n][0][3]);
          if constexpr (TWO) M::mma(f[n], lo.z, hi.z, lo.w, hi.w, b[i][n][PARTS - 1][2], b[i][n][PARTS - 1][3]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[n][i] += f[n][i];
      if (--left == 0) release();
    };
    auto meet = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    // The sum over the warps of row r of column t.
    auto total_of = [&](int t, int r) {
      const uint32_t* from = red + t * RED + r;
      Acc sum = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const uint32_t v = from[w * NT * 8 * RED];
        if constexpr (I8) sum += (int)v;
        else sum += __uint_as_float(v);
      }
      return sum;
    };

    // Hidden values: a = silu(gate) * up. The tokens' values of this warp's steps
    // are loaded a chunk ahead.
    uint4 next[STEPS];
    auto fetch = [&](int a, int c, int n, uint4 (&to)[STEPS]) {
      const int len = up.length(c), col = n * 8 + gq;
      const bool is = col < s_many[a];
      const int t = is ? s_who[a * g.T + col] >> 5 : 0;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int off = (warp + i * WARPS) * 64 + cq * 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (is && off < len) {
          const int64_t k0 = ((int64_t)c * up.chunk + off) / ES;
          if constexpr (I8) {
            v = *reinterpret_cast<const uint4*>(g.x_codes + (int64_t)t * g.x_pitch + k0);
          } else {
            const uint16_t* x = static_cast<const uint16_t*>(g.x) + t * g.ldx + k0;
            if (g.vec_x && k0 + 8 <= g.H) {
              v = *reinterpret_cast<const uint4*>(x);
            } else {
              uint32_t h[8];
#pragma unroll
              for (int u = 0; u < 8; ++u) h[u] = k0 + u < g.H ? x[u] : 0;
              v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
            }
          }
        }
        to[i] = v;
      }
    };
    auto operands = [&](int n, const uint4 (&from)[STEPS]) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const uint4 v = from[i];
        b[i][n][0][0] = v.x, b[i][n][0][1] = v.y, b[i][n][0][2] = v.z, b[i][n][0][3] = v.w;
      }
    };
    if (p0 < p1) fetch((int)(p0 / g.D), 0, 0, next);
    for (int64_t p = p0; p < p1;) {
      const int a = (int)(p / g.D), i0 = (int)(p - (int64_t)a * g.D);
      const int n = (int)min((int64_t)min(PAIRS, g.D - i0), p1 - p);
      const bool wide = NT > 1 && s_many[a] > 8;
      clear();
      for (int c = 0; c < up.chunks; ++c) {
        operands(0, next);
        if (wide) {
          fetch(a, c, NT - 1, next);
          operands(NT - 1, next);
        }
        if (c + 1 < up.chunks) fetch(a, c + 1, 0, next);
        else if (p + n < p1) fetch(i0 + n < g.D ? a : a + 1, 0, 0, next);
        const int len = up.length(c);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (m * 8 < n) multiply(up, len, wide, One(), acc[m]);
      }
      // This warp's partial sums: column, then row.
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if (nt > 0 && !wide) break;
          uint32_t* to = red + ((warp * NT + nt) * 8 + 2 * cq) * RED + m * 16 + gq;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const Acc v = acc[m][nt][i];
            to[(i & 1) * RED + (i >> 1) * 8] = *reinterpret_cast<const uint32_t*>(&v);
          }
        }
      meet();
      // A warp a column, a lane a value.
      for (int col = warp; col < s_many[a]; col += WARPS) {
        const int who = s_who[a * g.T + col], t = who >> 5, choice = t * g.k + (who & 31);
        const int row = lane / 8 * 16 + lane % 8, i = i0 + lane;
        float gate = (float)total_of(col, row), value = (float)total_of(col, row + 8);
        if constexpr (I8) {
          const float s = g.x_scale[t];
          const float* scale = g.in_scale + (int64_t)s_active[a] * 2 * g.D + i;
          gate *= s * (lane < n ? scale[0] : 0.f);
          value *= s * (lane < n ? scale[g.D] : 0.f);
        }
        const float h = gate / (1.f + expf(-gate)) * value;
        if constexpr (SPLIT) {
          if (lane < n && ok) {
            TX* to = static_cast<TX*>(g.hidden) + (int64_t)choice * 2 * g.d_pitch + i;
            const TX hi = from_float<TX>(h);
            to[0] = hi;
            to[g.d_pitch] = from_float<TX>(isinf(to_float(hi)) ? 0.f : h - to_float(hi));  // what the rounding left
          }
        } else {
          if (lane < n && ok) static_cast<float*>(g.hidden)[(int64_t)choice * g.d_pitch + i] = h;
          const uint32_t top = __reduce_max_sync(0xffffffffu, lane < n ? abs_bits(h) : 0u);
          if (lane == 0) atomicMax(g.top + choice, top);
        }
      }
      meet();
      p += n;
    }
    if (left > 0) release();

    // The grid barrier.
    __threadfence();
    meet();
    if (threadIdx.x == 0) {
      asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(g.arrived) : "memory");
      const uint64_t t0 = globaltimer();
      for (uint32_t it = 1;; ++it) {
        uint32_t n;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(g.arrived) : "memory");
        if (n >= (uint32_t)ctas) break;
        if ((it & 63u) == 0u) {
          if (!aborted(ctx.status) && globaltimer() - t0 <= ctx.timeout_ns) continue;
          record_error(ctx.status, DEV_TIMEOUT, SITE_GRID);
          s_count[1] = 1;
          break;
        }
      }
      __threadfence();
    }
    meet();
    if (s_count[1]) ok = false;
    // What a choice's values are multiplied by before they are rounded, and its
    // products after: the inverse, and the choice's weight.
    for (int i = threadIdx.x; i < choices; i += 32 * WARPS) {
      float inverse = 1.f;
      if constexpr (I8) {
        const RowScale code = row_scale(__ldcg(g.top + i));
        s_scale[i] = code.inv;
        inverse = code.scale;
      } else if constexpr (!SPLIT) {
        s_scale[i] = power_for(__ldcg(g.top + i), inverse);
      }
      s_factor[i] = s_weight[i] * inverse;
    }
    meet();

    // Outputs. The hidden values are loaded a chunk ahead, too.
    uint4 raw[STEPS][RAW];
    auto load = [&](int a, int c, int n) {
      const int len = down.length(c), col = n * 8 + gq;
      const bool is = col < s_many[a];
      const int who = is ? s_who[a * g.T + col] : 0, choice = (who >> 5) * g.k + (who & 31);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int off = (warp + i * WARPS) * 64 + cq * 16;
        const int64_t k0 = ((int64_t)c * down.chunk + off) / ES;
        const uint4* from;
        if constexpr (SPLIT) from = reinterpret_cast<const uint4*>(static_cast<const TX*>(g.hidden) + (int64_t)choice * 2 * g.d_pitch + k0);
        else from = reinterpret_cast<const uint4*>(static_cast<const float*>(g.hidden) + (int64_t)choice * g.d_pitch + k0);
        const int64_t step = SPLIT ? g.d_pitch / 8 : 1;
#pragma unroll
        for (int u = 0; u < RAW; ++u)
          raw[i][u] = is && off < len ? __ldcg(from + u * step) : make_uint4(0, 0, 0, 0);
      }
    };
    auto convert = [&](int a, int n) {
      if constexpr (SPLIT) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const uint4 v = raw[i][p];
            uint32_t* to = b[i][n][p % PARTS];
            to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
          }
      } else {
        const int col = n * 8 + gq;
        const bool is = col < s_many[a];
        const int who = is ? s_who[a * g.T + col] : 0;
        const float scale = is ? s_scale[(who >> 5) * g.k + (who & 31)] : 0.f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          float v[RAW * 4];
#pragma unroll
          for (int u = 0; u < RAW; ++u) {
            v[4 * u] = __uint_as_float(raw[i][u].x), v[4 * u + 1] = __uint_as_float(raw[i][u].y);
            v[4 * u + 2] = __uint_as_float(raw[i][u].z), v[4 * u + 3] = __uint_as_float(raw[i][u].w);
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if constexpr (I8) {
              uint32_t code[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) code[u] = code_bits(v[4 * q + u], scale);
              b[i][n][0][q] = scale == 0.f ? 0u : pack4(code[0], code[1], code[2], code[3]);
            } else {
              const float x0 = v[2 * q] * scale, x1 = v[2 * q + 1] * scale;
              const __half2 hi = __floats2half2_rn(x0, x1);
              const float2 h = __half22float2(hi);
              // What the rounding left; of an infinity nothing.
              const __half2 lo = __floats2half2_rn(isinf(x0) ? 0.f : x0 - h.x, isinf(x1) ? 0.f : x1 - h.y);
              b[i][n][0][q] = *reinterpret_cast<const uint32_t*>(&hi);
              b[i][n][PARTS - 1][q] = *reinterpret_cast<const uint32_t*>(&lo);
            }
          }
        }
      }
    };
    if (n0 < n1) load(0, 0, 0);
    float* sums = reinterpret_cast<float*>(red) + warp * NT * 8 * RED;  // this warp's: token, then row
    for (int r0 = n0; r0 < n1; r0 += ROWS) {
      const int n = min(ROWS, n1 - r0);
      for (int i = lane; i < NT * 8 * RED; i += 32) sums[i] = 0.f;
      __syncwarp();
      for (int a = 0; a < active; ++a) {
        const bool wide = NT > 1 && s_many[a] > 8;
        clear();
        for (int c = 0; c < down.chunks; ++c) {
          convert(a, 0);
          if (wide) {
            load(a, c, NT - 1);
            convert(a, NT - 1);
          }
          if (c + 1 < down.chunks) load(a, c + 1, 0);
          else load(a + 1 < active ? a + 1 : 0, 0, 0);
          const int len = down.length(c);
#pragma unroll
          for (int m = 0; m < MT; ++m)
            if (m * 16 < n) multiply(down, len, wide, All(), acc[m]);
        }
        // Onto the tokens' sums.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int col = nt * 8 + 2 * cq + u;
            if (col >= s_many[a]) continue;
            const int who = s_who[a * g.T + col], t = who >> 5;
            const float factor = s_factor[t * g.k + (who & 31)];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              if (m * 16 >= n) break;
#pragma unroll
              for (int v = 0; v < 2; ++v) {
                float f = factor;
                if constexpr (I8) {
                  const int r = r0 + m * 16 + v * 8 + gq;
                  f *= r < n1 ? g.out_scale[(int64_t)s_active[a] * g.H + r] : 0.f;
                }
                sums[t * RED + m * 16 + v * 8 + gq] += f * (float)acc[m][nt][2 * v + u];
              }
            }
          }
        __syncwarp();  // another lane may have the token's column of the next expert
      }
      meet();
      for (int t = warp; t < g.T; t += WARPS) {
        for (int r = lane; r < n; r += 32) {
          const float* from = reinterpret_cast<const float*>(red) + t * RED + r;
          float sum = 0.f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) sum += from[w * NT * 8 * RED];
          if (ok) static_cast<TX*>(g.y)[t * g.ldy + r0 + r] = from_float<TX>(sum);
        }
      }
      meet();
    }
    if (left > 0) release();
  }
  // A wait ran out: what is in flight has to land before the CTA leaves.
  if (__syncthreads_or(!ok)) settle();
}

// ---------------------------------------------------------------- host side

struct Sizes {
  int64_t T, E, k, H, D;
};

int64_t up16(int64_t v) { return (v + 15) / 16 * 16; }

// logits, hidden values, their largest, the tokens' scales, the barrier's count; the tokens' codes.
int64_t words(const Sizes& s) { return up16(s.T * s.E * 4) + s.T * s.k * up16(s.D) * 4 + up16(s.T * s.k * 4) + 64 + 16; }
int64_t bytes(const Sizes& s) { return words(s) + s.T * up16(s.H); }

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
  if (s.H <= 0 || s.D <= 0 || s.H > (1 << 24) || s.D > (1 << 24))
    return fail(KEBAB_EINVAL, w + ": invalid dimensions H=" + std::to_string(s.H) + " D=" + std::to_string(s.D));
  if (ldx < s.H || ldy < s.H) return fail(KEBAB_EINVAL, w + ": a row pitch is below the row length");
  if (s.T == 0) return KEBAB_OK;
  if (!x || !router || !w_in || !w_out || !y) return fail(KEBAB_EINVAL, w + ": null pointer");
  if (!ws || ws_bytes < bytes(s) || (reinterpret_cast<uintptr_t>(ws) & 15u))
    return fail(KEBAB_EINVAL, w + ": the workspace is null, too small or not 16-byte aligned");
  return KEBAB_OK;
}

template <typename TX, bool I8, int NT>
int launch(LayerArgs& g, cudaStream_t stream) {
  int rc;
  DeviceInfo* dev = nullptr;
  if ((rc = device_info(&dev)) || (rc = wait_ctx(&g.ctx))) return rc;
  g.pdl = pdl_enabled();
  auto kern = layer_kernel<TX, I8, NT>;
  static std::once_flag once[64];
  static cudaError_t err[64];
  const int di = dev->device & 63;
  std::call_once(once[di], [&] {
    err[di] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   LayerSmem<NT>::MOST);
  });
  if (err[di] != cudaSuccess) return cuda_fail(err[di], "cudaFuncSetAttribute(max dynamic smem)");
  PdlLaunch first(dim3((unsigned)(g.E + (I8 ? g.T : 0))), dim3(256), 0, stream);
  cudaError_t e = cudaLaunchKernelEx(&first.cfg, layer_logits_kernel<TX>, (const LayerArgs)g, (int)is_split<TX, I8>());
  if (e != cudaSuccess) return cuda_fail(e, "expert_layer: logits launch");
  const int smem = LayerSmem<NT>::bytes(g.T, g.k, g.E);
  PdlLaunch l(dim3((unsigned)dev->sm_count), dim3(THREADS), smem, stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  if (l.cfg.numAttrs) attr[1] = l.attr[0];
  l.cfg.attrs = attr;
  ++l.cfg.numAttrs;
  e = cudaLaunchKernelEx(&l.cfg, kern, (const LayerArgs)g);
  return e == cudaSuccess ? KEBAB_OK : cuda_fail(e, "expert_layer launch");
}

template <bool I8>
int run(int dtype, LayerArgs g, const Sizes& s, void* ws, kebab_stream_t stream) {
  constexpr int ES = I8 ? 1 : 2;
  g.T = (int)s.T, g.E = (int)s.E, g.k = (int)s.k, g.H = (int)s.H, g.D = (int)s.D;
  uint8_t* at = static_cast<uint8_t*>(ws);
  auto take = [&](int64_t n) {
    uint8_t* p = at;
    at += up16(n);
    return p;
  };
  g.logits = reinterpret_cast<float*>(take(s.T * s.E * 4));
  g.d_pitch = (int)up16(s.D);
  g.hidden = take(s.T * s.k * g.d_pitch * 4);
  g.top = reinterpret_cast<uint32_t*>(take(s.T * s.k * 4));
  g.x_scale = reinterpret_cast<float*>(take(64));
  g.arrived = reinterpret_cast<uint32_t*>(take(16));
  g.x_codes = reinterpret_cast<int8_t*>(at);
  g.x_pitch = (int)up16(s.H);
  auto on16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  g.fast = on16(g.w_in) && on16(g.w_out) && s.H * ES % 16 == 0 && s.D * ES % 16 == 0;
  g.vec_x = on16(g.x) && g.ldx % 8 == 0;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == KEBAB_F16) return s.T <= 8 ? launch<__half, I8, 1>(g, st) : launch<__half, I8, 2>(g, st);
  return s.T <= 8 ? launch<__nv_bfloat16, I8, 1>(g, st) : launch<__nv_bfloat16, I8, 2>(g, st);
}
}  // namespace
}  // namespace kb

using namespace kb;

extern "C" {

int64_t kebab_expert_layer_workspace(int64_t T, int64_t E, int k, int64_t H, int64_t D) {
  if (T < 0 || T > KEBAB_FEW_TOKENS || E < 1 || E > kMaxExperts || k < 1 || k > MAX_K || H <= 0 || D <= 0 ||
      H > (1 << 24) || D > (1 << 24))
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
