// Which rows a block of a grouped product takes, found on the device.
#pragma once
#include "grouped.h"

namespace kb {
namespace {

// The group that holds the `nth` of the tiles (of up to WIDTH rows of one group)
// of all groups, its rows begin .. begin + rows - 1, and which of its tiles that
// is; by all THREADS threads of the block, a group a thread. False if there are
// fewer tiles. offsets null: one group of all R rows.
template <int THREADS, int WIDTH>
__device__ bool nth_tile(const int32_t* offsets, int E, int R, int nth, int& e, int& begin, int& rows, int& at) {
  __shared__ int s_count[THREADS / 32], s_found[4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  at = nth;
  if (offsets == nullptr) {
    e = 0;
    begin = 0;
    rows = R;
  } else {
    if (threadIdx.x == 0) s_found[0] = -1;
    int before = 0;
    for (int e0 = 0; e0 < E; e0 += THREADS) {
      int b = 0, n = 0;
      if (e0 + (int)threadIdx.x < E) group_range(offsets, e0 + threadIdx.x, R, b, n);
      const int tiles = (n + WIDTH - 1) / WIDTH;
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (lane == 31) s_count[warp] = sum;
      __syncthreads();
      int first = before + sum - tiles;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) first += s_count[w];
        before += s_count[w];
      }
      if (first <= nth && nth < first + tiles) {
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
  return at < (rows + WIDTH - 1) / WIDTH;
}

// The same with a group in as many equal shares as it has tiles: rows begin ..
// begin + rows - 1 of group e.
template <int THREADS, int WIDTH>
__device__ bool nth_share(const int32_t* offsets, int E, int R, int nth, int& e, int& begin, int& rows) {
  int at;
  if (!nth_tile<THREADS, WIDTH>(offsets, E, R, nth, e, begin, rows, at)) return false;
  const int shares = (rows + WIDTH - 1) / WIDTH, share = (rows + shares - 1) / shares;
  begin += at * share;
  rows = min(share, rows - at * share);
  return rows > 0;
}

// 16 bytes into a peer's shared memory; the bytes count towards the peer's
// mbarrier (both given as shared::cluster addresses).
__device__ __forceinline__ void send16(uint32_t dst, uint32_t bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(dst),
               "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
               : "memory");
}

}  // namespace
}  // namespace kb
