// The token sort of one chunk of routes, and the keys and wavefront maximum, that the routers share (moe.hip,
// router_grouped.hip).
#pragma once

#include "mx_common.h"

namespace mxl {

constexpr int kChunk = 1024;

// Routes of the same key in the earlier lanes of this wavefront (the rank of the lane's
// route among its expert's routes in the wavefront); key = the expert id, or E for a
// route whose expert is outside [0, E).  The lanes holding the same key are found one key
// bit at a time with a ballot -- a bit's ballot, or its complement where the lane's bit
// is 0, keeps the lanes that agree on it -- bit_width(E) ballots (9 for 256 experts)
// instead of 64 lane-by-lane comparisons; only wavefront-uniform control flow, so every
// lane takes part in every ballot.
__device__ __forceinline__ int same_expert_rank(int key, int E, int lane) {
  const int bits = 32 - __builtin_clz((unsigned)E);
  uint64_t same = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const bool bit = (key >> b) & 1;
    const uint64_t on = __ballot(bit);
    same &= bit ? on : ~on;
  }
  return __popcll(same & ((1ull << lane) - 1ull));
}

// All routes in one chunk (R <= 1024, E <= 1024): the three passes in one
// workgroup -- per-wavefront expert counts in LDS, per-expert totals scanned into
// the offsets, then the same rank and scatter -- so a decode-sized step pays one
// launch.  The result is the multi-chunk path's (chunk base 0).
constexpr int kSingleMaxExperts = 1024;
// Largest expert count any route schedule launches: the scatter's (kChunk / 64) * E
// ints of LDS must fit gfx950's 160 KiB per workgroup.
constexpr int kRouteMaxExperts = 160 * 1024 / ((kChunk / 64) * (int)sizeof(int32_t));
static_assert(kRouteMaxExperts == 2560, "the documented expert limit");

// The single-chunk sort for route t (expert e, -1 if none): per-wavefront expert counts in
// LDS, per-expert totals scanned into the offsets, then the rank and scatter.  Called by
// every thread of a 1024-thread workgroup (t = threadIdx.x).
__device__ __forceinline__ void single_chunk_sort(int32_t e, int64_t R, int E, int64_t* __restrict__ expert_offsets,
                                                  int32_t* __restrict__ sorted_routes,
                                                  int32_t* __restrict__ inverse, int32_t* whist,
                                                  int32_t (*tot)[kSingleMaxExperts]) {
  constexpr int W = kChunk / 64;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  for (int i = t; i < W * E; i += kChunk) whist[i] = 0;
  const bool valid = e >= 0 && e < E;
  const int rank = same_expert_rank(valid ? e : E, E, lane);
  __syncthreads();
  if (valid) atomicAdd(&whist[w * E + e], 1);
  __syncthreads();
  for (int x = t; x < E; x += kChunk) {  // per-wavefront bases and the expert's total
    int32_t run = 0;
    for (int v = 0; v < W; ++v) {
      const int32_t n = whist[v * E + x];
      whist[v * E + x] = run;
      run += n;
    }
    tot[0][x] = run;
  }
  __syncthreads();
  int src = 0;  // inclusive scan of the totals (ping-pong)
  for (int d = 1; d < E; d <<= 1) {
    for (int x = t; x < E; x += kChunk) {
      int32_t v = tot[src][x];
      if (x >= d) v += tot[src][x - d];
      tot[1 - src][x] = v;
    }
    __syncthreads();
    src = 1 - src;
  }
  for (int x = t; x < E; x += kChunk) expert_offsets[x + 1] = tot[src][x];
  if (t == 0) expert_offsets[0] = 0;
  if (t >= R) return;
  if (!valid) {
    inverse[t] = -1;
    return;
  }
  const int32_t pos = (e > 0 ? tot[src][e - 1] : 0) + whist[w * E + e] + rank;
  sorted_routes[pos] = t;
  inverse[t] = pos;
}

// Binary32 as an unsigned key in value order (-0 read as +0, so equal values tie; NaNs
// order outside the finite values by sign).
__device__ __forceinline__ uint32_t order_key(float x) {
  uint32_t u = f2u(x);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The wavefront's largest value, in every lane: an inclusive maximum along the lanes (rows of
// 16, then across rows), read from lane 63.  Lanes without a source keep 0.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define MXL_DPP_MAX(CTRL_, ROWS_)                                                              \
  {                                                                                            \
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL_, ROWS_, 0xf, false); \
    v = o > v ? o : v;                                                                         \
  }
  MXL_DPP_MAX(0x111, 0xf)  // row_shr:1, 2, 4, 8
  MXL_DPP_MAX(0x112, 0xf)
  MXL_DPP_MAX(0x114, 0xf)
  MXL_DPP_MAX(0x118, 0xf)
  MXL_DPP_MAX(0x142, 0xa)  // row_bcast:15 into rows 1 and 3
  MXL_DPP_MAX(0x143, 0xc)  // row_bcast:31 into rows 2 and 3
#undef MXL_DPP_MAX
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

}  // namespace mxl
