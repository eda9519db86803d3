// MoE token sort and weighted combine for gfx950.
//
// Token sort: routes r = t * topk + k are grouped by expert id, keeping
// ascending r inside each expert (a stable counting sort), which yields
//   expert_offsets[E + 1]  exclusive prefix of per-expert route counts
//   sorted_routes[pos]     route at each sorted position
//   inverse[r]             sorted position of each route (-1 if dropped)
// Three passes over 1024-route chunks: per-chunk histograms (LDS atomics,
// order free), a scan over the chunks, 16 experts a workgroup, then a pass that adds up the
// experts' totals, ranks each route inside its chunk (a ballot match of the expert id's bits inside the
// wavefront plus an LDS prefix over the chunk's 16 wavefronts) and scatters.  A single chunk
// (decode-sized steps) runs all three in one workgroup; up to 40 chunks (32 past 256
// experts) run them in one launch that counts in every workgroup.
//
// Combine: out[t, h] = bf16(sum_k y[inverse[t*topk + k], h] * w[t, k]),
// each product rounded to binary32 and added in ascending k from zero.
#include "moe_sort.h"

namespace mxl {

int cu_count();  // compute units of the current device (gemm_stream.hip)

__global__ __launch_bounds__(kChunk) void route_hist_kernel(const int32_t* __restrict__ ids, int64_t R, int E,
                                                           int32_t* __restrict__ chunk_counts) {
  extern __shared__ int32_t hist[];
  const int64_t c = blockIdx.x;
  for (int e = threadIdx.x; e < E; e += blockDim.x) hist[e] = 0;
  __syncthreads();
  const int64_t r = c * kChunk + threadIdx.x;
  if (r < R) {
    const int32_t e = ids[r];
    if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) chunk_counts[c * E + e] = hist[e];
}

// Chunk counts per expert to their inclusive sums over the chunks, in place.  A workgroup takes 16 experts, 64 threads
// of it one's chunks, each first adding up its own.  (131072 routes of 256 experts, 128 chunks: 29 us in one workgroup
// with a thread an expert, 10 us with four, 4.4 here.)
constexpr int kScanExperts = 16;
__global__ __launch_bounds__(1024) void route_scan_kernel(int32_t* __restrict__ chunk_counts, int64_t C, int E) {
  constexpr int B = 8, P = 1024 / kScanExperts;
  __shared__ int32_t waves[16][kScanExperts];
  const int t = threadIdx.x, col = t % kScanExperts, e = blockIdx.x * kScanExperts + col, w = t >> 6;
  const int64_t per = (C + P - 1) / P, c0 = t / kScanExperts * per, c1 = e < E ? (c0 + per < C ? c0 + per : C) : c0;
  int32_t v[B], sum = 0;
  for (int64_t c = c0; c < c1; c += B) {
#pragma unroll
    for (int k = 0; k < B; ++k) v[k] = c + k < c1 ? chunk_counts[(c + k) * E + e] : 0;
#pragma unroll
    for (int k = 0; k < B; ++k) sum += v[k];
  }
  int32_t run = sum;  // over the wavefront's four threads of the expert, then over the wavefronts
#pragma unroll
  for (int d = kScanExperts; d < 64; d <<= 1) {
    const int32_t before = __shfl_up(run, d, 64);
    if ((t & 63) >= d) run += before;
  }
  if ((t & 63) >= 64 - kScanExperts) waves[w][col] = run;
  __syncthreads();
  run -= sum;
  for (int k = 0; k < w; ++k) run += waves[k][col];
  for (int64_t c = c0; c < c1; c += B) {
    if (per > B) {  // (else v holds them)
#pragma unroll
      for (int k = 0; k < B; ++k) v[k] = c + k < c1 ? chunk_counts[(c + k) * E + e] : 0;
    }
#pragma unroll
    for (int k = 0; k < B; ++k)
      if (c + k < c1) {
        run += v[k];
        chunk_counts[(c + k) * E + e] = run;
      }
  }
}

// A chunk's routes to their places; every workgroup adds up the experts' totals (the last chunk's sums) to their
// offsets, the first writes those out.
__global__ __launch_bounds__(kChunk) void route_scatter_kernel(const int32_t* __restrict__ ids, int64_t R, int64_t C,
                                                              int E, const int32_t* __restrict__ chunk_sums,
                                                              int64_t* __restrict__ expert_offsets,
                                                              int32_t* __restrict__ sorted_routes,
                                                              int32_t* __restrict__ inverse) {
  extern __shared__ int32_t whist[];  // [kChunk / 64][E]
  const int64_t c = blockIdx.x;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  constexpr int W = kChunk / 64, X = (kRouteMaxExperts + kChunk - 1) / kChunk;
  const int64_t r = c * kChunk + t;
  const int32_t e = r < R ? ids[r] : -1;
  int32_t first[X], carry = 0;  // of experts t, t + kChunk, ..: the chunk's first place behind its own routes
#pragma unroll
  for (int i = 0; i < X; ++i) {
    const int x = t + i * kChunk;
    first[i] = 0;
    if (i * kChunk >= E) break;
    const int32_t total = x < E && C > 0 ? chunk_sums[(C - 1) * E + x] : 0;
    const int32_t here = x < E && C > 0 ? chunk_sums[c * E + x] : 0;
    int32_t run = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t before = __shfl_up(run, d, 64);
      if (lane >= d) run += before;
    }
    if (lane == 63) whist[w] = run;
    __syncthreads();
    run += carry;
    for (int k = 0; k < W; ++k) {
      const int32_t n = whist[k];
      run += k < w ? n : 0;
      carry += n;
    }
    if (c == 0 && x < E) expert_offsets[x + 1] = run;
    first[i] = run - total + here;
    __syncthreads();
  }
  if (c == 0 && t == 0) expert_offsets[0] = 0;
  for (int i = t; i < W * E; i += blockDim.x) whist[i] = 0;
  const bool valid = e >= 0 && e < E;
  const int rank = same_expert_rank(valid ? e : E, E, lane);
  __syncthreads();
  if (valid) atomicAdd(&whist[w * E + e], 1);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < X; ++i) {
    const int x = t + i * kChunk;
    if (x < E) {
      int32_t n[W];
#pragma unroll
      for (int v = 0; v < W; ++v) n[v] = whist[v * E + x];
      int32_t run = first[i];
#pragma unroll
      for (int v = W - 1; v >= 0; --v) {
        run -= n[v];
        whist[v * E + x] = run;
      }
    }
  }
  __syncthreads();
  if (r >= R) return;
  if (!valid) {
    inverse[r] = -1;
    return;
  }
  const int32_t pos = whist[w * E + e] + rank;
  sorted_routes[pos] = (int32_t)r;
  inverse[r] = pos;
}

__global__ __launch_bounds__(kChunk) void route_single_kernel(const int32_t* __restrict__ ids, int64_t R, int E,
                                                             int64_t* __restrict__ expert_offsets,
                                                             int32_t* __restrict__ sorted_routes,
                                                             int32_t* __restrict__ inverse) {
  __shared__ int32_t whist[(kChunk / 64) * kSingleMaxExperts];
  __shared__ int32_t tot[2][kSingleMaxExperts];
  const int t = threadIdx.x;
  single_chunk_sort(t < R ? ids[t] : -1, R, E, expert_offsets, sorted_routes, inverse, whist, tot);
}

// 2 .. sort_max_chunks chunks in one launch (E <= 1024): every workgroup counts all routes for
// itself, those of the chunks before its own apart from the rest (one LDS atomic per route and
// workgroup), scans the totals into the offsets, which workgroup 0 writes, and ranks and
// scatters its chunk as route_scatter_kernel does.  Repeating the counts costs less than the
// three launches that share them up to 40 chunks, where a thread counts 40 (256 experts, us: 16
// chunks 6.9, 40 9.6, 48 10.5, 128 20.4, against 10.0 at 49 and 11.0 at 128; 1024 experts 33
// chunks 11.6 against 11.0, so 32).
constexpr int sort_max_chunks(int64_t E) { return E <= 256 ? 40 : 32; }
__global__ __launch_bounds__(kChunk) void route_sort_kernel(const int32_t* __restrict__ ids, int64_t R, int C, int E,
                                                           int64_t* __restrict__ expert_offsets,
                                                           int32_t* __restrict__ sorted_routes,
                                                           int32_t* __restrict__ inverse) {
  constexpr int W = kChunk / 64;
  extern __shared__ int32_t lds[];
  int32_t* const whist = lds;                                           // [W][E]
  int32_t *const before = whist + W * E, *const rest = before + E;      // routes of earlier chunks, of the others
  int32_t* const tot[2] = {rest + E, rest + 2 * E};
  const int c = blockIdx.x, t = threadIdx.x, w = t >> 6, lane = t & 63;
  for (int i = t; i < W * E + 2 * E; i += kChunk) lds[i] = 0;
  __syncthreads();
  int32_t e = -1;
  for (int c0 = 0; c0 < C; c0 += 8) {
    int32_t x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t r = (int64_t)(c0 + k) * kChunk + t;
      x[k] = r < R ? ids[r] : -1;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c0 + k == c) e = x[k];
      if (x[k] >= 0 && x[k] < E) atomicAdd((c0 + k < c ? before : rest) + x[k], 1);
    }
  }
  const int64_t r = (int64_t)c * kChunk + t;
  const bool valid = e >= 0 && e < E;
  const int rank = same_expert_rank(valid ? e : E, E, lane);
  if (valid) atomicAdd(&whist[w * E + e], 1);
  __syncthreads();
  for (int x = t; x < E; x += kChunk) tot[0][x] = before[x] + rest[x];
  int src = 0;  // inclusive scan of the totals (ping-pong)
  for (int d = 1; d < E; d <<= 1) {
    __syncthreads();
    for (int x = t; x < E; x += kChunk) {
      int32_t v = tot[src][x];
      if (x >= d) v += tot[src][x - d];
      tot[1 - src][x] = v;
    }
    src = 1 - src;
  }
  __syncthreads();
  if (c == 0) {
    for (int x = t; x < E; x += kChunk) expert_offsets[x + 1] = tot[src][x];
    if (t == 0) expert_offsets[0] = 0;
  }
  for (int x = t; x < E; x += kChunk) {
    int32_t run = before[x] + (x > 0 ? tot[src][x - 1] : 0);
    for (int v = 0; v < W; ++v) {
      const int32_t n = whist[v * E + x];
      whist[v * E + x] = run;
      run += n;
    }
  }
  __syncthreads();
  if (r >= R) return;
  if (!valid) {
    inverse[r] = -1;
    return;
  }
  const int32_t pos = whist[w * E + e] + rank;
  sorted_routes[pos] = (int32_t)r;
  inverse[r] = pos;
}

// ------------------------------------------------------------------ router
//
// softmax -> top-k -> (renormalize) from router logits, the selection of vLLM's fused
// top-k softmax that the reference's MoE layer runs before its experts (select_experts;
// src/vllm_mach/mxfp6/moe.py:142-152 fuses it into qwen35_router_quant_out): the k largest
// logits of a token (softmax is increasing, so they are its k largest probabilities), ties
// to the lower expert index, weights exp(x - max) / sum, the sum over the k selected
// (renormalize) or over every expert.  One wavefront per token, the token's logits spread
// over its lanes (expert i at lane i % 64, slot i / 64; NS slots, 4 for up to 256 experts); each
// of the k rounds takes the wavefront maximum of the keys not yet taken by DPP moves, and the
// lowest expert that holds it from one ballot per slot.  The rounds are a serial chain of some
// 30 instructions each, so the routing is spread over the chip, one wavefront per SIMD, whenever
// one workgroup's wavefronts would have to take several tokens each.  (With 16 slots of 64-bit
// keys, exchanged over the LDS crossbar, and all tokens of a chunk of 1024 routes in one
// workgroup: 64 tokens of 256 experts, top 8, with the sort 38.5 us, now 8.1; 2048 tokens 78,
// now 11.5.)

constexpr int kRouterSlots = kSingleMaxExperts / 64;  // logits per lane: E <= 1024
constexpr int kRouterMaxTopk = 64;

__device__ __forceinline__ float key_value(uint32_t k) { return u2f((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); }

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = v + __shfl_xor(v, m, 64);
  return v;
}

// Route token t with the calling wavefront: ids / weights [t * topk + r] for r < topk;
// returns the lane's id (lane r < topk holds selection r, other lanes -1).
template <bool BF16, int NS>
__device__ __forceinline__ int32_t route_token(const void* __restrict__ logits, int64_t t, int E, int topk,
                                               bool renorm, int lane, int32_t* __restrict__ ids,
                                               float* __restrict__ weights) {
  uint32_t key[NS];   // of the logits not yet taken, else 0
  uint64_t left[NS];  // the lanes whose logit is not yet taken
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int i = lane + 64 * j;
    float x = 0.0f;
    if (i < E) x = BF16 ? bf16_to_f32(static_cast<const uint16_t*>(logits)[t * E + i])
                        : static_cast<const float*>(logits)[t * E + i];
    key[j] = i < E ? order_key(x) : 0u;
    left[j] = __ballot(i < E);
  }
  float my_x = 0.0f;
  int32_t my_id = -1;
  float top = 0.0f, part = 0.0f;
  for (int r = 0; r < topk; ++r) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < NS; ++j) best = key[j] > best ? key[j] : best;
    best = wave_max_u32(best);
    const float x = key_value(best);
    if (r == 0) {
      top = x;
      if (!renorm) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
          if (lane + 64 * j < E) part = part + mx_exp(key_value(key[j]) - top);
      }
    }
    int idx = 0;  // the lowest expert left with that key
#pragma unroll
    for (int j = NS - 1; j >= 0; --j) {
      const uint64_t m = __ballot(key[j] == best) & left[j];
      if (m) idx = 64 * j + __builtin_ctzll(m);
    }
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (j == idx >> 6) {
        left[j] &= ~(1ull << (idx & 63));
        if (lane == (idx & 63)) key[j] = 0u;
      }
    if (lane == r) {
      my_x = x;
      my_id = idx;
    }
  }
  const float e = lane < topk ? mx_exp(my_x - top) : 0.0f;
  const float denom = wave_sum(renorm ? e : part);
  if (lane < topk) {
    ids[t * topk + lane] = my_id;
    weights[t * topk + lane] = e / denom;
  }
  return my_id;
}

// Up to kRouterSingleTokens tokens, T * topk <= 1024 routes: routing and the token sort in one
// workgroup, a token per wavefront (256 experts, top 8: 1 / 16 tokens 6.3 / 7.8 us;
// 17 / 64 tokens 8.9 / 18.0, with router_kernel ahead of the sort 7.7 / 8.1).
constexpr int kRouterSingleTokens = 16;
template <bool BF16, int NS>
__global__ __launch_bounds__(kChunk) void router_single_kernel(const void* __restrict__ logits, int64_t T, int E,
                                                              int topk, int renorm, int32_t* __restrict__ ids,
                                                              float* __restrict__ weights,
                                                              int64_t* __restrict__ expert_offsets,
                                                              int32_t* __restrict__ sorted_routes,
                                                              int32_t* __restrict__ inverse) {
  __shared__ int32_t whist[(kChunk / 64) * kSingleMaxExperts];
  __shared__ int32_t tot[2][kSingleMaxExperts];
  __shared__ int32_t sids[kChunk];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  for (int64_t tok = w; tok < T; tok += kChunk / 64) {
    const int32_t id = route_token<BF16, NS>(logits, tok, E, topk, renorm != 0, lane, ids, weights);
    if (lane < topk) sids[tok * topk + lane] = id;
  }
  __syncthreads();
  const int64_t R = T * topk;
  single_chunk_sort(t < R ? sids[t] : -1, R, E, expert_offsets, sorted_routes, inverse, whist, tot);
}

// Routing only: ids and weights, sorted by mxl_moe_route afterwards.
template <bool BF16, int NS>
__global__ __launch_bounds__(256) void router_kernel(const void* __restrict__ logits, int64_t T, int E, int topk,
                                                     int renorm, int32_t* __restrict__ ids,
                                                     float* __restrict__ weights) {
  const int64_t tok = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tok < T) route_token<BF16, NS>(logits, tok, E, topk, renorm != 0, threadIdx.x & 63, ids, weights);
}

// One thread: 8 consecutive hidden columns of one token, its routes four at a time, whose places, then rows, load
// together (64 tokens of 8 routes, H = 2048: 4.0 us, 6.2 route after route; one token 2.9, 4.1; 777 of 6, H = 1920, 5.4, 6.6).
// ids (or null): the rows lie in the order of their routes, and count where the id is one of the E experts
// addend (bf16 [T, H] or null): added to the fp32 sum after the routes, before the one rounding
__global__ __launch_bounds__(256) void moe_reduce_kernel(const uint16_t* __restrict__ y,
                                                         const float* __restrict__ topk_weights,
                                                         const int32_t* __restrict__ inverse,
                                                         const int32_t* __restrict__ ids, int E, int64_t T, int topk,
                                                         int64_t H, const uint16_t* __restrict__ addend,
                                                         uint16_t* __restrict__ out) {
  const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t per_row = H / 8;
  if (id >= T * per_row) return;
  const int64_t t = id >> 32 ? id / per_row : (int64_t)((uint32_t)id / (uint32_t)per_row), h0 = (id - t * per_row) * 8;
  constexpr int B = 4;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
  for (int k0 = 0; k0 < topk; k0 += B) {
    int32_t p[B];
    float wk[B];
    uint4 raw[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int64_t at = t * topk + (k0 + b < topk ? k0 + b : topk - 1);
      p[b] = (ids ? ids : inverse)[at];
      if (ids) p[b] = p[b] >= 0 && p[b] < E ? (int32_t)at : -1;
      p[b] = k0 + b < topk ? p[b] : -1;
      wk[b] = topk_weights[at];
    }
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (p[b] >= 0) raw[b] = *reinterpret_cast<const uint4*>(y + (int64_t)p[b] * H + h0);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      if (p[b] < 0) continue;
      float v[8];
      bf16x8_to_f32(raw[b], v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float term = v[i] * wk[b];
        acc[i] = acc[i] + term;
      }
    }
  }
  if (addend) {
    float v[8];
    bf16x8_to_f32(*reinterpret_cast<const uint4*>(addend + t * H + h0), v);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = acc[i] + v[i];
  }
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (uint32_t)f32_to_bf16(acc[2 * i]) | ((uint32_t)f32_to_bf16(acc[2 * i + 1]) << 16);
  *reinterpret_cast<uint4*>(out + t * H + h0) = make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_moe_route_workspace_bytes(int64_t T, int64_t topk, int64_t E) {
  const int64_t R = T * topk;
  const int64_t C = (R + kChunk - 1) / kChunk;
  return C * E * (int64_t)sizeof(int32_t);
}

extern "C" int mxl_moe_route(const int32_t* topk_ids, int64_t T, int64_t topk, int64_t E, int32_t* sorted_routes,
                             int64_t* expert_offsets, int32_t* inverse, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  MXL_CHECK_ARG(T >= 0 && topk > 0 && E > 0, "mxl_moe_route: need T >= 0, topk > 0, E > 0");
  // route_scatter_kernel keeps one histogram per wavefront of a chunk in LDS:
  // (kChunk / 64) * E ints must fit gfx950's 160 KiB per workgroup
  MXL_CHECK_ARG(E <= kRouteMaxExperts, "mxl_moe_route: at most %d experts (E=%lld)", kRouteMaxExperts, (long long)E);
  const int64_t R = T * topk;
  const int64_t C = (R + kChunk - 1) / kChunk;
  MXL_CHECK_ARG(workspace_bytes >= mxl_moe_route_workspace_bytes(T, topk, E) && (C == 0 || workspace),
                "mxl_moe_route: workspace too small (%lld < %lld bytes)", (long long)workspace_bytes,
                (long long)mxl_moe_route_workspace_bytes(T, topk, E));
  hipStream_t s = (hipStream_t)stream;
  if (R <= kChunk && E <= kSingleMaxExperts) {  // one chunk: one launch
    route_single_kernel<<<1, kChunk, 0, s>>>(topk_ids, R, (int)E, expert_offsets, sorted_routes, inverse);
    MXL_CHECK_LAUNCH("mxl_moe_route(single)");
    return MXL_OK;
  }
  if (C > 1 && C <= sort_max_chunks(E) && E <= kSingleMaxExperts) {
    route_sort_kernel<<<dim3((unsigned)C), kChunk, (kChunk / 64 + 4) * E * sizeof(int32_t), s>>>(
        topk_ids, R, (int)C, (int)E, expert_offsets, sorted_routes, inverse);
    MXL_CHECK_LAUNCH("mxl_moe_route(sort)");
    return MXL_OK;
  }
  int32_t* counts = (int32_t*)workspace;
  if (C > 0) {
    route_hist_kernel<<<dim3((unsigned)C), kChunk, E * sizeof(int32_t), s>>>(topk_ids, R, (int)E, counts);
    MXL_CHECK_LAUNCH("mxl_moe_route(hist)");
    route_scan_kernel<<<dim3((unsigned)((E + kScanExperts - 1) / kScanExperts)), 1024, 0, s>>>(counts, C, (int)E);
    MXL_CHECK_LAUNCH("mxl_moe_route(scan)");
  }
  // (without routes one workgroup writes the offsets)
  route_scatter_kernel<<<dim3((unsigned)(C > 0 ? C : 1)), kChunk, (kChunk / 64) * E * sizeof(int32_t), s>>>(
      topk_ids, R, C, (int)E, counts, expert_offsets, sorted_routes, inverse);
  MXL_CHECK_LAUNCH("mxl_moe_route(scatter)");
  return MXL_OK;
}

// Router workspace: mxl_moe_route's.
extern "C" int64_t mxl_moe_router_workspace_bytes(int64_t T, int64_t topk, int64_t E) {
  return mxl_moe_route_workspace_bytes(T, topk, E);
}

// The routing launch: routing alone, or (expert_offsets set) with the sort.
template <bool BF16, int NS>
static void launch_router(const void* logits, int64_t T, int64_t E, int64_t topk, int renorm, float* weights,
                          int32_t* ids, int32_t* sorted_routes, int64_t* expert_offsets, int32_t* inverse,
                          hipStream_t s) {
  if (expert_offsets)
    router_single_kernel<BF16, NS><<<1, kChunk, 0, s>>>(logits, T, (int)E, (int)topk, renorm, ids, weights,
                                                        expert_offsets, sorted_routes, inverse);
  else
    router_kernel<BF16, NS><<<(unsigned)((T + 3) / 4), 256, 0, s>>>(logits, T, (int)E, (int)topk, renorm, ids,
                                                                    weights);
}
template <bool BF16, class... Args>
static void launch_router_slots(int64_t E, const void* logits, int64_t T, Args... args) {
  if (E <= 256) launch_router<BF16, 4>(logits, T, E, args...);
  else launch_router<BF16, kRouterSlots>(logits, T, E, args...);
}

extern "C" int mxl_moe_router(const void* logits, int logits_bf16, int64_t T, int64_t E, int64_t topk,
                              int renormalize, float* topk_weights, int32_t* topk_ids, int32_t* sorted_routes,
                              int64_t* expert_offsets, int32_t* inverse, void* workspace, int64_t workspace_bytes,
                              void* stream) {
  MXL_CHECK_ARG(T >= 0 && E > 0 && E <= kSingleMaxExperts && topk > 0 && topk <= kRouterMaxTopk && topk <= E,
                "mxl_moe_router: need 0 < topk <= min(E, %d) and 0 < E <= %d (E=%lld topk=%lld)", kRouterMaxTopk,
                kSingleMaxExperts, (long long)E, (long long)topk);
  MXL_CHECK_ARG(logits_bf16 == 0 || logits_bf16 == 1, "mxl_moe_router: logits are fp32 (0) or bf16 (1)");
  const int64_t R = T * topk;
  const int64_t C = (R + kChunk - 1) / kChunk;
  MXL_CHECK_ARG(workspace_bytes >= mxl_moe_router_workspace_bytes(T, topk, E) && (C == 0 || workspace),
                "mxl_moe_router: workspace too small (%lld < %lld bytes)", (long long)workspace_bytes,
                (long long)mxl_moe_router_workspace_bytes(T, topk, E));
  hipStream_t s = (hipStream_t)stream;
  const int renorm = renormalize ? 1 : 0;
  // few tokens (also T = 0: the offsets): routing and the sort in one launch
  const bool single = R <= kChunk && T <= kRouterSingleTokens;
  int64_t* const offsets = single ? expert_offsets : nullptr;
  if (logits_bf16)
    launch_router_slots<true>(E, logits, T, topk, renorm, topk_weights, topk_ids, sorted_routes, offsets, inverse, s);
  else
    launch_router_slots<false>(E, logits, T, topk, renorm, topk_weights, topk_ids, sorted_routes, offsets, inverse, s);
  MXL_CHECK_LAUNCH("mxl_moe_router(route)");
  if (single) return MXL_OK;
  return mxl_moe_route(topk_ids, T, topk, E, sorted_routes, expert_offsets, inverse, workspace, workspace_bytes,
                       stream);
}

static int moe_reduce_common(const char* who, const void* routed_output, const float* topk_weights,
                             const int32_t* inverse, const int32_t* ids, int64_t E, int64_t T, int64_t topk, int64_t H,
                             const void* addend, void* out, void* stream) {
  MXL_CHECK_ARG(T >= 0 && topk > 0 && H > 0 && H % 8 == 0, "%s: need H %% 8 == 0 (H=%lld)", who, (long long)H);
  MXL_CHECK_ARG(((uintptr_t)routed_output & 15) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)addend & 15) == 0,
                "%s: misaligned", who);
  if (T == 0) return MXL_OK;
  const int64_t n = T * (H / 8);
  // (few rows: single wavefronts, over more CUs)
  const int threads = n < 256 * (int64_t)cu_count() ? 64 : 256;
  moe_reduce_kernel<<<dim3((unsigned)((n + threads - 1) / threads)), threads, 0, (hipStream_t)stream>>>(
      (const uint16_t*)routed_output, topk_weights, inverse, ids, (int)E, T, (int)topk, H, (const uint16_t*)addend,
      (uint16_t*)out);
  MXL_CHECK_LAUNCH(who);
  return MXL_OK;
}

// mxl_moe_reduce of routed rows in the order of their routes (row t topk + k) instead of sorted by expert: those whose
// id is one of the E experts.
namespace mxl {
int moe_reduce_by_route(const char* who, const void* routed_output, const float* topk_weights, const int32_t* topk_ids,
                        int64_t T, int64_t topk, int64_t E, int64_t H, void* out, void* stream) {
  return moe_reduce_common(who, routed_output, topk_weights, nullptr, topk_ids, E, T, topk, H, nullptr, out, stream);
}
}  // namespace mxl

extern "C" int mxl_moe_reduce(const void* routed_output, const float* topk_weights, const int32_t* inverse, int64_t T,
                              int64_t topk, int64_t H, void* out, void* stream) {
  return moe_reduce_common("mxl_moe_reduce", routed_output, topk_weights, inverse, nullptr, 0, T, topk, H, nullptr, out,
                           stream);
}

extern "C" int mxl_moe_reduce_add(const void* routed_output, const float* topk_weights, const int32_t* inverse,
                                  int64_t T, int64_t topk, int64_t H, const void* addend, void* out, void* stream) {
  MXL_CHECK_ARG(addend != nullptr, "mxl_moe_reduce_add: no addend");
  return moe_reduce_common("mxl_moe_reduce_add", routed_output, topk_weights, inverse, nullptr, 0, T, topk, H, addend,
                           out, stream);
}
