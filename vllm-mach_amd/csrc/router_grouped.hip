// Routing with group-limited, bias-corrected scores for gfx950: softmax or sigmoid scores of the router
// logits, the best groups of experts, the k best experts among them, their weights.
//
//   s = softmax(x) or 1 / (1 + exp(-x));  c = s + b (the choice score; b = 0 without a bias)
//   group score: the largest c of the group, or with a bias the sum of its two largest
//   the topk_groups best groups are kept, and of their experts the k with the largest c are chosen
//   weights: s (not c) of the chosen, divided by their sum + 1e-20 if renormalized, times a factor
//
// Ties go to the lower index.  Scores, biases and sums are held in binary64: which experts are chosen is a
// whole number, and two sigmoid scores a rounding of exp apart must not decide it.  NaN choice scores rank
// below every other.
//
// One wavefront per token.  Each group has LPG lanes (a power of two, the most that fit), its experts dealt over
// them (expert SUB + LPG j of the group in slot j), so that a group's two largest c come from log2(LPG) exchanges of
// all groups at once, and a lane holds few experts.  A choice round takes the wavefront maximum of the lanes' best
// keys -- c as a 64-bit integer in value order -- by their upper halves, one DPP maximum each; where several lanes
// share it (c closer than 2^-20 of its value) the lower halves and then the index decide.  The chosen experts' lanes then
// recompute their s from the logits, so that only the keys stay in registers.
#include "moe_sort.h"

namespace mxl {

constexpr int kGroupedMaxExperts = 1024, kGroupedMaxTopk = 64, kGroupedMaxGroups = 64;

struct GroupedRouting {
  const void* logits;   // fp32 or bf16 [T, E]
  const float* bias;    // fp32 [E] or null
  int64_t T;
  int E, topk, sigmoid, groups, size, lpg_log, keep, renorm;  // size: experts of a group; 2^lpg_log lanes each
  double factor;
  float* weights;
  int32_t* ids;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = v + __shfl_xor(v, m, 64);
  return v;
}

// The value of the lane that DPP control CTRL names.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double readlane_f64(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Binary64 as a key in value order (-0 as +0), never 0; NaNs as -infinity.
__device__ __forceinline__ uint64_t order_key(double c) {
  const uint64_t u = __builtin_bit_cast(uint64_t, c != c ? -__builtin_inf() : c + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// Token t by the calling wavefront; returns the lane's id (lane k < topk holds choice k, other lanes -1).
template <bool BF16, int NS>
__device__ __forceinline__ int32_t route_grouped_token(const GroupedRouting& g, int64_t t, int lane) {
  const int lpg = 1 << g.lpg_log, grp = lane >> g.lpg_log, sub = lane & (lpg - 1), first = grp * g.size;
  auto logit = [&](int i) -> float {
    return BF16 ? bf16_to_f32(static_cast<const uint16_t*>(g.logits)[t * g.E + i])
                : static_cast<const float*>(g.logits)[t * g.E + i];
  };
  float x[NS];
  uint32_t held = 0;  // slots that hold an expert
  uint32_t top_key = 0;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int i = sub + (j << g.lpg_log);
    x[j] = 0.0f;
    if (grp < g.groups && i < g.size) {
      x[j] = logit(first + i);
      held |= 1u << j;
      const uint32_t k = order_key(x[j]);
      top_key = k > top_key ? k : top_key;
    }
  }
  double top = 0.0, sum = 1.0;
  if (!g.sigmoid) {
    const uint32_t k = wave_max_u32(top_key);
    top = u2f((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
  }
  auto score = [&](float v) -> double {  // (softmax: before the division by `sum`)
    const double e = exp(g.sigmoid ? -(double)v : (double)v - top);
    return g.sigmoid ? 1.0 / (1.0 + e) : e;
  };
  double s[NS];
#pragma unroll
  for (int j = 0; j < NS; ++j) s[j] = score(x[j]);
  if (!g.sigmoid) {
    double part = 0.0;
#pragma unroll
    for (int j = 0; j < NS; ++j) part += held >> j & 1 ? s[j] : 0.0;
    sum = wave_sum(part);
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j] = s[j] / sum;
  }
  uint64_t key[NS];  // of the experts that may still be chosen, else 0
  double a1 = -__builtin_inf(), a2 = a1;  // the lane's two largest c
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    double c = s[j];
    key[j] = 0;
    if (held >> j & 1) {
      if (g.bias) c += (double)g.bias[first + sub + (j << g.lpg_log)];
      key[j] = order_key(c);
      c = c != c ? -__builtin_inf() : c;
      a2 = __builtin_fmax(a2, __builtin_fmin(a1, c));
      a1 = __builtin_fmax(a1, c);
    }
  }
  if (g.keep < g.groups) {
    // the group's two largest: merged with the lanes 1, 2, 4, ... apart
    auto merge = [&](double b1, double b2) {
      a2 = __builtin_fmax(__builtin_fmin(a1, b1), __builtin_fmax(a2, b2));
      a1 = __builtin_fmax(a1, b1);
    };
    if (g.lpg_log > 0) merge(dpp_f64<0xB1>(a1), dpp_f64<0xB1>(a2));    // quad_perm 1 0 3 2
    if (g.lpg_log > 1) merge(dpp_f64<0x4E>(a1), dpp_f64<0x4E>(a2));    // quad_perm 2 3 0 1
    if (g.lpg_log > 2) merge(dpp_f64<0x141>(a1), dpp_f64<0x141>(a2));  // row_half_mirror
    if (g.lpg_log > 3) merge(dpp_f64<0x140>(a1), dpp_f64<0x140>(a2));  // row_mirror
    if (g.lpg_log > 4) merge(__shfl_xor(a1, 16, 64), __shfl_xor(a2, 16, 64));
    double mine = g.bias && g.size > 1 ? a1 + a2 : a1;
    mine = mine != mine ? -__builtin_inf() : mine;  // (infinities of both signs)
    int ahead = 0;  // groups before this one
    for (int h = 0; h < g.groups; ++h) {
      const double other = readlane_f64(mine, h << g.lpg_log);
      ahead += other > mine || (other == mine && h < grp) ? 1 : 0;
    }
    if (ahead >= g.keep) {
#pragma unroll
      for (int j = 0; j < NS; ++j) key[j] = 0;
    }
  }
  uint64_t best;  // the lane's largest key and its slot, the lower of equals
  int at;
  auto refresh = [&] {
    best = key[NS - 1];
    at = NS - 1;
#pragma unroll
    for (int j = NS - 2; j >= 0; --j)
      if (key[j] >= best) {
        best = key[j];
        at = j;
      }
  };
  refresh();
  int32_t my_id = -1;
  for (int k = 0; k < g.topk; ++k) {
    const uint32_t hi = (uint32_t)(best >> 32), top_hi = wave_max_u32(hi);
    uint64_t who = __ballot(hi == top_hi);
    const int idx = first + sub + (at << g.lpg_log);
    if (who & (who - 1)) {
      const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = wave_max_u32(lo);
      who = __ballot(hi == top_hi && lo == top_lo);
      if (who & (who - 1)) {  // equal c: the lowest index
        const uint32_t inv = (who >> lane & 1) ? ~(uint32_t)idx : 0u;
        who = __ballot(inv == wave_max_u32(inv));
      }
    }
    const int w = __builtin_ctzll(who), chosen = __builtin_amdgcn_readlane(idx, w);
    if (lane == k) my_id = chosen;
    if (lane == w) {
#pragma unroll
      for (int j = 0; j < NS; ++j) key[j] = j == at ? 0ull : key[j];
      refresh();
    }
  }
  double v = 0.0;
  if (lane < g.topk) v = score(logit(my_id)) / sum;
  const double total = wave_sum(v);
  if (lane < g.topk) {
    g.ids[t * g.topk + lane] = my_id;
    g.weights[t * g.topk + lane] = (float)((g.renorm ? v / (total + 1e-20) : v) * g.factor);
  }
  return my_id;
}

template <bool BF16, int NS>
__global__ __launch_bounds__(256) void router_grouped_kernel(GroupedRouting g) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t < g.T) route_grouped_token<BF16, NS>(g, t, threadIdx.x & 63);
}

// Up to 16 tokens: routing and the token sort in one workgroup, a token per wavefront.
constexpr int kGroupedSingleTokens = kChunk / 64;
template <bool BF16, int NS>
__global__ __launch_bounds__(kChunk) void router_grouped_single_kernel(GroupedRouting g, int64_t* __restrict__ offsets,
                                                                       int32_t* __restrict__ sorted_routes,
                                                                       int32_t* __restrict__ inverse) {
  __shared__ int32_t whist[(kChunk / 64) * kSingleMaxExperts];
  __shared__ int32_t tot[2][kSingleMaxExperts];
  __shared__ int32_t sids[kChunk];
  const int t = threadIdx.x, w = t >> 6, lane = t & 63;
  if (w < g.T) {
    const int32_t id = route_grouped_token<BF16, NS>(g, w, lane);
    if (lane < g.topk) sids[w * g.topk + lane] = id;
  }
  __syncthreads();
  const int64_t R = g.T * g.topk;
  single_chunk_sort(t < R ? sids[t] : -1, R, g.E, offsets, sorted_routes, inverse, whist, tot);
}

// The routing launch: routing alone, or (offsets set) with the sort.
template <bool BF16, int NS>
static void launch_grouped(const GroupedRouting& g, int64_t* offsets, int32_t* sorted_routes, int32_t* inverse,
                           hipStream_t s) {
  if (offsets) router_grouped_single_kernel<BF16, NS><<<1, kChunk, 0, s>>>(g, offsets, sorted_routes, inverse);
  else router_grouped_kernel<BF16, NS><<<dim3((unsigned)((g.T + 3) / 4)), 256, 0, s>>>(g);
}
template <bool BF16>
static void launch_grouped_slots(const GroupedRouting& g, int64_t* offsets, int32_t* sorted_routes, int32_t* inverse,
                                 hipStream_t s) {
  const int slots = (g.size + (1 << g.lpg_log) - 1) >> g.lpg_log;
  if (slots <= 2) launch_grouped<BF16, 2>(g, offsets, sorted_routes, inverse, s);
  else if (slots <= 4) launch_grouped<BF16, 4>(g, offsets, sorted_routes, inverse, s);
  else if (slots <= 8) launch_grouped<BF16, 8>(g, offsets, sorted_routes, inverse, s);
  else launch_grouped<BF16, 32>(g, offsets, sorted_routes, inverse, s);
}

}  // namespace mxl

using namespace mxl;

extern "C" int64_t mxl_moe_route_workspace_bytes(int64_t T, int64_t topk, int64_t E);
extern "C" int mxl_moe_route(const int32_t* topk_ids, int64_t T, int64_t topk, int64_t E, int32_t* sorted_routes,
                             int64_t* expert_offsets, int32_t* inverse, void* workspace, int64_t workspace_bytes,
                             void* stream);

extern "C" int mxl_moe_router_grouped(const void* logits, int logits_bf16, const float* bias, int64_t T, int64_t E,
                                      int64_t topk, int scoring, int64_t groups, int64_t topk_groups, int renormalize,
                                      float factor, float* topk_weights, int32_t* topk_ids, int32_t* sorted_routes,
                                      int64_t* expert_offsets, int32_t* inverse, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_moe_router_grouped";
  MXL_CHECK_ARG(T >= 0 && E > 0 && E <= kGroupedMaxExperts, "%s: need T >= 0 and 0 < E <= %d (T=%lld E=%lld)", who,
                kGroupedMaxExperts, (long long)T, (long long)E);
  MXL_CHECK_ARG(groups > 0 && groups <= kGroupedMaxGroups && E % groups == 0 && topk_groups > 0 && topk_groups <= groups,
                "%s: need 0 < topk_groups <= groups <= %d and E %% groups == 0 (E=%lld groups=%lld topk_groups=%lld)", who,
                kGroupedMaxGroups, (long long)E, (long long)groups, (long long)topk_groups);
  MXL_CHECK_ARG(topk > 0 && topk <= kGroupedMaxTopk && topk <= topk_groups * (E / groups),
                "%s: need 0 < topk <= min(%d, experts of the kept groups) (topk=%lld)", who, kGroupedMaxTopk,
                (long long)topk);
  MXL_CHECK_ARG(logits_bf16 == 0 || logits_bf16 == 1, "%s: logits are fp32 (0) or bf16 (1)", who);
  MXL_CHECK_ARG(scoring == 0 || scoring == 1, "%s: scoring is softmax (0) or sigmoid (1), got %d", who, scoring);
  MXL_CHECK_ARG(factor - factor == 0.0f, "%s: the weights' factor must be finite", who);
  MXL_CHECK_ARG(T * topk <= 0x7FFFFFFF, "%s: too many routes (T=%lld topk=%lld)", who, (long long)T, (long long)topk);
  MXL_CHECK_ARG(workspace_bytes >= mxl_moe_route_workspace_bytes(T, topk, E) && (T == 0 || workspace),
                "%s: workspace too small (%lld < %lld bytes)", who, (long long)workspace_bytes,
                (long long)mxl_moe_route_workspace_bytes(T, topk, E));
  hipStream_t s = (hipStream_t)stream;
  if (T > 0) {
    GroupedRouting g{logits, bias, T, (int)E, (int)topk, scoring, (int)groups, (int)(E / groups), 0, (int)topk_groups,
                     renormalize != 0, (double)factor, topk_weights, topk_ids};
    while ((2 << g.lpg_log) * groups <= 64) ++g.lpg_log;
    const bool single = T <= kGroupedSingleTokens && T * topk <= kChunk;
    if (logits_bf16) launch_grouped_slots<true>(g, single ? expert_offsets : nullptr, sorted_routes, inverse, s);
    else launch_grouped_slots<false>(g, single ? expert_offsets : nullptr, sorted_routes, inverse, s);
    MXL_CHECK_LAUNCH(who);
    if (single) return MXL_OK;
  }
  return mxl_moe_route(topk_ids, T, topk, E, sorted_routes, expert_offsets, inverse, workspace, workspace_bytes, stream);
}
