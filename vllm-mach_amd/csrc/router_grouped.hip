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
// One wavefront per token, expert i at lane i % 64, slot i / 64 (the layout of the softmax router).
#include "mx_common.h"

namespace mxl {

constexpr int kGroupedMaxExperts = 1024, kGroupedMaxTopk = 64, kGroupedMaxGroups = 64;

struct GroupedRouting {
  const void* logits;   // fp32 or bf16 [T, E]
  const float* bias;    // fp32 [E] or null
  int64_t T;
  int E, topk, sigmoid, groups, keep, renorm;
  double factor;
  float* weights;
  int32_t* ids;
};

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = __builtin_fmax(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = v + __shfl_xor(v, m, 64);
  return v;
}

template <bool BF16, int NS>
__device__ __forceinline__ void route_grouped_token(const GroupedRouting& g, int64_t t, int lane) {
  const double none = -__builtin_inf();
  const int E = g.E, size = E / g.groups;
  double s[NS], c[NS];
  uint32_t left = 0;  // bit j: the lane's expert of slot j may still be chosen
  double top = none;
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int i = lane + 64 * j;
    s[j] = none;
    if (i < E) {
      s[j] = BF16 ? (double)bf16_to_f32(static_cast<const uint16_t*>(g.logits)[t * E + i])
                  : (double)static_cast<const float*>(g.logits)[t * E + i];
      left |= 1u << j;
    }
    top = __builtin_fmax(top, s[j]);
  }
  if (g.sigmoid) {
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j] = 1.0 / (1.0 + exp(-s[j]));
  } else {
    top = wave_max(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      s[j] = left >> j & 1 ? exp(s[j] - top) : 0.0;
      sum += s[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < NS; ++j) s[j] = s[j] / sum;
  }
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int i = lane + 64 * j;
    c[j] = i < E ? s[j] + (g.bias ? (double)g.bias[i] : 0.0) : none;
    if (c[j] != c[j]) c[j] = none;
  }
  // takes from `left` the lowest expert of its largest c, which goes to `best` (there is one left)
  auto take = [&](double& best) -> int {
    double m = none;
#pragma unroll
    for (int j = 0; j < NS; ++j) m = __builtin_fmax(m, left >> j & 1 ? c[j] : none);
    best = wave_max(m);
    int idx = 0;
#pragma unroll
    for (int j = NS - 1; j >= 0; --j) {
      const uint64_t at = __ballot((left >> j & 1) && c[j] == best);
      if (at) idx = 64 * j + __builtin_ctzll(at);
    }
    if (lane == (idx & 63)) left &= ~(1u << (idx >> 6));
    return idx;
  };
  if (g.keep < g.groups) {
    auto of_group = [&](int k) -> uint32_t {  // the lane's slots that hold experts of group k
      uint32_t in = 0;
#pragma unroll
      for (int j = 0; j < NS; ++j) in |= lane + 64 * j >= k * size && lane + 64 * j < (k + 1) * size ? 1u << j : 0u;
      return in;
    };
    double score = none;  // lane k: of group k
    for (int k = 0; k < g.groups; ++k) {
      left = of_group(k);
      double a, b = 0.0;
      take(a);
      if (g.bias && size > 1) take(b);
      if (lane == k) score = a + b;
    }
    if (score != score) score = none;  // (infinities of both signs)
    uint64_t open = g.groups < 64 ? (1ull << g.groups) - 1 : ~0ull;
    left = 0;
    for (int k = 0; k < g.keep; ++k) {
      const double best = wave_max((open >> lane & 1) ? score : none);
      const int grp = __builtin_ctzll(__ballot(score == best) & open);
      open &= ~(1ull << grp);
      left |= of_group(grp);
    }
  }
  double my = 0.0;
  int32_t my_id = -1;
  for (int k = 0; k < g.topk; ++k) {
    double best;
    const int idx = take(best);
    double v = 0.0;
#pragma unroll
    for (int j = 0; j < NS; ++j)
      if (j == idx >> 6) v = s[j];
    v = __shfl(v, idx & 63, 64);
    if (lane == k) {
      my = v;
      my_id = idx;
    }
  }
  const double sum = wave_sum(my);
  if (lane < g.topk) {
    g.ids[t * g.topk + lane] = my_id;
    g.weights[t * g.topk + lane] = (float)((g.renorm ? my / (sum + 1e-20) : my) * g.factor);
  }
}

template <bool BF16, int NS>
__global__ __launch_bounds__(256) void router_grouped_kernel(GroupedRouting g) {
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t < g.T) route_grouped_token<BF16, NS>(g, t, threadIdx.x & 63);
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
    const GroupedRouting g{logits, bias, T, (int)E, (int)topk, scoring, (int)groups, (int)topk_groups, renormalize != 0,
                           (double)factor, topk_weights, topk_ids};
    const dim3 grid((unsigned)((T + 3) / 4));
    if (logits_bf16) {
      if (E <= 256) router_grouped_kernel<true, 4><<<grid, 256, 0, s>>>(g);
      else router_grouped_kernel<true, 16><<<grid, 256, 0, s>>>(g);
    } else {
      if (E <= 256) router_grouped_kernel<false, 4><<<grid, 256, 0, s>>>(g);
      else router_grouped_kernel<false, 16><<<grid, 256, 0, s>>>(g);
    }
    MXL_CHECK_LAUNCH(who);
  }
  return mxl_moe_route(topk_ids, T, topk, E, sorted_routes, expert_offsets, inverse, workspace, workspace_bytes, stream);
}
