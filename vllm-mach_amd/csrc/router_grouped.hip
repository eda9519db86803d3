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
// LPT lanes per token: 16, four tokens to a wavefront, or 64 (few tokens; more than 16 choices, groups or experts to a
// lane).
// Each group has 2^lpg_log of them (the most that fit), each lane successive experts of its group, so that a group's
// two largest c come from lpg_log exchanges of all groups at once and the lowest lane is the lowest index.
//
// Its instructions and what they wait for bound it (256 logits are 1 KiB and a thousand operations; 16384 tokens read at
// 0.9 TB/s, with the VALU busy a third of the time, 1.6 wavefronts a SIMD and 41 % of theirs spent in waits).  Scores of
// every expert in binary64 are most of the instructions, so the choice is first made in binary32 (choose_fast):
// - the values are 32-bit keys in value order, their lowest log2(NS) bits the slot.  Each lane sorts its own once, by
//   a network; a round of the choice then is one DPP maximum of the lanes' first keys, and the winner moves up by one.
// - without a bias the values are the logits themselves.  Logits 2^-20 apart have binary64 scores apart, where none is
//   so large that its sigmoid is 1 or so small that its score is subnormal.  Equal ones have equal scores (and equal
//   keys, if the logits' lowest bits are all 0, as those of bf16 are).
// - with a bias they are c in binary32.  With u = 2^-24: exp2's argument is off by 2.2 u of itself, which moves sigmoid
//   by 0.5 u at most (s (1 - s) |x| < 0.23) and a softmax term by 0.81 u (e^-d d < 0.37); the hardware exp2 and
//   reciprocal are off by 2 u each, so sigmoid is within 4 u.  Softmax's sum takes NS + 5 roundings, so s is within
//   (NS + 14) u < 46 u of its largest, 1 / sum.  The bias adds u |c|, the key's cut 2 (NS - 1) u |c|.
// Where every call -- the groups', each expert's against the next -- stands apart by more than the errors of both
// sides, the choice is the true one; for a token with a closer call (or an infinity or NaN, a group's sum among them),
// one in some hundred, the whole wavefront makes it in binary64 (choose_exact: 64-bit keys, compared by their halves).
// The weights are of binary64 scores of the k chosen, one a lane.
//
// 16384 tokens of 256 experts, 8 of 128 in 4 of 8 groups: 19 us (31.3 with every score in binary64 and a token per
// wavefront, 27 with the binary32 choice alone, 26 with four tokens to a wavefront that all made a close one's choice).
#include "moe_sort.h"

namespace mxl {

constexpr int kGroupedMaxExperts = 1024, kGroupedMaxTopk = 64, kGroupedMaxGroups = 64;

struct GroupedRouting {
  const void* logits;   // fp32 or bf16 [T, E]
  const float* bias;    // fp32 [E] or null
  int64_t T;
  int E, topk, sigmoid, groups, size, keep, renorm;  // size: experts of a group
  int quads;  // whether four experts from a multiple of 4 are a group's and aligned
  // 2^lpg_log lanes of a group, `per` experts (fours) a lane: of the kernel's lanes per token, and of 64
  struct Deal {
    int lpg_log, per;
  } deal, deal64;
  double factor;
  float* weights;
  int32_t* ids;
};

// The value of the lane that DPP control CTRL names.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;  // quad_perm 1032, 2301; row mirrors
__device__ __forceinline__ uint32_t max_u32(uint32_t a, uint32_t b) { return a > b ? a : b; }

// Over the LPT lanes of a token, in every lane: the maximum (of no NaNs), the sum.
template <int LPT>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  v = max_u32(v, dpp_u32<kXor1>(v));
  v = max_u32(v, dpp_u32<kXor2>(v));
  v = max_u32(v, dpp_u32<kHalfMirror>(v));
  v = max_u32(v, dpp_u32<kMirror>(v));
#pragma unroll
  for (int m = 16; m < LPT; m <<= 1) v = max_u32(v, (uint32_t)__shfl_xor((int)v, m, 64));
  return v;
}
template <int LPT>
__device__ __forceinline__ float lanes_max(float v) {
  v = __builtin_fmaxf(v, u2f(dpp_u32<kXor1>(f2u(v))));
  v = __builtin_fmaxf(v, u2f(dpp_u32<kXor2>(f2u(v))));
  v = __builtin_fmaxf(v, u2f(dpp_u32<kHalfMirror>(f2u(v))));
  v = __builtin_fmaxf(v, u2f(dpp_u32<kMirror>(f2u(v))));
#pragma unroll
  for (int m = 16; m < LPT; m <<= 1) v = __builtin_fmaxf(v, __shfl_xor(v, m, 64));
  return v;
}
template <int LPT, typename T>
__device__ __forceinline__ T lanes_sum(T v) {
#pragma unroll
  for (int m = LPT / 2; m >= 1; m >>= 1) v = v + __shfl_xor(v, m, 64);
  return v;
}

// Binary64 as a key in value order (-0 as +0), never 0; NaNs as -infinity.
__device__ __forceinline__ uint64_t order_key(double c) {
  const uint64_t u = __builtin_bit_cast(uint64_t, c != c ? -__builtin_inf() : c + 0.0);
  return u >> 63 ? ~u : u | 1ull << 63;
}

// Keys in descending order, by Batcher's odd-even merges.
template <int NS>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[NS]) {
#pragma unroll
  for (int p = 1; p < NS; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int i = 0; i < NS - k; ++i)
        if (i >= k % p && (i - k % p) % (2 * k) < k && i / (2 * p) == (i + k) / (2 * p)) {
          const uint32_t a = key[i], b = key[i + k];
          key[i] = a > b ? a : b;
          key[i + k] = a > b ? b : a;
        }
}

// A lane's share of its token: slot j < count is expert first + j, of logit x[j].
template <bool BF16, int LPT, int NS>
struct GroupedToken {
  const GroupedRouting& g;
  const GroupedRouting::Deal deal;
  int64_t t;
  int lane, base, at, grp, first, count;  // lane of the wavefront, the token's first, place from there, its group
  float x[NS];

  __device__ __forceinline__ float logit(int i) const {
    return BF16 ? bf16_to_f32(static_cast<const uint16_t*>(g.logits)[t * g.E + i])
                : static_cast<const float*>(g.logits)[t * g.E + i];
  }

  __device__ __forceinline__ GroupedToken(const GroupedRouting& g_, const GroupedRouting::Deal& deal_, int64_t t_, int lane_)
      : g(g_), deal(deal_), t(t_), lane(lane_) {
    at = lane & (LPT - 1);
    base = lane - at;
    grp = at >> deal.lpg_log;
    const int from = (at & ((1 << deal.lpg_log) - 1)) * deal.per;  // of the group's experts
    first = grp * g.size + from;
    const int left = grp < g.groups ? g.size - from : 0;
    count = left < deal.per ? (left < 0 ? 0 : left) : deal.per;
#pragma unroll
    for (int j = 0; j < NS; ++j) x[j] = 0.0f;
    if (g.quads) {
#pragma unroll
      for (int j = 0; j < NS; j += 4)
        if (j < count) {
          const int64_t o = t * g.E + first + j;
          if (BF16) {
            const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g.logits) + o);
            x[j] = u2f(v.x << 16), x[j + 1] = u2f(v.x & 0xffff0000u);
            x[j + 2] = u2f(v.y << 16), x[j + 3] = u2f(v.y & 0xffff0000u);
          } else {
            const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(g.logits) + o);
            x[j] = v.x, x[j + 1] = v.y, x[j + 2] = v.z, x[j + 3] = v.w;
          }
        }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (j < count) x[j] = logit(first + j);
    }
  }
  // the slots' biases
  __device__ __forceinline__ void biases(float (&b)[NS]) const {
#pragma unroll
    for (int j = 0; j < NS; ++j) b[j] = 0.0f;
    if (g.quads) {
#pragma unroll
      for (int j = 0; j < NS; j += 4)
        if (j < count) {
          const float4 v = *reinterpret_cast<const float4*>(g.bias + first + j);
          b[j] = v.x, b[j + 1] = v.y, b[j + 2] = v.z, b[j + 3] = v.w;
        }
    } else {
#pragma unroll
      for (int j = 0; j < NS; ++j)
        if (j < count) b[j] = g.bias[first + j];
    }
  }
  // the largest logit (softmax), but for NaNs
  __device__ __forceinline__ float largest() const {
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < NS; ++j) top = __builtin_fmaxf(top, j < count ? x[j] : top);
    return lanes_max<LPT>(top);
  }
  // s of a logit, softmax's before the division by the sum
  __device__ __forceinline__ double score(float v, double top) const {
    const double e = exp(g.sigmoid ? -(double)v : (double)v - top);
    return g.sigmoid ? 1.0 / (1.0 + e) : e;
  }
  __device__ __forceinline__ double softmax_sum(double top) const {
    double part = 0.0;
#pragma unroll
    for (int j = 0; j < NS; ++j) part += j < count ? score(x[j], top) : 0.0;
    return lanes_sum<LPT>(part);
  }
  // the lowest of the token's lanes for which `is` holds; it does for one
  __device__ __forceinline__ int lowest(bool is) const {
    const uint64_t who = __ballot(is) >> base;
    return base + (LPT < 64 ? __builtin_ctz((uint32_t)who) : __builtin_ctzll(who));
  }

  // The choices in binary64: lane k < topk of the token its expert, other lanes -1.
  __device__ __forceinline__ int32_t choose_exact(double top, double sum) const {
    uint64_t key[NS];  // of the experts that may still be chosen, else 0
    double a1 = -__builtin_inf(), a2 = a1;  // the lane's two largest c
#pragma unroll
    for (int j = 0; j < NS; ++j) {
      key[j] = 0;
      if (j < count) {
        double c = score(x[j], top) / sum;
        if (g.bias) c += (double)g.bias[first + j];
        key[j] = order_key(c);
        c = c != c ? -__builtin_inf() : c;
        a2 = __builtin_fmax(a2, __builtin_fmin(a1, c));
        a1 = __builtin_fmax(a1, c);
      }
    }
    if (g.keep < g.groups) {
      // the group's two largest: merged with the lanes 1, 2, 4, ... apart
      for (int m = 1; m < 1 << deal.lpg_log; m <<= 1) {
        const double b1 = __shfl_xor(a1, m, 64), b2 = __shfl_xor(a2, m, 64);
        a2 = __builtin_fmax(__builtin_fmin(a1, b1), __builtin_fmax(a2, b2));
        a1 = __builtin_fmax(a1, b1);
      }
      double mine = g.bias && g.size > 1 ? a1 + a2 : a1;
      mine = mine != mine ? -__builtin_inf() : mine;  // (infinities of both signs)
      int ahead = 0;  // groups before this one
      for (int h = 0; h < g.groups; ++h) {
        const double other = __shfl(mine, base + (h << deal.lpg_log), 64);
        ahead += other > mine || (other == mine && h < grp) ? 1 : 0;
      }
      if (ahead >= g.keep) {
#pragma unroll
        for (int j = 0; j < NS; ++j) key[j] = 0;
      }
    }
    int32_t my_id = -1;
    for (int k = 0; k < g.topk; ++k) {
      uint64_t best = 0;
#pragma unroll
      for (int j = 0; j < NS; ++j) best = key[j] > best ? key[j] : best;
      const uint32_t hi = (uint32_t)(best >> 32), top_hi = lanes_max<LPT>(hi);
      const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = lanes_max<LPT>(lo);
      const int w = lowest(hi == top_hi && lo == top_lo);
      int slot = 0;  // the lane's lowest of its best; the winner's is taken out
#pragma unroll
      for (int j = NS - 1; j >= 0; --j) slot = key[j] == best ? j : slot;
#pragma unroll
      for (int j = 0; j < NS; ++j) key[j] = lane == w && slot == j ? 0ull : key[j];
      const int chosen = __shfl(first + slot, w, 64);
      if (at == k) my_id = chosen;
    }
    return my_id;
  }

  // The choices in binary32, in choice[0 .. topk); false (in every lane of the token) where one is too close to call.
  __device__ __forceinline__ bool choose_fast(float top, volatile int32_t* choice) const {
    constexpr uint32_t kSlot = NS - 1;
    constexpr float kPart = 0x1p-23f * NS;
    uint32_t key[NS];
    float unit = 0x1p-20f, nan = 0.0f;  // calls are apart by unit + kPart (|c| + |c'|)
    bool close = false, same = false;   // same: keys are equal only of equal logits
    auto set = [&](int j, float c) {
      key[j] = j < count ? (order_key(c) & ~kSlot) | (kSlot - j) : 0u;
    };
    if (!g.bias) {
      float low = g.sigmoid ? 0.0f : top, high = low;
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        low = __builtin_fminf(low, j < count ? x[j] : low);
        high = __builtin_fmaxf(high, x[j]);
        nan = __builtin_fmaf(0.0f, x[j], nan);
        bits |= f2u(x[j]);
        set(j, x[j]);
      }
      close = g.sigmoid ? !(low >= -600.0f && high <= 16.0f) : !(low - top >= -600.0f);
      same = (__ballot((bits & kSlot) != 0) >> base & lanes()) == 0;
    } else {
      float b[NS], c[NS];
      biases(b);
#pragma unroll
      for (int j = 0; j < NS; ++j) nan = __builtin_fmaf(0.0f, x[j], __builtin_fmaf(0.0f, b[j], nan));
      if (g.sigmoid) {
#pragma unroll
        for (int j = 0; j < NS; ++j)
          c[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[j] * -1.44269504f)) + b[j];
      } else {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NS; ++j) {
          c[j] = __builtin_amdgcn_exp2f((x[j] - top) * 1.44269504f);
          sum += j < count ? c[j] : 0.0f;
        }
        const float inv = __builtin_amdgcn_rcpf(lanes_sum<LPT>(sum));
        unit = 0x1p-17f * inv;
#pragma unroll
        for (int j = 0; j < NS; ++j) c[j] = c[j] * inv + b[j];
      }
#pragma unroll
      for (int j = 0; j < NS; ++j) set(j, c[j]);
    }
    close |= !(nan == 0.0f);
    sort_keys(key);
    auto value = [](uint32_t k) { return u2f((k & 0x80000000u) ? k ^ 0x80000000u : ~k); };
    auto apart = [&](float d, float mag) {
      d = __builtin_fabsf(d);
      return d > unit + kPart * mag || (same && d == 0.0f);
    };
    if (g.keep < g.groups) {
      float a1 = key[0] ? value(key[0] & ~kSlot) : -__builtin_inff(), a2 = key[1] ? value(key[1] & ~kSlot) : -__builtin_inff();
      auto merge = [&](float b1, float b2) {
        a2 = __builtin_fmaxf(__builtin_fminf(a1, b1), __builtin_fmaxf(a2, b2));
        a1 = __builtin_fmaxf(a1, b1);
      };
      if (deal.lpg_log > 0) merge(u2f(dpp_u32<kXor1>(f2u(a1))), u2f(dpp_u32<kXor1>(f2u(a2))));
      if (deal.lpg_log > 1) merge(u2f(dpp_u32<kXor2>(f2u(a1))), u2f(dpp_u32<kXor2>(f2u(a2))));
      if (deal.lpg_log > 2) merge(u2f(dpp_u32<kHalfMirror>(f2u(a1))), u2f(dpp_u32<kHalfMirror>(f2u(a2))));
      if (deal.lpg_log > 3) merge(u2f(dpp_u32<kMirror>(f2u(a1))), u2f(dpp_u32<kMirror>(f2u(a2))));
      if (LPT > 16 && deal.lpg_log > 4) merge(__shfl_xor(a1, 16, 64), __shfl_xor(a2, 16, 64));
      const bool two = g.bias && g.size > 1;
      const float mine = two ? a1 + a2 : a1;
      close |= grp < g.groups && __builtin_fabsf(mine) == __builtin_inff();  // (past the largest binary32: not in order)
      // (sums of two have twice the error, on both sides; the group of the larger magnitudes finds a close call)
      const float scale = two ? 0.25f : 1.0f, mag = 2 * (two ? __builtin_fabsf(a1) + __builtin_fabsf(a2) : __builtin_fabsf(a1));
      int ahead = 0;
      bool kept = false;
      uint64_t which = 0;
      // the groups' scores, eight at a time: the groups before this one; then whether a kept one is near one that is not
      auto each = [&](auto&& f) {
        for (int h0 = 0; h0 < g.groups; h0 += 8) {
          float other[8];
#pragma unroll
          for (int h = 0; h < 8; ++h) other[h] = __shfl(mine, base + ((h0 + h) << deal.lpg_log), 64);
#pragma unroll
          for (int h = 0; h < 8; ++h)
            if (h0 + h < g.groups) f(h0 + h, other[h] - mine);
        }
      };
      each([&](int h, float d) { ahead += d > 0.0f || (d == 0.0f && h < grp) ? 1 : 0; });
      kept = ahead < g.keep;
      which = __ballot(kept) >> base;
      each([&](int h, float d) {
        close |= grp < g.groups && kept != (bool)(which >> (h << deal.lpg_log) & 1) && !apart(scale * d, mag);
      });
      if (!kept) {
#pragma unroll
        for (int j = 0; j < NS; ++j) key[j] = 0;
      }
    }
    // (a few rounds more where the last choice ties with the next: what follows them must be apart as well)
    constexpr int kMore = 4;
    float last = 0.0f;
    bool open = true;  // the token has calls left
    for (int k = 0;; ++k) {
      const uint32_t mine = key[0] & ~kSlot, most = lanes_max<LPT>(mine);
      const float v = value(most);
      close |= open && k > 0 && most != 0 && !apart(last - v, __builtin_fabsf(last) + __builtin_fabsf(v));
      if (k >= g.topk) {
        open = open && most != 0 && v == last;
        if (!__ballot(open)) break;
        if (k == g.topk + kMore) {
          close |= open;
          break;
        }
      }
      last = v;
      if (lane == lowest(mine == most)) {
        if (k < g.topk) choice[k] = first + (int)(kSlot - (key[0] & kSlot));
#pragma unroll
        for (int j = 0; j < NS - 1; ++j) key[j] = key[j + 1];
        key[NS - 1] = 0;
      }
    }
    return (__ballot(close) >> base & lanes()) == 0;
  }
  __device__ static constexpr uint64_t lanes() { return LPT == 64 ? ~0ull : (1ull << (LPT & 63)) - 1; }
};

// The wavefront's tokens; returns the lane's id (lane k < topk of a token holds choice k, other lanes -1).  Lanes of a
// token past the last route that one again and write nothing.  choices: the wavefront's 64 words of LDS.
template <bool BF16, int LPT, int NS>
__device__ __forceinline__ int32_t route_grouped_tokens(const GroupedRouting& g, int64_t t, int lane, int32_t* choices) {
  const bool real = t < g.T;
  t = real ? t : g.T - 1;
  const GroupedToken<BF16, LPT, NS> tok(g, g.deal, t, lane);
  const float top = g.sigmoid ? 0.0f : tok.largest();
  const bool fast = tok.choose_fast(top, choices + tok.base);
  for (uint64_t left = __ballot(!fast); left;) {
    const int first = __builtin_ctzll(left) & ~(LPT - 1);
    const int64_t close = __shfl(t, first, 64);
    const GroupedToken<BF16, 64, LPT == 16 ? 4 : NS> whole(g, g.deal64, close, lane);
    const float most = g.sigmoid ? 0.0f : whole.largest();
    const int32_t id = whole.choose_exact(most, g.sigmoid ? 1.0 : whole.softmax_sum(most));
    if (lane < g.topk) choices[first + lane] = id;
    left &= ~(tok.lanes() << first);
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one lane's choice is another's to read)
  const int32_t my_id = tok.at < g.topk ? choices[lane] : -1;
  const double sum = g.sigmoid ? 1.0 : tok.softmax_sum(top);
  double v = 0.0;
  if (tok.at < g.topk) v = tok.score(tok.logit(my_id), top) / sum;
  const double total = lanes_sum<LPT>(v);
  if (real && tok.at < g.topk) {
    g.ids[t * g.topk + tok.at] = my_id;
    g.weights[t * g.topk + tok.at] = (float)((g.renorm ? v / (total + 1e-20) : v) * g.factor);
  }
  return my_id;
}

template <bool BF16, int LPT, int NS>
__global__ __launch_bounds__(256) void router_grouped_kernel(GroupedRouting g) {
  __shared__ int32_t choices[256];
  route_grouped_tokens<BF16, LPT, NS>(g, (int64_t)blockIdx.x * (256 / LPT) + threadIdx.x / LPT, threadIdx.x & 63,
                                      choices + (threadIdx.x & ~63));
}

// Up to 16 tokens: routing and the token sort in one workgroup.
constexpr int kGroupedSingleTokens = kChunk / 64;
template <bool BF16, int LPT, int NS>
__global__ __launch_bounds__(kChunk) void router_grouped_single_kernel(GroupedRouting g, int64_t* __restrict__ offsets,
                                                                       int32_t* __restrict__ sorted_routes,
                                                                       int32_t* __restrict__ inverse) {
  __shared__ int32_t whist[(kChunk / 64) * kSingleMaxExperts];
  __shared__ int32_t tot[2][kSingleMaxExperts];
  __shared__ int32_t sids[kChunk];
  const int t = threadIdx.x, token = t / LPT, at = t & (LPT - 1);
  int32_t id = -1;
  if ((t & ~63) / LPT < g.T) {  // (whole wavefronts)
    id = route_grouped_tokens<BF16, LPT, NS>(g, token, t & 63, sids + (t & ~63));
  }
  __syncthreads();  // (the choices are read)
  if (token < g.T && at < g.topk) sids[token * g.topk + at] = id;
  __syncthreads();
  const int64_t R = g.T * g.topk;
  single_chunk_sort(t < R ? sids[t] : -1, R, g.E, offsets, sorted_routes, inverse, whist, tot);
}

// The routing launch, with the sort (offsets set, and a lane's experts few enough for the registers of a workgroup of
// 1024) or alone; whether it sorted.
template <bool BF16, int LPT, int NS>
static bool launch_grouped(const GroupedRouting& g, int64_t* offsets, int32_t* sorted_routes, int32_t* inverse,
                           hipStream_t s) {
  constexpr int kTokens = 256 / LPT;
  if constexpr (NS <= 16) {
    if (offsets) {
      router_grouped_single_kernel<BF16, LPT, NS><<<1, kChunk, 0, s>>>(g, offsets, sorted_routes, inverse);
      return true;
    }
  }
  router_grouped_kernel<BF16, LPT, NS><<<dim3((unsigned)((g.T + kTokens - 1) / kTokens)), 256, 0, s>>>(g);
  return false;
}
// The lanes of a group and the experts of a lane, of LPT lanes for a token.
static GroupedRouting::Deal deal_groups(const GroupedRouting& g, int LPT) {
  GroupedRouting::Deal d{0, 0};
  while ((2 << d.lpg_log) * g.groups <= LPT) ++d.lpg_log;
  d.per = ((g.size + (1 << d.lpg_log) - 1 >> d.lpg_log) + 3) / 4 * 4;
  return d;
}
template <bool BF16>
static bool launch_grouped_slots(GroupedRouting& g, int64_t* offsets, int32_t* sorted_routes, int32_t* inverse,
                                 hipStream_t s) {
  g.deal = deal_groups(g, 16);
  g.deal64 = deal_groups(g, 64);
  // A wavefront per token where tokens are few, its walk over four experts a lane being the shorter (256 experts,
  // routing and sort in us, 64 lanes against 16: 10.7 to 11.6 at 17 tokens, 14.3 to 17.1 at 512, 18.4 to 18.5 at 2000,
  // 37.6 to 29.7 at 16384; 9.3 to 9.0 at 8, 10.6 to 9.3 at 16, which share a CU; 64 experts 10.4 to 9.6 at 512).
  const bool few = g.deal.per > 4 && g.T <= (offsets ? 8 : 2048);
  if (!few && g.topk <= 16 && g.groups <= 16 && g.deal.per <= 16) {  // (then four experts a lane of 64 at most)
    if (g.deal.per <= 4) return launch_grouped<BF16, 16, 4>(g, offsets, sorted_routes, inverse, s);
    if (g.deal.per <= 8) return launch_grouped<BF16, 16, 8>(g, offsets, sorted_routes, inverse, s);
    return launch_grouped<BF16, 16, 16>(g, offsets, sorted_routes, inverse, s);
  }
  g.deal = g.deal64;
  if (g.deal.per <= 4) return launch_grouped<BF16, 64, 4>(g, offsets, sorted_routes, inverse, s);
  if (g.deal.per <= 8) return launch_grouped<BF16, 64, 8>(g, offsets, sorted_routes, inverse, s);
  return launch_grouped<BF16, 64, 32>(g, offsets, sorted_routes, inverse, s);
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
    GroupedRouting g{logits, bias, T, (int)E, (int)topk, scoring, (int)groups, (int)(E / groups), (int)topk_groups,
                     renormalize != 0, 0, {}, {}, (double)factor, topk_weights, topk_ids};
    const uintptr_t logits_at = (uintptr_t)logits, bias_at = (uintptr_t)bias;
    g.quads = g.size % 4 == 0 && logits_at % (logits_bf16 ? 8 : 16) == 0 && bias_at % 16 == 0;
    int64_t* const offsets = T <= kGroupedSingleTokens && T * topk <= kChunk ? expert_offsets : nullptr;
    const bool sorted = logits_bf16 ? launch_grouped_slots<true>(g, offsets, sorted_routes, inverse, s)
                                    : launch_grouped_slots<false>(g, offsets, sorted_routes, inverse, s);
    MXL_CHECK_LAUNCH(who);
    if (sorted) return MXL_OK;
  }
  return mxl_moe_route(topk_ids, T, topk, E, sorted_routes, expert_offsets, inverse, workspace, workspace_bytes, stream);
}
