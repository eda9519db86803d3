// Low-rank adapters of many requests beside a shared linear layer on gfx950, and their gradients.
//
// Token t of a batch belongs to adapter a(t) (or to none): y[t] += s[a] B[a] (A[a] x[t]), A [R, K] and B [N, r] bf16 of
// each adapter, R = parts r: a merged layer's part p (columns [cols[p], cols[p + 1])) has the rows [p r, p r + r) of A.
//
//   shrink   v[t] = s A x[t]                                                        (also dv = s B^T dy, from B^T)
//   expand   y[t] += B v[t], in place                                               (also dx += A^T dv, from A^T)
//   outer    dB = sum_t dy[t] v[t]^T, dA = sum_t dv[t] x[t]^T over an adapter's tokens
//
// An infinity times v is one: it has to meet v's value alone, for with the rest, of either sign or zero, the sum would be NaN.
// So where a sum is NaN the kernels go over their values again, finite ones only against the rests (48 tokens of 32 adapters,
// the whole layer: 38.5 -> 39.0 us).
//
// v is never rounded to bf16: it is kept as bf16 v_hi = v and v_lo = v - v_hi, side by side along the MFMA's K (16 ranks
// of each in its 32), which leaves 2^-16 of it and costs nothing, for every one of these kernels waits for memory.  Sums
// are fp32 in the MFMA, joined in a fixed order.
#include <algorithm>
#include <type_traits>

#include "adapters.h"
#include "fp4.h"
#include "gemm_wide.h"

namespace mxl {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

// The tile's adapter and positions [lo, hi); false past the last tile.
__device__ __forceinline__ bool batch_tile(const AdapterBatch& b, int tile, int& slot, int64_t& lo, int64_t& hi) {
  const int4 t = reinterpret_cast<const int4*>(b.tiles)[tile];
  slot = t.x;
  lo = t.y;
  hi = t.z;
  return slot >= 0;
}

__device__ __forceinline__ bf16x8_t as_bf16x8(const u32x4& v) { return __builtin_bit_cast(bf16x8_t, v); }
__device__ __forceinline__ u32x4 keep(const u32x4& v, bool in) {
  return u32x4{in ? v[0] : 0u, in ? v[1] : 0u, in ? v[2] : 0u, in ? v[3] : 0u};
}

constexpr int kMaxShares = 8;  // of a column sum (the shrink kernel's)

// The wave's own writes to LDS are there for its other lanes.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// What the bf16 pair h leaves of (a, b), as bf16.  (Of an infinity nothing, where the difference would be NaN.)
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t h) {
  const float h0 = u2f(h << 16), h1 = u2f(h & 0xFFFF0000u);
  return cvt_pk_bf16(__builtin_isfinite(h0) ? a - h0 : 0.0f, __builtin_isfinite(h1) ? b - h1 : 0.0f);
}

// ------------------------------------------------------------------ tiles of a batch

__global__ __launch_bounds__(1024) void adapter_tiles_kernel(const int64_t* offsets, int slots, int num_tiles,
                                                             int32_t* tiles) {
  __shared__ int first[kMaxSlots + 1];  // the first tile of each adapter
  __shared__ int sums[16];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int before = 0;
  for (int base = 0; base < slots; base += 1024) {
    const int s = base + t;
    int n = s < slots ? (int)((offsets[s + 1] - offsets[s] + kAdapterTile - 1) / kAdapterTile) : 0, x = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    if (lane == 63) sums[wv] = x;
    __syncthreads();
    int at = before, all = 0;
    for (int w = 0; w < 16; ++w) {
      at += w < wv ? sums[w] : 0;
      all += sums[w];
    }
    if (s < slots) first[s] = at + x - n;
    before += all;
    __syncthreads();
  }
  if (t == 0) first[slots] = before;
  __syncthreads();
  for (int i = t; i < num_tiles; i += 1024) {
    int slot = -1, pos = 0, to = 0;
    if (i < before) {
      int lo = 0, hi = slots;  // the last adapter whose first tile is not past i
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= i) lo = mid; else hi = mid;
      }
      slot = lo;
      pos = (int)offsets[lo] + (i - first[lo]) * kAdapterTile;
      to = pos + kAdapterTile < (int)offsets[lo + 1] ? pos + kAdapterTile : (int)offsets[lo + 1];
    }
    reinterpret_cast<int4*>(tiles)[i] = int4{slot, pos, to, 0};
  }
}

// ------------------------------------------------------------------ shrink

// v[t] (adapters.h) of s sum_k rows[j][k] x[t][k].  BY_PART: part p's rows are [0, r) of the adapter's and its columns
// [cols[p], cols[p + 1]) (B^T [r, N]); else rows [p r, p r + r) and all columns (A).  A workgroup is a tile of 16 tokens
// by RC groups of 16 ranks; its waves share the columns and meet in LDS.  x is read once, the rows' A from L2, where its
// tiles share it.  Bound: memory (dy 2048 x 18432 to 2 x 16 ranks: 17.5 us, 4.3 TB/s); of many ranks A's loads (4096 x 5120
// to 64 ranks: 24 us, of which x alone is 8).  Loads by rows of the MFMA's operand put sixteen lines into every sixteen
// lanes, 64 cycles an instruction: 37.0 and 34 us where the loads are turned in LDS now.  SHARES: few tiles fill the card by splitting the columns over
// workgroups, whose fp32 sums [blockIdx.z][token][width] the expand kernel joins (48 tokens of 32 adapters, K = 5120, both
// kernels: 20.0 us whole, 14.1 in shares).
template <int RC, bool BY_PART, bool SHARES>
__global__ __launch_bounds__(RC < 4 ? 1024 : 512) void adapter_shrink_kernel(AdapterBatch b, LowRank l, const uint16_t* x, int64_t ldx,
                                                              int64_t cols, const uint16_t* rows, int64_t slot_stride,
                                                              int64_t ldr, const float* scaling, uint16_t* v,
                                                              float* shares) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  int slot;
  int64_t lo, hi;
  if (!batch_tile(b, blockIdx.x, slot, lo, hi)) return;
  const int per_part = (l.groups + RC - 1) / RC, part = blockIdx.y / per_part, g0 = (blockIdx.y - part * per_part) * RC;
  const int64_t c0 = BY_PART ? l.cols[part] : 0, c1 = BY_PART ? l.cols[part + 1] : cols;
  // Loads: lane 4 i + j has 16 bytes of row i, so that four lanes read a row's 64; the piece is j ^ (i >> 2), and through
  // the wave's own LDS, written as the lanes stand and read by row r and piece q, no two of sixteen lanes share a bank.
  const int i = lane >> 2, piece = (lane & 3) ^ (lane >> 4), from = 4 * r + (q ^ (r >> 2));
  const uint16_t* const xr = x + (int64_t)b.order[lo + i < hi ? lo + i : hi - 1] * ldx + 8 * piece;
  const int token = b.order[lo + r < hi ? lo + r : hi - 1];
  u32x4* const turn = reinterpret_cast<u32x4*>(red) + wv * (1 + RC) * 64;
  const uint16_t* ar[RC];
#pragma unroll
  for (int g = 0; g < RC; ++g) {
    const int j = 16 * (g0 + g) + i, row = (BY_PART ? 0 : part * l.rank) + (j < l.rank ? j : l.rank - 1);
    ar[g] = rows + slot * slot_stride + row * ldr + 8 * piece;
  }
  v4f acc[RC];
#pragma unroll
  for (int g = 0; g < RC; ++g) acc[g] = v4f{0.f, 0.f, 0.f, 0.f};
  // This wave's columns: 32 an MFMA, up to U of them loaded together; the waves' shares of a pass lie side by side.
  constexpr int U = RC == 1 ? 8 : 4;
  const int all = waves * (SHARES ? (int)gridDim.z : 1), who = (SHARES ? (int)blockIdx.z * waves : 0) + wv;
  const int units = (int)((c1 - c0 + 31) / 32), each = (units + all - 1) / all, passes = (each + U - 1) / U;
  const int step = (each + passes - 1) / passes;
  for (int u0 = who * step; u0 < units; u0 += all * step) {
    const int64_t k = c0 + 32 * (int64_t)u0, k1 = k + 32 * step < c1 ? k + 32 * step : c1;
    u32x4 xv[U], av[U][RC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= step) break;
      const int64_t at = k + 32 * u + 8 * piece < k1 ? k + 32 * u : c0 - 8 * piece;  // (columns come in eights)
#pragma unroll
      for (int g = 0; g < RC; ++g) av[u][g] = *reinterpret_cast<const u32x4*>(ar[g] + at);
      xv[u] = *reinterpret_cast<const u32x4*>(xr + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= step) break;
      const bool in = k + 32 * u + 8 * q < k1;
#pragma unroll
      for (int g = 0; g < RC; ++g) turn[64 * g + lane] = av[u][g];
      turn[64 * RC + lane] = xv[u];
      wave_lds_fence();
      const bf16x8_t xs = as_bf16x8(keep(turn[64 * RC + from], in));
#pragma unroll
      for (int g = 0; g < RC; ++g)
        acc[g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(keep(turn[64 * g + from], in)), xs, acc[g], 0, 0, 0);
      wave_lds_fence();
    }
  }
  __syncthreads();  // the sums take the same LDS
#pragma unroll
  for (int g = 0; g < RC; ++g) *reinterpret_cast<v4f*>(red + ((g * waves + wv) * 64 + lane) * 4) = acc[g];
  __syncthreads();
  const float s = scaling[slot];
  for (int f = wv; f < RC; f += waves) {
    v4f sum = *reinterpret_cast<const v4f*>(red + (f * waves * 64 + lane) * 4);
#pragma unroll 4
    for (int w = 1; w < waves; ++w) {
      const v4f one = *reinterpret_cast<const v4f*>(red + ((f * waves + w) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += one[e];
    }
    const int g = g0 + f;
    if constexpr (SHARES) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = 16 * g + 4 * q + e < l.rank ? sum[e] * s : 0.0f;
      if (lo + r < hi && g < l.groups)
        *reinterpret_cast<v4f*>(shares + (blockIdx.z * b.M + token) * l.width() + (part * l.groups + g) * 16 + 4 * q) = sum;
    } else if (lo + r < hi && g < l.groups) {
      uint32_t hl[2][2];
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float v0 = 16 * g + 4 * q + e < l.rank ? sum[e] * s : 0.0f, v1 = 16 * g + 4 * q + e + 1 < l.rank ? sum[e + 1] * s : 0.0f;
        hl[0][e / 2] = cvt_pk_bf16(v0, v1);
        hl[1][e / 2] = rest_of(v0, v1, hl[0][e / 2]);
      }
      uint16_t* const to = v + (int64_t)token * (2 * l.width()) + (part * l.groups + g) * 16 + 4 * q;
      *reinterpret_cast<uint2*>(to) = uint2{hl[0][0], hl[0][1]};
      *reinterpret_cast<uint2*>(to + l.width()) = uint2{hl[1][0], hl[1][1]};
    }
  }
}

// ------------------------------------------------------------------ expand

// y[t][n] += sum_j mat[n][j] v[t][j], mat [N, ldm] (j < valid) of the tile's adapter, j the ranks of n's part.  A wave is a
// tile of 16 tokens by 64 columns of one part: MFMA i's row 4 q + e is column 16 q + 4 i + e, so that after the four a
// lane holds 16 columns of one token side by side (the rows of y in 32-byte pieces; `wide`: they start on 16 bytes).
// SHARES: v comes as the shrink kernel's shares, and the first columns' workgroup writes it down.  y is the layer's output,
// rounded to bf16 by its launch, and is rounded again here: the layers' kernels write bf16, and an fp32 y between the two
// launches would be twice its bytes (against 64 bits, relative: 0.0022 instead of the one rounding's 0.0017).  Bound: B's bytes
// and two dependent round trips to memory (48 tokens of 32 adapters, rank 16, N = 17408: 9.2 us, 2.3 TB/s).
template <bool SHARES>
__global__ __launch_bounds__(256) void adapter_expand_kernel(AdapterBatch b, LowRank l, uint16_t* v, const float* shares,
                                                             int num_shares, const uint16_t* mat, int64_t slot_stride, int64_t ldm,
                                                             int valid, uint16_t* y, int64_t ldy, int wide) {
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, q = lane >> 4;
  int slot;
  int64_t lo, hi;
  if (!batch_tile(b, blockIdx.x, slot, lo, hi)) return;
  int part = 0, blk = 4 * blockIdx.y + wv;  // of 64 columns
  for (; part < l.parts; ++part) {
    const int n = (int)((l.cols[part + 1] - l.cols[part] + 63) / 64);
    if (blk < n) break;
    blk -= n;
  }
  if (part == l.parts) return;
  const int64_t c0 = l.cols[part] + (int64_t)blk * 64, c1 = l.cols[part + 1];
  const bool live = lo + r < hi;
  const int64_t token = b.order[live ? lo + r : hi - 1];
  uint16_t* const yr = y + token * ldy + c0 + 16 * q;
  const bool whole = wide && c0 + 64 <= c1;
  u32x4 old[2];
  if (whole) {
    old[0] = *reinterpret_cast<const u32x4*>(yr);
    old[1] = *reinterpret_cast<const u32x4*>(yr + 8);
  }
  const uint16_t* const vr = v + token * (2 * l.width()) + (q >> 1) * l.width() + part * l.groups * 16 + 8 * (q & 1);
  const uint16_t* mr[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = c0 + 16 * (r >> 2) + 4 * i + (r & 3);
    mr[i] = mat + slot * slot_stride + (n < c1 ? n : c1 - 1) * ldm + 8 * (q & 1);
  }
  extern __shared__ __attribute__((aligned(16))) float red[];
  // SHARES: the wave's rows of v, halves side by side, a row's 16-byte pieces exchanged by its number
  const int pieces = 4 * l.groups;
  u32x4* const joined = reinterpret_cast<u32x4*>(red) + wv * 16 * pieces;
  if constexpr (SHARES) {
    for (int i = lane; i < (int)(hi - lo) * pieces; i += 64) {  // four values
      const int row = i / pieces, c = i - row * pieces;
      const int64_t at = b.order[lo + row];
      const float* const src = shares + at * l.width() + part * l.groups * 16 + 4 * c;
      v4f one[kMaxShares];
#pragma unroll
      for (int z = 0; z < kMaxShares; ++z)
        one[z] = *reinterpret_cast<const v4f*>(src + (z < num_shares ? z : 0) * (b.M * l.width()));
      v4f sum = one[0];
#pragma unroll
      for (int z = 1; z < kMaxShares; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += z < num_shares ? one[z][e] : 0.0f;
      const uint32_t h0 = cvt_pk_bf16(sum[0], sum[1]), h1 = cvt_pk_bf16(sum[2], sum[3]);
      const uint2 big{h0, h1}, rest{rest_of(sum[0], sum[1], h0), rest_of(sum[2], sum[3], h1)};
      uint2* const to = reinterpret_cast<uint2*>(joined + row * pieces);
      to[2 * ((c >> 1) ^ (row & 3)) + (c & 1)] = big;
      to[2 * ((2 * l.groups + (c >> 1)) ^ (row & 3)) + (c & 1)] = rest;
      if (blk == 0) {
        uint16_t* const out = v + at * (2 * l.width()) + part * l.groups * 16 + 4 * c;
        *reinterpret_cast<uint2*>(out) = big;
        *reinterpret_cast<uint2*>(out + l.width()) = rest;
      }
    }
    wave_lds_fence();
  }
  v4f acc[4];
  auto product = [&](auto ODD) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int g = 0; g < l.groups; ++g) {
      const bool in = 16 * g + 8 * (q & 1) < valid;  // (ranks come in eights)
      u32x4 m[4], h;
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = *reinterpret_cast<const u32x4*>(mr[i] + (in ? 16 * g : -8 * (q & 1)));
      if constexpr (SHARES)
        h = joined[r * pieces + ((2 * l.groups * (q >> 1) + 2 * g + (q & 1)) ^ (r & 3))];
      else
        h = *reinterpret_cast<const u32x4*>(vr + 16 * g);
      if constexpr (decltype(ODD)::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) m[i][e] = q >> 1 ? adapter_finite(m[i][e]) : m[i][e];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(keep(m[i], in)), as_bf16x8(h), acc[i], 0, 0, 0);
    }
  };
  product(std::false_type{});
  bool nan = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) nan |= acc[i][e] != acc[i][e];
  if (__builtin_amdgcn_ballot_w64(live && nan) != 0) product(std::true_type{});
  if (!live) return;
  if (whole) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 d;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int i = 2 * h + w / 2, e = 2 * (w & 1);
        d[w] = f32_to_bf16(u2f(old[h][w] << 16) + acc[i][e]) | (uint32_t)f32_to_bf16(u2f(old[h][w] & 0xFFFF0000u) + acc[i][e + 1]) << 16;
      }
      *reinterpret_cast<u32x4*>(yr + 8 * h) = d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + 16 * q + 4 * i + e < c1) yr[4 * i + e] = f32_to_bf16(bf16_to_f32(yr[4 * i + e]) + acc[i][e]);
  }
}

// ------------------------------------------------------------------ outer products over an adapter's tokens

// sum_t big[t][c] v[t][j] over the adapter's positions of split z: to out [N, r] (OF_B: c a column of dy, j the ranks of
// its part) or out [R, K] (c a column of x, j all ranks).  A workgroup is 128 columns by RC groups; 32 tokens at a time
// go through LDS, both operands read from it transposed; the next 32 are on their way.  Bound: the big matrix' bytes where
// the shares fill the card (2048 x 18432 of dy 25.5 us, 3.0 TB/s), else a token tile's latency.
constexpr int kOuterCols = 128, kOuterStride = kOuterCols + 16, kOuterTokens = 32;
template <int RC, bool OF_B>
__global__ __launch_bounds__(256) void adapter_outer_kernel(AdapterBatch b, LowRank l, const uint16_t* big, int64_t ldb,
                                                            const uint16_t* v, int64_t slots, int splits,
                                                            int64_t out_cols, uint16_t* out, float* partial) {
  constexpr int VS = 16 * RC + 16;  // elements of a token's row of v in LDS, a half
  __shared__ __attribute__((aligned(16))) uint16_t tile[kOuterTokens * kOuterStride];
  __shared__ __attribute__((aligned(16))) uint16_t vt[2 * kOuterTokens * VS];
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, q = lane >> 4;
  const int64_t slot = blockIdx.z / splits;
  const int split = blockIdx.z - (int)slot * splits;
  // the workgroup's columns (of one part, where they are dy's) and groups of v
  int part = 0, blk = blockIdx.x;
  int64_t end = out_cols, c0;
  if (OF_B) {
    for (; part + 1 < l.parts; ++part) {
      const int n = (int)((l.cols[part + 1] - l.cols[part] + kOuterCols - 1) / kOuterCols);
      if (blk < n) break;
      blk -= n;
    }
    c0 = l.cols[part] + (int64_t)blk * kOuterCols;
    end = l.cols[part + 1];
  } else {
    c0 = (int64_t)blk * kOuterCols;
  }
  const int all = OF_B ? l.groups : l.parts * l.groups, g0 = blockIdx.y * RC, gv = (OF_B ? part * l.groups : 0) + g0;
  int64_t lo = b.offsets[slot], hi = b.offsets[slot + 1];
  hi = hi < b.M ? hi : b.M;
  const int64_t per = ((hi - lo + splits - 1) / splits + kOuterTokens - 1) / kOuterTokens * kOuterTokens;
  lo += split * per;
  hi = lo + per < hi ? lo + per : hi;
  v4f acc[2][RC];
  // pieces of 8: of the big matrix token t / 16 + 16 u, columns 8 (t % 16); of v half, token and ranks
  constexpr int VP = 2 * kOuterTokens * RC * 2, VU = (VP + 255) / 256;
  u32x4 d[2], x[VU];
  auto load = [&](int64_t p0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t pos = p0 + (t >> 4) + 16 * u, c = c0 + 8 * (t & 15);
      const bool in = pos < hi && c < end;
      d[u] = keep(*reinterpret_cast<const u32x4*>(big + (int64_t)b.order[pos < hi ? pos : hi - 1] * ldb + (c < end ? c : c0)), in);
    }
#pragma unroll
    for (int u = 0; u < VU; ++u) {
      const int at = t + 256 * u, h = at / (kOuterTokens * RC * 2), tok = at / (RC * 2) % kOuterTokens, j = 8 * (at % (RC * 2));
      const int64_t pos = p0 + tok;
      const bool in = pos < hi && g0 + j / 16 < all && at < VP;
      x[u] = keep(*reinterpret_cast<const u32x4*>(v + (int64_t)b.order[pos < hi ? pos : hi - 1] * (2 * l.width()) +
                                                  (in ? h * l.width() + gv * 16 + j : 0)), in);
    }
  };
  // a transposed fragment: eight tokens 8 q .. of column (of 16) r
  auto frag = [&](const uint16_t* at, int stride) {
    const uint16_t* const src = at + (8 * q + (r >> 2)) * stride + 4 * (r & 3);
    const uint2 y0 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src));
    const uint2 y1 = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 4 * stride)));
    return as_bf16x8(u32x4{y0.x, y0.y, y1.x, y1.y});
  };
  auto product = [&](auto ODD) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int g = 0; g < RC; ++g) acc[i][g] = v4f{0.f, 0.f, 0.f, 0.f};
    if (lo < hi) load(lo);
    for (int64_t p0 = lo; p0 < hi; p0 += kOuterTokens) {
      __syncthreads();  // the last tokens' reads
#pragma unroll
      for (int u = 0; u < 2; ++u) *reinterpret_cast<u32x4*>(tile + ((t >> 4) + 16 * u) * kOuterStride + 8 * (t & 15)) = d[u];
#pragma unroll
      for (int u = 0; u < VU; ++u) {
        const int at = t + 256 * u, row = at / (RC * 2), j = 8 * (at % (RC * 2));  // row: half 32 + token
        if (at < VP) *reinterpret_cast<u32x4*>(vt + row * VS + j) = x[u];
      }
      if (p0 + kOuterTokens < hi) load(p0 + kOuterTokens);
      __syncthreads();
      bf16x8_t cf[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) cf[i] = frag(tile + 32 * wv + 16 * i, kOuterStride);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (decltype(ODD)::value) {
          if (h == 1) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              u32x4 c = __builtin_bit_cast(u32x4, cf[i]);
#pragma unroll
              for (int e = 0; e < 4; ++e) c[e] = adapter_finite(c[e]);
              cf[i] = as_bf16x8(c);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < RC; ++g) {
          const bf16x8_t rf = frag(vt + h * kOuterTokens * VS + 16 * g, VS);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(OF_B ? rf : cf[i], OF_B ? cf[i] : rf, acc[i][g], 0, 0, 0);
        }
      }
    }
  };
  product(std::false_type{});
  int nan = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int g = 0; g < RC; ++g)
#pragma unroll
      for (int e = 0; e < 4; ++e) nan |= acc[i][g][e] != acc[i][g][e] ? 1 : 0;
  if (__syncthreads_or(nan)) product(std::true_type{});
  // OF_B: lane holds ranks 4 q .. + 3 of column r; else columns 4 q .. + 3 of rank r
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int g = 0; g < RC; ++g) {
      if (g0 + g >= all) continue;
      const int64_t c = c0 + 32 * wv + 16 * i + (OF_B ? r : 4 * q);
      const int j = 16 * ((g0 + g) % l.groups) + (OF_B ? 4 * q : r);  // rank of its part
      if (c >= end || j >= l.rank) continue;
      const int64_t at = OF_B ? (slot * out_cols + c) * l.rank + j
                              : ((slot * l.parts + (g0 + g) / l.groups) * l.rank + j) * out_cols + c;
      if (splits > 1) {
        *reinterpret_cast<v4f*>(partial + split * slots * out_cols * l.rank * (OF_B ? 1 : l.parts) + at) = acc[i][g];
      } else {
        uint16_t h[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = f32_to_bf16(acc[i][g][e]);
        *reinterpret_cast<uint2*>(out + at) = uint2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
      }
    }
}

// out[i] = the sum of `splits` partials, rounded; four values a thread.
__global__ __launch_bounds__(256) void adapter_join_kernel(const float* partial, int splits, int64_t count, uint16_t* out) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= count) return;
  v4f s = *reinterpret_cast<const v4f*>(partial + at);
#pragma unroll 4
  for (int k = 1; k < splits; ++k) {
    const v4f x = *reinterpret_cast<const v4f*>(partial + k * count + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += x[e];
  }
  uint16_t h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = f32_to_bf16(s[e]);
  *reinterpret_cast<uint2*>(out + at) = uint2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
}

// dst [cols, width] = the transpose of src [rows, cols] of each adapter; row p rank + j of src goes to column p 16 groups + j
// (zeros between the parts), with parts = 1 and width = rank simply to its own.  32 x 32 tiles through LDS.
__global__ __launch_bounds__(256) void adapter_transpose_kernel(const uint16_t* src, int64_t rows, int64_t cols, int parts,
                                                                int rank, int width, uint16_t* dst) {
  __shared__ uint16_t tile[32][34];
  const int64_t slot = blockIdx.z, c0 = (int64_t)blockIdx.x * 32;
  const int w0 = blockIdx.y * 32, x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int per = width / parts;
  for (int i = y; i < 32; i += 8) {
    const int w = w0 + i, p = w / per, j = w - p * per;
    const int64_t c = c0 + x;
    tile[i][x] = w < width && j < rank && c < cols ? src[(slot * rows + p * rank + j) * cols + c] : (uint16_t)0;
  }
  __syncthreads();
  for (int i = y; i < 32; i += 8)
    if (c0 + i < cols && w0 + x < width) dst[(slot * cols + c0 + i) * width + w0 + x] = tile[x][i];
}

}  // namespace mxl

// ------------------------------------------------------------------- C ABI

using namespace mxl;

namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t tile_count(int64_t M, int64_t slots) { return std::min(M, ceil_div(M, kAdapterTile) + std::min(slots, M)); }

// Groups of 16 ranks a workgroup of shrink takes: up to four, which share the reads of x, once the tiles fill the card
// without more workgroups (4096 x 5120 to 64 ranks: one group 33.0 us, two 25.9, four 24.4).
int shrink_groups(int64_t tiles, int groups) { return tiles < 256 || groups < 2 ? 1 : groups < 4 ? 2 : 4; }

// The sizes that a call takes; queries of others say 0.
bool batch_ok(int64_t M, int64_t slots) { return M > 0 && M <= 0x7FFFFFFF && slots > 0 && slots <= kMaxSlots; }
bool low_rank_ok(int64_t parts, int64_t rank) {
  return parts >= 1 && parts <= kMaxParts && rank > 0 && rank <= kMaxRank && rank % 8 == 0;
}

int check_batch(const char* who, int64_t M, int64_t slots, const int32_t* order, const int64_t* offsets,
                const int32_t* tiles, int64_t num_tiles) {
  MXL_CHECK_ARG(M >= 0 && M <= 0x7FFFFFFF && slots > 0 && slots <= kMaxSlots, "%s: need 0 <= M < 2^31 and 0 < slots <= %d (M=%lld slots=%lld)",
                who, kMaxSlots, (long long)M, (long long)slots);
  MXL_CHECK_ARG(num_tiles == tile_count(M, slots), "%s: %lld tiles for M=%lld slots=%lld, need %lld", who,
                (long long)num_tiles, (long long)M, (long long)slots, (long long)tile_count(M, slots));
  MXL_CHECK_ARG(M == 0 || (order && offsets && tiles && ((uintptr_t)tiles & 15) == 0),
                "%s: needs the batch's order, offsets and tiles (16-byte aligned)", who);
  return MXL_OK;
}

int make_low_rank(const char* who, int64_t parts, const int64_t* cols, int64_t rank, int64_t K, LowRank& l) {
  MXL_CHECK_ARG(parts >= 1 && parts <= kMaxParts && cols, "%s: need 1 to %d parts (%lld)", who, kMaxParts, (long long)parts);
  MXL_CHECK_ARG(rank > 0 && rank <= kMaxRank && rank % 8 == 0, "%s: need a rank of 8 to %d, a multiple of 8 (%lld)", who,
                kMaxRank, (long long)rank);
  MXL_CHECK_ARG(K > 0 && K % 8 == 0, "%s: need K > 0, K %% 8 == 0 (K=%lld)", who, (long long)K);
  MXL_CHECK_ARG(cols[0] == 0, "%s: the parts start at column 0", who);
  l.parts = (int)parts;
  l.rank = (int)rank;
  l.groups = (int)((rank + 15) / 16);
  for (int p = 0; p <= parts; ++p) {
    MXL_CHECK_ARG(p == 0 || cols[p] > cols[p - 1], "%s: part %d has no columns", who, p - 1);
    MXL_CHECK_ARG(p == parts || cols[p] % 16 == 0, "%s: part %d does not start on a multiple of 16 columns", who, p);
    l.cols[p] = cols[p];
  }
  return MXL_OK;
}

int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return MXL_OK;
  set_error("%s: launch failed: %s", who, hipGetErrorString(e));
  return MXL_EHIP;
}

// Shares of the columns where the expand kernel follows: until some 256 workgroups run, or a wave has 32 columns.  (48
// tokens of 32 adapters of rank 16, K = 5120, N = 17408, us of both kernels: one share 20.0, two 15.2, five 14.1.)
int shrink_shares(int64_t tiles, const LowRank& l, int64_t cols) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({kMaxShares, 256 / (tiles * l.parts * l.groups), cols / 256}));
}

template <bool BY_PART>
int launch_shrink(const char* who, const AdapterBatch& b, const LowRank& l, const uint16_t* x, int64_t ldx, int64_t cols,
                  const uint16_t* rows, int64_t slot_stride, int64_t ldr, const float* scaling, uint16_t* v,
                  float* shares, int num_shares, hipStream_t s) {
  const int rc = num_shares > 1 ? 1 : shrink_groups(b.num_tiles, l.groups);
  const int64_t chunks = l.parts * ceil_div(l.groups, rc);
  const int waves = num_shares == 1 && rc < 4 && b.num_tiles * chunks <= 512 ? 16 : 8;
  const dim3 grid((unsigned)b.num_tiles, (unsigned)chunks, (unsigned)num_shares);
  const unsigned lds = (unsigned)((1 + rc) * waves * 1024);
#define MXL_SHRINK(RC_, SHARES_)                                                                                          \
  if (rc == RC_ && (num_shares > 1) == SHARES_)                                                                           \
    adapter_shrink_kernel<RC_, BY_PART, SHARES_><<<grid, 64 * waves, lds, s>>>(b, l, x, ldx, cols, rows, slot_stride, ldr, \
                                                                               scaling, v, shares);
  MXL_SHRINK(1, false) MXL_SHRINK(2, false) MXL_SHRINK(4, false)
  if constexpr (!BY_PART) MXL_SHRINK(1, true)
#undef MXL_SHRINK
  return launched(who);
}

int launch_expand(const char* who, const AdapterBatch& b, const LowRank& l, uint16_t* v, const float* shares,
                  int num_shares, const uint16_t* mat, int64_t slot_stride, int64_t ldm, int valid, uint16_t* y,
                  int64_t ldy, hipStream_t s) {
  int64_t blocks = 0;
  for (int p = 0; p < l.parts; ++p) blocks += ceil_div(l.cols[p + 1] - l.cols[p], 64);
  MXL_CHECK_ARG(blocks <= 4 * 0xFFFF, "%s: too many columns", who);
  const dim3 grid((unsigned)b.num_tiles, (unsigned)ceil_div(blocks, 4));
  const int wide = ldy % 8 == 0 && ((uintptr_t)y & 15) == 0;
  if (num_shares > 1)
    adapter_expand_kernel<true><<<grid, 256, (unsigned)(4096 * l.groups), s>>>(b, l, v, shares, num_shares, mat, slot_stride, ldm, valid, y, ldy, wide);
  else
    adapter_expand_kernel<false><<<grid, 256, 0, s>>>(b, l, v, shares, num_shares, mat, slot_stride, ldm, valid, y, ldy, wide);
  return launched(who);
}

// Shares of an adapter's tokens in the outer products, where columns and groups alone are too few workgroups: some 128
// tokens each (of adapters with as many), and none while an adapter has fewer than 256: a share costs the join's launch.
// (2048 tokens of one adapter, rank 16, us with the join: of N = 18432 one share 69.4, four 35.2, here 29.5; of K = 2560
// 70.3, 26.7, 14.4.  333 tokens of three, N = 5120, K = 2688: one share 10.3 and 10.8, four 9.5 and 8.2 and two launches
// more, which the host pays for.)
int outer_splits(int64_t M, int64_t slots, int64_t wgs) {
  const int64_t each = M / slots;
  return each < 256 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>({32, ceil_div(768, wgs * slots), each / 128}));
}
int64_t outer_blocks(const LowRank& l, int64_t cols, bool of_b) {
  int64_t blocks = 0;
  if (!of_b) return ceil_div(cols, kOuterCols);
  for (int p = 0; p < l.parts; ++p) blocks += ceil_div(l.cols[p + 1] - l.cols[p], kOuterCols);
  return blocks;
}
int outer_groups(const LowRank& l, bool of_b) {
  const int all = of_b ? l.groups : l.parts * l.groups;
  return all >= 4 ? 4 : all >= 2 ? 2 : 1;
}
int outer_splits(const LowRank& l, int64_t M, int64_t slots, int64_t cols, bool of_b) {
  const int all = of_b ? l.groups : l.parts * l.groups;
  return outer_splits(M, slots, outer_blocks(l, cols, of_b) * ceil_div(all, outer_groups(l, of_b)));
}

template <bool OF_B>
int launch_outer(const char* who, const AdapterBatch& b, const LowRank& l, int64_t slots, const uint16_t* big, int64_t ldb,
                 int64_t cols, const uint16_t* v, uint16_t* out, float* partial, hipStream_t s) {
  const int splits = outer_splits(l, b.M, slots, cols, OF_B), rc = outer_groups(l, OF_B);
  MXL_CHECK_ARG(slots * splits <= 0xFFFF, "%s: too many adapters", who);
  const dim3 grid((unsigned)outer_blocks(l, cols, OF_B), (unsigned)ceil_div(OF_B ? l.groups : l.parts * l.groups, rc),
                  (unsigned)(slots * splits));
#define MXL_OUTER(RC_) \
  if (rc == RC_)       \
    adapter_outer_kernel<RC_, OF_B><<<grid, 256, 0, s>>>(b, l, big, ldb, v, slots, splits, cols, out, partial);
  MXL_OUTER(1) MXL_OUTER(2) MXL_OUTER(4)
#undef MXL_OUTER
  const int rc2 = launched(who);
  if (rc2 != MXL_OK || splits == 1) return rc2;
  const int64_t count = slots * cols * l.rank * (OF_B ? 1 : l.parts);
  adapter_join_kernel<<<dim3((unsigned)ceil_div(count, 1024)), 256, 0, s>>>(partial, splits, count, out);
  return launched(who);
}

// Pieces of a workspace, each on 256 bytes.  Without a base only the sizes count.
struct Pieces {
  uint8_t* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* const at = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
};

struct GradScratch {
  void *bt, *at, *dv, *partial;
  int64_t bytes;
};
GradScratch grad_scratch(uint8_t* base, int64_t M, int64_t K, int64_t slots, const LowRank& l) {
  const int64_t N = l.cols[l.parts], nb = outer_splits(l, M, slots, N, true), na = outer_splits(l, M, slots, K, false);
  Pieces p{base};
  GradScratch g;
  g.bt = p.take(slots * l.rank * N * 2);
  g.at = p.take(rows_add(M, slots) ? 0 : slots * K * l.width() * 2);
  g.dv = p.take(M * l.width() * 4);
  g.partial = p.take(slots * l.rank * 4 * std::max(nb > 1 ? nb * N : 0, na > 1 ? na * l.parts * K : 0));
  g.bytes = p.used;
  return g;
}

}  // namespace

extern "C" int64_t mxl_adapter_tile_count(int64_t M, int64_t slots) {
  return batch_ok(M, slots) ? tile_count(M, slots) : 0;
}

extern "C" int mxl_adapter_tiles(const int64_t* offsets, int64_t M, int64_t slots, int32_t* tiles, int64_t num_tiles,
                                 void* stream) {
  const char* who = "mxl_adapter_tiles";
  MXL_CHECK_ARG(M >= 0 && M <= 0x7FFFFFFF && slots > 0 && slots <= kMaxSlots, "%s: need 0 <= M < 2^31 and 0 < slots <= %d", who, kMaxSlots);
  if (M == 0) return MXL_OK;
  MXL_CHECK_ARG(offsets && tiles && ((uintptr_t)tiles & 15) == 0 && num_tiles == tile_count(M, slots), "%s: needs %lld tiles", who,
                (long long)tile_count(M, slots));
  adapter_tiles_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(offsets, (int)slots, (int)num_tiles, tiles);
  return launched(who);
}

extern "C" int64_t mxl_adapter_v_elems(int64_t M, int64_t parts, int64_t rank) {
  return batch_ok(M, 1) && low_rank_ok(parts, rank) ? M * 2 * parts * ceil_div(rank, 16) * 16 : 0;
}

extern "C" int64_t mxl_adapter_apply_workspace_bytes(int64_t M, int64_t K, int64_t slots, int64_t parts, int64_t rank) {
  if (!batch_ok(M, slots) || !low_rank_ok(parts, rank) || K <= 0) return 0;
  LowRank l{};
  l.parts = (int)parts;
  l.groups = (int)ceil_div(rank, 16);
  const int shares = shrink_shares(tile_count(M, slots), l, K);
  return shares > 1 ? shares * M * l.width() * 4 : 0;
}

extern "C" int mxl_adapter_apply(const void* x, int64_t M, int64_t K, int64_t ldx, const void* a, const void* b,
                                 const float* scaling, int64_t slots, int64_t parts, const int64_t* cols, int64_t rank,
                                 const int32_t* order, const int64_t* offsets, const int32_t* tiles, int64_t num_tiles,
                                 void* v, int64_t v_elems, void* y, int64_t ldy, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_adapter_apply";
  LowRank l;
  int rc = check_batch(who, M, slots, order, offsets, tiles, num_tiles);
  if (rc == MXL_OK) rc = make_low_rank(who, parts, cols, rank, K, l);
  if (rc != MXL_OK || M == 0) return rc;
  const int64_t N = l.cols[l.parts];
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0 && ldy >= N, "%s: need ldx >= K, a multiple of 8, and ldy >= N", who);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)v) & 15) == 0, "%s: x, a, b and v must be 16-byte aligned", who);
  MXL_CHECK_ARG(v_elems >= mxl_adapter_v_elems(M, parts, rank), "%s: v holds %lld values, needs %lld", who,
                (long long)v_elems, (long long)mxl_adapter_v_elems(M, parts, rank));
  const int64_t need = mxl_adapter_apply_workspace_bytes(M, K, slots, parts, rank);
  MXL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "%s: needs a 16-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  const AdapterBatch batch{order, offsets, tiles, (int)num_tiles, M};
  const int64_t R = parts * rank;
  const int shares = shrink_shares(num_tiles, l, K);
  rc = launch_shrink<false>(who, batch, l, (const uint16_t*)x, ldx, K, (const uint16_t*)a, R * K, K, scaling, (uint16_t*)v,
                            (float*)workspace, shares, (hipStream_t)stream);
  if (rc != MXL_OK) return rc;
  return launch_expand(who, batch, l, (uint16_t*)v, (const float*)workspace, shares, (const uint16_t*)b, N * rank, rank,
                       l.rank, (uint16_t*)y, ldy, (hipStream_t)stream);
}

// ---- the layer and its adapters in one call

extern "C" int mxl_quantize_mxfp8(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes, void* scales,
                                  void* stream);
extern "C" int mxl_quantize_mxfp4(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes, void* scales,
                                  void* stream);
extern "C" int mxl_quantize_block_fp8(const void* x, int64_t M, int64_t K, void* codes, void* scales, void* stream);

static int64_t code_bytes(int64_t M, int64_t K, int fmt) { return ceil_div(fmt == kE2M1 ? M * (K / 2) : M * K, 256) * 256; }

// The product adds the adapters where it runs in the tiles anyway (from 17 rows) and walks few of them a tile; 32-bit
// offsets.
extern "C" int mxl_adapter_linear_supported(int64_t M, int64_t N, int64_t K, int fmt, int block, int64_t slots,
                                            int64_t parts, int64_t rank) {
  if (!batch_ok(M, slots) || !low_rank_ok(parts, rank) || N <= 0 || N > 0x7FFFFFFF || K <= 0 || K > 0x7FFFFFFF) return 0;
  if (fmt != kE4M3 && fmt != kE2M3 && fmt != kE3M2 && fmt != kE2M1) return 0;
  return M >= 17 && K % 128 == 0 && rows_add(M, slots) &&
         wide_tiles_eligible(M, N, K, block != 0) && M <= (int64_t(1) << 32) / (4 * parts * ceil_div(rank, 16) * 16) &&
         N <= (int64_t(1) << 31) / (2 * rank) && (fmt == kE4M3 || !block);
}

extern "C" int64_t mxl_adapter_linear_workspace_bytes(int64_t M, int64_t K, int fmt, int block) {
  if (M <= 0 || M > 0x7FFFFFFF || K <= 0 || K > 0x7FFFFFFF) return 0;
  return code_bytes(M, K, fmt) + (block ? M * (K / 128) * 4 : M * (K / 32));
}

extern "C" int mxl_adapter_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, const void* w_tiled,
                                  const void* sw, int fmt, int block, const void* bias, const void* a, const void* b,
                                  const float* scaling, int64_t slots, int64_t parts, const int64_t* cols, int64_t rank,
                                  const int32_t* ids, const int32_t* order, const int64_t* offsets, const int32_t* tiles,
                                  int64_t num_tiles, void* v, int64_t v_elems, void* y, int64_t ldy, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_adapter_linear";
  LowRank l;
  int rc = check_batch(who, M, slots, order, offsets, tiles, num_tiles);
  if (rc == MXL_OK) rc = make_low_rank(who, parts, cols, rank, K, l);
  if (rc != MXL_OK || M == 0) return rc;
  const int64_t N = l.cols[l.parts], R = parts * rank;
  MXL_CHECK_ARG(fmt == kE4M3 || fmt == kE2M3 || fmt == kE3M2 || fmt == kE2M1, "%s: unknown format %d", who, fmt);
  MXL_CHECK_ARG(!block || (fmt == kE4M3 && ldx == K), "%s: block-FP8 takes E4M3 weights and contiguous rows", who);
  MXL_CHECK_ARG(fmt != kE2M1 || fp4_rule(rule), "%s: unknown rule %d", who, rule);
  if (!mxl_adapter_linear_supported(M, N, K, fmt, block, slots, parts, rank)) {
    set_error("%s: %lld rows of %lld adapters do not run in one product (N=%lld K=%lld)", who, (long long)M,
              (long long)slots, (long long)N, (long long)K);
    return MXL_EUNSUPPORTED;
  }
  MXL_CHECK_ARG(ids && ldx >= K && ldx % 8 == 0 && ldy >= N, "%s: need ids, ldx >= K, a multiple of 8, and ldy >= N", who);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)w_tiled | (uintptr_t)a | (uintptr_t)b | (uintptr_t)v) & 15) == 0 &&
                    ((uintptr_t)sw & 3) == 0 && ((uintptr_t)y & 1) == 0, "%s: x, w, a, b and v must be 16-byte aligned", who);
  MXL_CHECK_ARG(v_elems >= mxl_adapter_v_elems(M, parts, rank), "%s: v holds %lld values, needs %lld", who,
                (long long)v_elems, (long long)mxl_adapter_v_elems(M, parts, rank));
  MXL_CHECK_ARG(workspace && workspace_bytes >= mxl_adapter_linear_workspace_bytes(M, K, fmt, block) &&
                    ((uintptr_t)workspace & 255) == 0, "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who,
                (long long)mxl_adapter_linear_workspace_bytes(M, K, fmt, block), (long long)workspace_bytes);
  hipStream_t s = (hipStream_t)stream;
  uint8_t* const codes = (uint8_t*)workspace;
  uint8_t* const scales = codes + code_bytes(M, K, fmt);
  rc = block          ? mxl_quantize_block_fp8(x, M, K, codes, scales, stream)
       : fmt == kE2M1 ? mxl_quantize_mxfp4(x, M, K, ldx, rule, codes, scales, stream)
                      : mxl_quantize_mxfp8(x, M, K, ldx, rule, codes, scales, stream);
  if (rc != MXL_OK) return rc;
  const AdapterBatch batch{order, offsets, tiles, (int)num_tiles, M};
  rc = launch_shrink<false>(who, batch, l, (const uint16_t*)x, ldx, K, (const uint16_t*)a, R * K, K, scaling, (uint16_t*)v,
                            nullptr, 1, s);
  if (rc != MXL_OK) return rc;
  GemmParams p{};
  p.M = p.a_rows = M; p.N = N; p.K = K; p.KT = ceil_div(K, kTileK);
  p.a = codes; p.sa = scales; p.lda = fmt == kE2M1 ? K / 2 : K;
  p.w = (const uint8_t*)w_tiled; p.sw = sw; p.bias = (const uint16_t*)bias; p.out = (uint16_t*)y; p.ldc = ldy;
  p.row_div = 1; p.S = 1;
  RowAdapters add;
  add.ids = ids; add.slots = (int)slots; add.v = (const uint16_t*)v; add.mat = (const uint16_t*)b;
  add.slot_stride = N * rank; add.ldm = rank; add.l = l;
  WideGrid g{};
  int64_t grid;
  const WideConfig c = wide_tiles_whole(M, N, K, fmt, block != 0, g, grid);
  const hipError_t e = launch_adapter_tiles(fmt, block != 0, c, p, g, add, grid, s);
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return MXL_EHIP;
  }
  return MXL_OK;
}

// ---- gradients

extern "C" int64_t mxl_adapter_grad_workspace_bytes(int64_t M, int64_t K, int64_t slots, int64_t parts,
                                                    const int64_t* cols, int64_t rank, int block) {
  LowRank l;
  if (!batch_ok(M, slots) || make_low_rank("mxl_adapter_grad_workspace_bytes", parts, cols, rank, K, l) != MXL_OK) return 0;
  return grad_scratch(nullptr, M, K, slots, l).bytes + input_grad_bytes(M, cols[parts], K, block);
}

extern "C" int mxl_adapter_grad(const void* x, int64_t M, int64_t K, int64_t ldx, const void* dy, int64_t lddy,
                                const void* w_tiled, const void* sw, int fmt, int block, const void* a, const void* b,
                                const float* scaling, int64_t slots, int64_t parts, const int64_t* cols, int64_t rank,
                                const int32_t* ids, const int32_t* order, const int64_t* offsets, const int32_t* tiles,
                                int64_t num_tiles, const void* v, int64_t v_elems, void* dx, int64_t lddx, void* da,
                                void* db, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_adapter_grad";
  LowRank l;
  int rc = check_batch(who, M, slots, order, offsets, tiles, num_tiles);
  if (rc == MXL_OK) rc = make_low_rank(who, parts, cols, rank, K, l);
  if (rc != MXL_OK || M == 0) return rc;
  const int64_t N = l.cols[l.parts], R = parts * rank;
  MXL_CHECK_ARG(N % 8 == 0, "%s: need N %% 8 == 0 (N=%lld)", who, (long long)N);
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0 && lddy >= N && lddy % 8 == 0 && (!dx || (ids && lddx >= K && lddx % 4 == 0)),
                "%s: need ldx >= K, lddy >= N, multiples of 8, and for dx ids and lddx >= K, a multiple of 4", who);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)a | (uintptr_t)b | (uintptr_t)v | (uintptr_t)da | (uintptr_t)db) & 15) == 0,
                "%s: operands must be 16-byte aligned", who);
  MXL_CHECK_ARG(!db || v_elems >= mxl_adapter_v_elems(M, parts, rank), "%s: v holds %lld values", who, (long long)v_elems);
  const int64_t need = mxl_adapter_grad_workspace_bytes(M, K, slots, parts, cols, rank, block);
  MXL_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
                "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  const GradScratch g = grad_scratch((uint8_t*)workspace, M, K, slots, l);
  hipStream_t s = (hipStream_t)stream;
  const AdapterBatch batch{order, offsets, tiles, (int)num_tiles, M};
  if (db) {
    rc = launch_outer<true>(who, batch, l, slots, (const uint16_t*)dy, lddy, N, (const uint16_t*)v, (uint16_t*)db,
                            (float*)g.partial, s);
    if (rc != MXL_OK) return rc;
  }
  if (!da && !dx) return MXL_OK;
  // B [N, r] -> [r, N]
  MXL_CHECK_ARG(ceil_div(std::max(N, K), 32) <= 0xFFFF && slots <= 0xFFFF, "%s: too large", who);
  adapter_transpose_kernel<<<dim3((unsigned)ceil_div(l.rank, 32), (unsigned)ceil_div(N, 32), (unsigned)slots), 256, 0, s>>>(
      (const uint16_t*)b, N, l.rank, 1, (int)N, (int)N, (uint16_t*)g.bt);
  rc = launched(who);
  if (rc == MXL_OK)
    rc = launch_shrink<true>(who, batch, l, (const uint16_t*)dy, lddy, N, (const uint16_t*)g.bt, l.rank * N, N, scaling,
                             (uint16_t*)g.dv, nullptr, 1, s);
  if (rc == MXL_OK && da)
    rc = launch_outer<false>(who, batch, l, slots, (const uint16_t*)x, ldx, K, (const uint16_t*)g.dv,
                             (uint16_t*)da, (float*)g.partial, s);
  if (rc != MXL_OK || !dx) return rc;
  RowAdapters more;
  more.ids = ids; more.slots = (int)slots; more.v = (const uint16_t*)g.dv; more.mat = (const uint16_t*)a;
  more.slot_stride = R * K; more.ldm = K; more.l = l;
  const bool within = rows_add(M, slots);
  rc = input_grad(who, dy, M, N, lddy, w_tiled, sw, K, fmt, block, dx, lddx, (uint8_t*)workspace + g.bytes,
                  workspace_bytes - g.bytes, within ? &more : nullptr, stream);
  if (rc != MXL_OK || within) return rc;
  // A [R, K] -> [K, parts 16 groups]
  adapter_transpose_kernel<<<dim3((unsigned)ceil_div(K, 32), (unsigned)ceil_div(l.width(), 32), (unsigned)slots), 256, 0, s>>>(
      (const uint16_t*)a, R, K, l.parts, l.rank, l.width(), (uint16_t*)g.at);
  rc = launched(who);
  LowRank one = l;  // all ranks at once
  one.parts = 1;
  one.groups = l.parts * l.groups;
  one.rank = one.groups * 16;
  one.cols[1] = K;
  if (rc == MXL_OK)
    rc = launch_expand(who, batch, one, (uint16_t*)g.dv, nullptr, 1, (const uint16_t*)g.at, K * l.width(), l.width(), one.rank,
                       (uint16_t*)dx, lddx, s);
  return rc;
}
