// Low-rank adapters of many requests beside a shared linear layer on gfx950, and their gradients.
//
// Token t of a batch belongs to adapter a(t) (or to none): y[t] += s[a] B[a] (A[a] x[t]), A [R, K] and B [N, r] bf16 of
// each adapter, R = parts r: a merged layer's part p (columns [cols[p], cols[p + 1])) has the rows [p r, p r + r) of A.
//
//   shrink   v[t] = s A x[t]: fp32, by position in the batch sorted by adapter      (also dv = s B^T dy, from B^T)
//   expand   y[t] += B v[t], in place                                               (also dx += A^T dv, from A^T)
//   outer    dB = sum_t dy[t] v[t]^T, dA = sum_t dv[t] x[t]^T over an adapter's tokens
//
// v is never rounded to bf16: a product with it takes bf16 v_hi = v and v_lo = v - v_hi side by side along the MFMA's
// K (16 ranks of each in its 32), which leaves 2^-17 of it and costs nothing, for every one of these kernels waits for
// memory.  Sums are fp32 in the MFMA, joined in a fixed order.
#include <algorithm>

#include "mx_common.h"

namespace mxl {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

constexpr int kMaxParts = 8, kMaxRank = 256, kMaxSlots = 4096;

// Tokens sorted by adapter: positions [offsets[a], offsets[a + 1]) of order are adapter a's, in tiles of `rows`
// positions: tile i is (adapter, first position), adapter -1 past the last.
struct Batch {
  const int32_t* order;
  const int64_t* offsets;
  const int32_t* tiles;
  int num_tiles, rows;
  int64_t M;
};

struct LowRank {
  int parts, rank, groups;  // groups: of 16 ranks of a part
  int64_t cols[kMaxParts + 1];
  __host__ __device__ int width() const { return parts * groups * 16; }  // of a row of v
};

// Adapter and positions [lo, hi) of piece i, `rows` positions (a divisor of b.rows); false where there are none.
__device__ __forceinline__ bool batch_tile(const Batch& b, int rows, int i, int& slot, int64_t& lo, int64_t& hi) {
  const int pieces = b.rows / rows, tile = i / pieces;
  slot = b.tiles[2 * tile];
  if (slot < 0) return false;
  lo = b.tiles[2 * tile + 1] + (i - tile * pieces) * rows;
  const int64_t end = b.offsets[slot + 1];
  hi = lo + rows < end ? lo + rows : end;
  hi = hi < b.M ? hi : b.M;
  return lo < hi;
}

__device__ __forceinline__ bf16x8_t as_bf16x8(const uint4& v) { return __builtin_bit_cast(bf16x8_t, v); }

__device__ __forceinline__ uint4 keep(const uint4& v, bool in) {
  return uint4{in ? v.x : 0u, in ? v.y : 0u, in ? v.z : 0u, in ? v.w : 0u};
}

// Eight fp32 as bf16: the values, or what they leave of the fp32.
__device__ __forceinline__ uint4 split8(const float* v, bool rest) {
  uint32_t d[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    d[i] = cvt_pk_bf16(v[2 * i], v[2 * i + 1]);
    if (rest) {
      // (an infinity leaves NaN of itself: its rest is zero)
      const float h0 = u2f(d[i] << 16), h1 = u2f(d[i] & 0xFFFF0000u);
      const float r0 = v[2 * i] - h0, r1 = v[2 * i + 1] - h1;
      d[i] = cvt_pk_bf16(__builtin_isfinite(h0) ? r0 : 0.0f, __builtin_isfinite(h1) ? r1 : 0.0f);
    }
  }
  return uint4{d[0], d[1], d[2], d[3]};
}

// ------------------------------------------------------------------ tiles of a batch

__global__ __launch_bounds__(1024) void adapter_tiles_kernel(const int64_t* offsets, int slots, int rows, int num_tiles,
                                                             int32_t* tiles) {
  __shared__ int first[kMaxSlots + 1];  // the first tile of each adapter
  __shared__ int sums[16];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  int before = 0;
  for (int base = 0; base < slots; base += 1024) {
    const int s = base + t;
    int n = s < slots ? (int)((offsets[s + 1] - offsets[s] + rows - 1) / rows) : 0, x = n;
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
    int slot = -1, pos = 0;
    if (i < before) {
      int lo = 0, hi = slots;  // the last adapter whose first tile is not past i
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (first[mid] <= i) lo = mid; else hi = mid;
      }
      slot = lo;
      pos = (int)offsets[lo] + (i - first[lo]) * rows;
    }
    tiles[2 * i] = slot;
    tiles[2 * i + 1] = pos;
  }
}

// ------------------------------------------------------------------ shrink

// v[split][position][16 group + j] = s sum_k rows[j][k] x[k] over the split's columns.  BY_PART: part p's rows are [0, r)
// of the adapter's and its columns [cols[p], cols[p + 1]) (B^T [r, N]); else rows [p r, p r + r) and all columns (A).
// A workgroup is a tile of 16 TS tokens by RC groups of 16 ranks; its waves share the columns and meet in LDS.  Both
// operands come straight from memory: the rows' A from L2, where its tiles share it, x once.
template <int TS, int RC, bool BY_PART>
__global__ __launch_bounds__(512) void adapter_shrink_kernel(Batch b, LowRank l, const uint16_t* x, int64_t ldx, int64_t cols,
                                                             const uint16_t* rows, int64_t slot_stride, int64_t ldr,
                                                             const float* scaling, float* v) {
  extern __shared__ __attribute__((aligned(16))) float red[];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  int slot;
  int64_t lo, hi;
  if (!batch_tile(b, 16 * TS, blockIdx.x, slot, lo, hi)) return;
  const int per_part = (l.groups + RC - 1) / RC, part = blockIdx.y / per_part, g0 = (blockIdx.y - part * per_part) * RC;
  const int64_t c0 = BY_PART ? l.cols[part] : 0, c1 = BY_PART ? l.cols[part + 1] : cols;
  const uint16_t* xr[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    const int64_t pos = lo + 16 * i + r < hi ? lo + 16 * i + r : hi - 1;
    xr[i] = x + (int64_t)b.order[pos] * ldx + 8 * q;
  }
  const uint16_t* ar[RC];
#pragma unroll
  for (int g = 0; g < RC; ++g) {
    const int j = 16 * (g0 + g) + r, row = (BY_PART ? 0 : part * l.rank) + (j < l.rank ? j : l.rank - 1);
    ar[g] = rows + slot * slot_stride + row * ldr + 8 * q;
  }
  v4f acc[TS][RC];
#pragma unroll
  for (int i = 0; i < TS; ++i)
#pragma unroll
    for (int g = 0; g < RC; ++g) acc[i][g] = v4f{0.f, 0.f, 0.f, 0.f};
  // this wave's columns: 32 an MFMA, U of them loaded together
  constexpr int U = TS * RC >= 8 ? 2 : 4;
  const int64_t units = (c1 - c0 + 31) / 32, shares = (int64_t)gridDim.z * waves, per = (units + shares - 1) / shares;
  const int64_t k0 = c0 + 32 * per * (blockIdx.z * waves + wv), k1 = k0 + 32 * per < c1 ? k0 + 32 * per : c1;
  for (int64_t k = k0; k < k1; k += 32 * U) {
    uint4 xv[U][TS], av[U][RC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = k + 32 * u + 8 * q < k1 ? k + 32 * u : c0 - 8 * q;  // (columns come in eights)
#pragma unroll
      for (int i = 0; i < TS; ++i) xv[u][i] = *reinterpret_cast<const uint4*>(xr[i] + at);
#pragma unroll
      for (int g = 0; g < RC; ++g) av[u][g] = *reinterpret_cast<const uint4*>(ar[g] + at);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = k + 32 * u + 8 * q < k1;
#pragma unroll
      for (int i = 0; i < TS; ++i) xv[u][i] = keep(xv[u][i], in);
#pragma unroll
      for (int g = 0; g < RC; ++g) av[u][g] = keep(av[u][g], in);
#pragma unroll
      for (int i = 0; i < TS; ++i)
#pragma unroll
        for (int g = 0; g < RC; ++g)
          acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(av[u][g]), as_bf16x8(xv[u][i]), acc[i][g], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < TS; ++i)
#pragma unroll
    for (int g = 0; g < RC; ++g) *reinterpret_cast<v4f*>(red + (((i * RC + g) * waves + wv) * 64 + lane) * 4) = acc[i][g];
  __syncthreads();
  const float s = scaling[slot];
  for (int f = wv; f < TS * RC; f += waves) {
    v4f sum = *reinterpret_cast<const v4f*>(red + ((int64_t)f * waves * 64 + lane) * 4);
    for (int w = 1; w < waves; ++w) {
      const v4f part_sum = *reinterpret_cast<const v4f*>(red + ((f * waves + w) * 64 + lane) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += part_sum[e];
    }
    const int i = f / RC, g = g0 + f % RC;
    const int64_t pos = lo + 16 * i + r;
    if (pos < hi && g < l.groups) {
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = 16 * g + 4 * q + e < l.rank ? sum[e] * s : 0.0f;
      *reinterpret_cast<v4f*>(v + (blockIdx.z * b.M + pos) * l.width() + (part * l.groups + g) * 16 + 4 * q) = sum;
    }
  }
}

// ------------------------------------------------------------------ expand

// y[t][n] += sum_j mat[n][j] v[t][j], mat [N, ldm] of the tile's adapter, j the ranks of n's part.  A workgroup is a tile
// of 16 TS tokens by `block` columns of one part (part_block: the first block of each part); v's halves wait in LDS.
template <int TS>
__global__ __launch_bounds__(256) void adapter_expand_kernel(Batch b, LowRank l, const float* v, int splits,
                                                             const uint16_t* mat, int64_t slot_stride, int64_t ldm,
                                                             int valid, uint16_t* y, int64_t ldy, int block) {
  extern __shared__ __attribute__((aligned(16))) uint16_t half[];  // [2][16 TS][stride]
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int r = lane & 15, q = lane >> 4;
  int slot;
  int64_t lo, hi;
  if (!batch_tile(b, 16 * TS, blockIdx.x, slot, lo, hi)) return;
  int part = 0, blk = blockIdx.y;
  for (; part + 1 < l.parts; ++part) {
    const int n = (int)((l.cols[part + 1] - l.cols[part] + block - 1) / block);
    if (blk < n) break;
    blk -= n;
  }
  const int64_t c0 = l.cols[part] + (int64_t)blk * block, end = l.cols[part + 1];
  const int64_t c1 = c0 + block < end ? c0 + block : end;
  const int ranks = 16 * l.groups, stride = ranks + 8;
  uint16_t* const rest = half + 16 * TS * stride;
  for (int at = t; at < 16 * TS * (ranks / 8); at += 256) {
    const int row = at / (ranks / 8), j = 8 * (at - row * (ranks / 8));
    const int64_t pos = lo + row < hi ? lo + row : hi - 1;
    float s[8] = {};
    for (int k = 0; k < splits; ++k) {
      const float* src = v + (k * b.M + pos) * l.width() + part * ranks + j;
      const v4f x0 = *reinterpret_cast<const v4f*>(src), x1 = *reinterpret_cast<const v4f*>(src + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] += x0[e];
        s[4 + e] += x1[e];
      }
    }
    *reinterpret_cast<uint4*>(half + row * stride + j) = split8(s, false);
    *reinterpret_cast<uint4*>(rest + row * stride + j) = split8(s, true);
  }
  __syncthreads();
  const uint16_t* const vf = (q < 2 ? half : rest) + r * stride + 8 * (q & 1);
  uint16_t* yr[TS];
  bool live[TS];
#pragma unroll
  for (int i = 0; i < TS; ++i) {
    const int64_t pos = lo + 16 * i + r;
    live[i] = pos < hi;
    yr[i] = y + (int64_t)b.order[live[i] ? pos : hi - 1] * ldy;
  }
  const bool wide = ldy % 4 == 0 && ((uintptr_t)y & 7) == 0;
  for (int64_t n0 = c0 + 16 * wv; n0 < c1; n0 += 64) {
    const int64_t n = n0 + r < c1 ? n0 + r : c1 - 1, col = n0 + 4 * q;
    const uint16_t* const mr = mat + slot * slot_stride + n * ldm;
    v4f acc[TS];
#pragma unroll
    for (int i = 0; i < TS; ++i) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int g = 0; g < l.groups; ++g) {
      const int j = 16 * g + 8 * (q & 1);
      uint4 m = {0, 0, 0, 0};
      if (j < valid) m = *reinterpret_cast<const uint4*>(mr + j);
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const uint4 h = *reinterpret_cast<const uint4*>(vf + 16 * i * stride + 16 * g);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(m), as_bf16x8(h), acc[i], 0, 0, 0);
      }
    }
#pragma unroll
    for (int i = 0; i < TS; ++i) {
      if (!live[i]) continue;
      if (wide && col + 4 <= c1) {
        uint2 d = *reinterpret_cast<const uint2*>(yr[i] + col);
        const uint16_t h[4] = {f32_to_bf16(u2f(d.x << 16) + acc[i][0]), f32_to_bf16(u2f(d.x & 0xFFFF0000u) + acc[i][1]),
                               f32_to_bf16(u2f(d.y << 16) + acc[i][2]), f32_to_bf16(u2f(d.y & 0xFFFF0000u) + acc[i][3])};
        *reinterpret_cast<uint2*>(yr[i] + col) = uint2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < c1) yr[i][col + e] = f32_to_bf16(bf16_to_f32(yr[i][col + e]) + acc[i][e]);
      }
    }
  }
}

// ------------------------------------------------------------------ outer products over an adapter's tokens

// sum_t big[t][c] v[t][j] over the adapter's positions of split z: to out [N, r] (OF_B: c a column of dy, j the ranks of
// its part) or out [R, K] (c a column of x, j all ranks).  A workgroup is 128 columns by RC groups; 32 tokens at a time
// go through LDS, the big matrix's read transposed (each of its bytes is read once), v's stored so.
constexpr int kOuterCols = 128, kOuterStride = kOuterCols + 16, kOuterTokens = 32, kOuterVStride = kOuterTokens + 8;
template <int RC, bool OF_B>
__global__ __launch_bounds__(256) void adapter_outer_kernel(Batch b, LowRank l, const uint16_t* big, int64_t ldb,
                                                            const float* v, int v_splits, int64_t slots, int splits,
                                                            int64_t out_cols, uint16_t* out, float* partial) {
  __shared__ __attribute__((aligned(16))) uint16_t tile[kOuterTokens * kOuterStride];
  __shared__ __attribute__((aligned(16))) uint16_t vt[2 * RC * 16 * kOuterVStride];  // [half][rank][token]
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
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int g = 0; g < RC; ++g) acc[i][g] = v4f{0.f, 0.f, 0.f, 0.f};
  const uint4 zero = {0, 0, 0, 0};
  for (int64_t p0 = lo; p0 < hi; p0 += kOuterTokens) {
    uint4 d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {  // piece: token t / 16 + 16 u, columns 8 (t % 16)
      const int64_t pos = p0 + (t >> 4) + 16 * u, c = c0 + 8 * (t & 15);
      d[u] = zero;
      if (pos < hi && c < end) d[u] = *reinterpret_cast<const uint4*>(big + (int64_t)b.order[pos] * ldb + c);
    }
    float x[RC * 2];
#pragma unroll
    for (int u = 0; u < RC * 2; ++u) {  // value: token u_all / (16 RC), rank u_all % (16 RC)
      const int at = t + 256 * u, tok = at / (16 * RC), j = at - tok * (16 * RC);
      const int64_t pos = p0 + tok;
      x[u] = 0.0f;
      if (pos < hi && g0 + j / 16 < all)
        for (int k = 0; k < v_splits; ++k) x[u] += v[(k * b.M + pos) * l.width() + gv * 16 + j];
    }
    __syncthreads();  // the last tokens' reads
#pragma unroll
    for (int u = 0; u < 2; ++u)
      *reinterpret_cast<uint4*>(tile + ((t >> 4) + 16 * u) * kOuterStride + 8 * (t & 15)) = d[u];
#pragma unroll
    for (int u = 0; u < RC * 2; ++u) {
      const int at = t + 256 * u, tok = at / (16 * RC), j = at - tok * (16 * RC);
      const uint32_t h = cvt_pk_bf16(x[u], 0.0f) & 0xFFFFu;
      const float hf = u2f(h << 16);
      vt[j * kOuterVStride + tok] = (uint16_t)h;
      vt[(RC * 16 + j) * kOuterVStride + tok] = (uint16_t)cvt_pk_bf16(__builtin_isfinite(hf) ? x[u] - hf : 0.0f, 0.0f);
    }
    __syncthreads();
    uint4 cf[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // columns 32 wv + 16 i + r, tokens 8 q .. + 7
      const uint16_t* const src = tile + (8 * q + (r >> 2)) * kOuterStride + 32 * wv + 16 * i + 4 * (r & 3);
      const s16x4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src));
      const s16x4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(src + 4 * kOuterStride));
      const uint2 y0 = __builtin_bit_cast(uint2, x0), y1 = __builtin_bit_cast(uint2, x1);
      cf[i] = uint4{y0.x, y0.y, y1.x, y1.y};
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < RC; ++g) {
        const uint4 rf = *reinterpret_cast<const uint4*>(vt + (h * RC * 16 + 16 * g + r) * kOuterVStride + 8 * q);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bf16x8_t a = as_bf16x8(OF_B ? rf : cf[i]), c = as_bf16x8(OF_B ? cf[i] : rf);
          acc[i][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, c, acc[i][g], 0, 0, 0);
        }
      }
  }
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

// Token rows of a tile: 16 while a batch has few, else 64, over which a workgroup's reads of A and B are shared.
int tile_rows(int64_t M) { return M <= 512 ? 16 : 64; }
int64_t tile_count(int64_t M, int64_t slots) {
  const int64_t rows = tile_rows(M);
  return std::min(M, ceil_div(M, rows) + std::min(slots, M));
}

// Groups a workgroup of shrink takes, and its shares of the columns: four waves each, until the launch has some 512
// workgroups or a share is 128 columns a wave.
int shrink_groups(int groups) { return groups >= 4 ? 4 : groups >= 2 ? 2 : 1; }
int shrink_splits(int64_t M, int64_t slots, int parts, int groups, int64_t cols) {
  const int64_t wgs = ceil_div(M, tile_rows(M)) * parts * ceil_div(groups, shrink_groups(groups));
  int64_t s = std::min<int64_t>(8, ceil_div(512, wgs));
  return (int)std::max<int64_t>(1, std::min(s, cols / 1024));
}

int check_batch(const char* who, int64_t M, int64_t slots, const int32_t* order, const int64_t* offsets,
                const int32_t* tiles, int64_t num_tiles) {
  MXL_CHECK_ARG(M >= 0 && M <= 0x7FFFFFFF && slots > 0 && slots <= kMaxSlots, "%s: need 0 <= M < 2^31 and 0 < slots <= %d (M=%lld slots=%lld)",
                who, kMaxSlots, (long long)M, (long long)slots);
  MXL_CHECK_ARG(num_tiles == tile_count(M, slots), "%s: %lld tiles for M=%lld slots=%lld, need %lld", who,
                (long long)num_tiles, (long long)M, (long long)slots, (long long)tile_count(M, slots));
  MXL_CHECK_ARG(M == 0 || (order && offsets && tiles), "%s: needs the batch's order, offsets and tiles", who);
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

template <bool BY_PART>
int launch_shrink(const char* who, const Batch& b, const LowRank& l, const uint16_t* x, int64_t ldx, int64_t cols,
                  const uint16_t* rows, int64_t slot_stride, int64_t ldr, const float* scaling, float* v, int splits,
                  hipStream_t s) {
  const int rc = shrink_groups(l.groups), waves = b.rows == 16 ? 8 : 4, ts = b.rows / 16;
  const dim3 grid((unsigned)b.num_tiles, (unsigned)(l.parts * ceil_div(l.groups, rc)), (unsigned)splits);
  const unsigned lds = (unsigned)(ts * rc * waves * 1024);
#define MXL_SHRINK(TS_, RC_)                                                                                          \
  if (ts == TS_ && rc == RC_)                                                                                         \
    adapter_shrink_kernel<TS_, RC_, BY_PART><<<grid, 64 * waves, lds, s>>>(b, l, x, ldx, cols, rows, slot_stride, ldr, \
                                                                           scaling, v);
  MXL_SHRINK(1, 1) MXL_SHRINK(1, 2) MXL_SHRINK(1, 4)
  MXL_SHRINK(4, 1) MXL_SHRINK(4, 2) MXL_SHRINK(4, 4)
#undef MXL_SHRINK
  return launched(who);
}

int launch_expand(const char* who, const Batch& b, const LowRank& l, const float* v, int splits, const uint16_t* mat,
                  int64_t slot_stride, int64_t ldm, int valid, uint16_t* y, int64_t ldy, hipStream_t s) {
  // (where the halves of 64 rows pass the LDS, 16 at a time)
  const int ts = b.rows == 64 && l.groups <= 32 ? 4 : 1;
  // (64 columns a workgroup where few tiles have to fill the card)
  const int block = b.num_tiles * ceil_div(l.cols[l.parts], 256) >= 1024 ? 256 : 64;
  int64_t blocks = 0;
  for (int p = 0; p < l.parts; ++p) blocks += ceil_div(l.cols[p + 1] - l.cols[p], block);
  MXL_CHECK_ARG(blocks <= 0xFFFF, "%s: too many columns", who);
  const dim3 grid((unsigned)(b.num_tiles * (b.rows / (16 * ts))), (unsigned)blocks);
  const unsigned lds = (unsigned)(2 * 16 * ts * (16 * l.groups + 8) * 2);
  if (ts == 1) adapter_expand_kernel<1><<<grid, 256, lds, s>>>(b, l, v, splits, mat, slot_stride, ldm, valid, y, ldy, block);
  else adapter_expand_kernel<4><<<grid, 256, lds, s>>>(b, l, v, splits, mat, slot_stride, ldm, valid, y, ldy, block);
  return launched(who);
}

// Shares of an adapter's tokens in the outer products: some 512 tokens each.
int outer_splits(int64_t M) { return (int)std::min<int64_t>(16, std::max<int64_t>(1, ceil_div(M, 512))); }

template <bool OF_B>
int launch_outer(const char* who, const Batch& b, const LowRank& l, int64_t slots, const uint16_t* big, int64_t ldb,
                 int64_t cols, const float* v, int v_splits, uint16_t* out, float* partial, hipStream_t s) {
  const int splits = outer_splits(b.M), all = OF_B ? l.groups : l.parts * l.groups, rc = shrink_groups(all);
  int64_t blocks = 0;
  if (OF_B)
    for (int p = 0; p < l.parts; ++p) blocks += ceil_div(l.cols[p + 1] - l.cols[p], kOuterCols);
  else
    blocks = ceil_div(cols, kOuterCols);
  MXL_CHECK_ARG(slots * splits <= 0xFFFF, "%s: too many adapters", who);
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(all, rc), (unsigned)(slots * splits));
#define MXL_OUTER(RC_)                                                                                             \
  if (rc == RC_)                                                                                                   \
    adapter_outer_kernel<RC_, OF_B><<<grid, 256, 0, s>>>(b, l, big, ldb, v, v_splits, slots, splits, cols, out, partial);
  MXL_OUTER(1) MXL_OUTER(2) MXL_OUTER(4)
#undef MXL_OUTER
  int rc2 = launched(who);
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
  const int64_t N = l.cols[l.parts], out = outer_splits(M) > 1 ? outer_splits(M) : 0;
  Pieces p{base};
  GradScratch g;
  g.bt = p.take(slots * l.rank * N * 2);
  g.at = p.take(slots * K * l.width() * 2);
  g.dv = p.take(shrink_splits(M, slots, l.parts, l.groups, N / l.parts) * M * l.width() * 4);
  g.partial = p.take(out * slots * l.rank * std::max(N, l.parts * K) * 4);
  g.bytes = p.used;
  return g;
}

}  // namespace

extern "C" int64_t mxl_adapter_tile_count(int64_t M, int64_t slots) {
  return M <= 0 || slots <= 0 ? 0 : tile_count(M, slots);
}

extern "C" int mxl_adapter_tiles(const int64_t* offsets, int64_t M, int64_t slots, int32_t* tiles, int64_t num_tiles,
                                 void* stream) {
  const char* who = "mxl_adapter_tiles";
  MXL_CHECK_ARG(M >= 0 && M <= 0x7FFFFFFF && slots > 0 && slots <= kMaxSlots, "%s: need 0 <= M < 2^31 and 0 < slots <= %d", who, kMaxSlots);
  if (M == 0) return MXL_OK;
  MXL_CHECK_ARG(offsets && tiles && num_tiles == tile_count(M, slots), "%s: needs %lld tiles", who,
                (long long)tile_count(M, slots));
  adapter_tiles_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(offsets, (int)slots, tile_rows(M), (int)num_tiles, tiles);
  return launched(who);
}

extern "C" int64_t mxl_adapter_v_floats(int64_t M, int64_t K, int64_t slots, int64_t parts, int64_t rank) {
  if (M <= 0 || K <= 0 || slots <= 0 || parts <= 0 || rank <= 0) return 0;
  const int groups = (int)((rank + 15) / 16);
  return shrink_splits(M, slots, (int)parts, groups, K) * M * parts * groups * 16;
}

extern "C" int mxl_adapter_apply(const void* x, int64_t M, int64_t K, int64_t ldx, const void* a, const void* b,
                                 const float* scaling, int64_t slots, int64_t parts, const int64_t* cols, int64_t rank,
                                 const int32_t* order, const int64_t* offsets, const int32_t* tiles, int64_t num_tiles,
                                 float* v, int64_t v_floats, void* y, int64_t ldy, void* stream) {
  const char* who = "mxl_adapter_apply";
  LowRank l;
  int rc = check_batch(who, M, slots, order, offsets, tiles, num_tiles);
  if (rc == MXL_OK) rc = make_low_rank(who, parts, cols, rank, K, l);
  if (rc != MXL_OK || M == 0) return rc;
  const int64_t N = l.cols[l.parts];
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0 && ldy >= N, "%s: need ldx >= K, a multiple of 8, and ldy >= N", who);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)a | (uintptr_t)b | (uintptr_t)v) & 15) == 0, "%s: x, a, b and v must be 16-byte aligned", who);
  MXL_CHECK_ARG(v_floats >= mxl_adapter_v_floats(M, K, slots, parts, rank), "%s: v holds %lld floats, needs %lld", who,
                (long long)v_floats, (long long)mxl_adapter_v_floats(M, K, slots, parts, rank));
  const Batch batch{order, offsets, tiles, (int)num_tiles, tile_rows(M), M};
  const int splits = shrink_splits(M, slots, l.parts, l.groups, K);
  const int64_t R = parts * rank;
  rc = launch_shrink<false>(who, batch, l, (const uint16_t*)x, ldx, K, (const uint16_t*)a, R * K, K, scaling, v, splits,
                            (hipStream_t)stream);
  if (rc != MXL_OK) return rc;
  return launch_expand(who, batch, l, v, splits, (const uint16_t*)b, N * rank, rank, l.rank, (uint16_t*)y, ldy,
                       (hipStream_t)stream);
}

extern "C" int64_t mxl_adapter_grad_workspace_bytes(int64_t M, int64_t K, int64_t slots, int64_t parts,
                                                    const int64_t* cols, int64_t rank) {
  LowRank l;
  if (M <= 0 || slots <= 0 || make_low_rank("mxl_adapter_grad_workspace_bytes", parts, cols, rank, K, l) != MXL_OK) return 0;
  return grad_scratch(nullptr, M, K, slots, l).bytes;
}

extern "C" int mxl_adapter_grad(const void* x, int64_t M, int64_t K, int64_t ldx, const void* dy, int64_t lddy,
                                const void* a, const void* b, const float* scaling, int64_t slots, int64_t parts,
                                const int64_t* cols, int64_t rank, const int32_t* order, const int64_t* offsets,
                                const int32_t* tiles, int64_t num_tiles, const float* v, int64_t v_floats, void* dx,
                                int64_t lddx, void* da, void* db, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_adapter_grad";
  LowRank l;
  int rc = check_batch(who, M, slots, order, offsets, tiles, num_tiles);
  if (rc == MXL_OK) rc = make_low_rank(who, parts, cols, rank, K, l);
  if (rc != MXL_OK || M == 0) return rc;
  const int64_t N = l.cols[l.parts], R = parts * rank;
  MXL_CHECK_ARG(N % 8 == 0, "%s: need N %% 8 == 0 (N=%lld)", who, (long long)N);
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0 && lddy >= N && lddy % 8 == 0 && (!dx || lddx >= K),
                "%s: need ldx >= K, lddy >= N, multiples of 8, and lddx >= K", who);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)dy | (uintptr_t)a | (uintptr_t)b | (uintptr_t)v | (uintptr_t)da | (uintptr_t)db) & 15) == 0,
                "%s: operands must be 16-byte aligned", who);
  MXL_CHECK_ARG(v_floats >= mxl_adapter_v_floats(M, K, slots, parts, rank), "%s: v holds %lld floats", who, (long long)v_floats);
  const GradScratch g = grad_scratch((uint8_t*)workspace, M, K, slots, l);
  MXL_CHECK_ARG(workspace && workspace_bytes >= g.bytes && ((uintptr_t)workspace & 255) == 0,
                "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who, (long long)g.bytes,
                (long long)workspace_bytes);
  hipStream_t s = (hipStream_t)stream;
  const Batch batch{order, offsets, tiles, (int)num_tiles, tile_rows(M), M};
  const int v_splits = shrink_splits(M, slots, l.parts, l.groups, K);
  const int dv_splits = shrink_splits(M, slots, l.parts, l.groups, N / l.parts);
  if (db) {
    rc = launch_outer<true>(who, batch, l, slots, (const uint16_t*)dy, lddy, N, v, v_splits, (uint16_t*)db,
                            (float*)g.partial, s);
    if (rc != MXL_OK) return rc;
  }
  if (!da && !dx) return MXL_OK;
  // B [N, r] -> [r, N]
  adapter_transpose_kernel<<<dim3((unsigned)ceil_div(l.rank, 32), (unsigned)ceil_div(N, 32), (unsigned)slots), 256, 0, s>>>(
      (const uint16_t*)b, N, l.rank, 1, (int)N, (int)N, (uint16_t*)g.bt);
  rc = launched(who);
  if (rc == MXL_OK)
    rc = launch_shrink<true>(who, batch, l, (const uint16_t*)dy, lddy, N, (const uint16_t*)g.bt, l.rank * N, N, scaling,
                             (float*)g.dv, dv_splits, s);
  if (rc == MXL_OK && da)
    rc = launch_outer<false>(who, batch, l, slots, (const uint16_t*)x, ldx, K, (const float*)g.dv, dv_splits,
                             (uint16_t*)da, (float*)g.partial, s);
  if (rc == MXL_OK && dx) {
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
      rc = launch_expand(who, batch, one, (const float*)g.dv, dv_splits, (const uint16_t*)g.at, K * l.width(), l.width(),
                         one.rank, (uint16_t*)dx, lddx, s);
  }
  return rc;
}
