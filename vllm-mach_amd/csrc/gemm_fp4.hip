// Products of MXFP4 activations and weights on gfx950, dense and MoE-grouped: y = A W^T with E2M1
// codes and E8M0 scales per 32 on both sides, fp32 sums, bf16 out.
//
// The scaled MFMA multiplies 16 x 16 x 128 with a scale byte per lane and operand: lane 16 q + r supplies
// the 16 bytes of K [32 q, + 32) -- one scale block -- of row r of either operand.  The weights take its
// A operand and the activations its B operand, so a lane holds four consecutive output columns of one row.
#include <algorithm>
#include <type_traits>

#include "fp4.h"
#include "gemm_common.h"

namespace mxl {

int moe_reduce_by_route(const char* who, const void* routed_output, const float* topk_weights, const int32_t* topk_ids,
                        int64_t T, int64_t topk, int64_t E, int64_t H, void* out, void* stream);  // (moe.hip)

// c += W A^T over a K128 slice whose scales are byte J of sw and byte JA of sa.
template <int J, int JA>
__device__ __forceinline__ v4f mfma_fp4(const uint4& w, const uint4& a, v4f c, uint32_t sw, uint32_t sa) {
  const v8i x = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const v8i y = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, kE2M1, kE2M1, J, (int)sw, JA, (int)sa);
}

// ------------------------------------------------------------ few rows: weights through registers
//
// Decode-sized products are their weights' way from memory.  A workgroup owns WN n-tiles; wave (wn, wk) loads its
// n-tile's super-tiles [wk CNT, + CNT) into registers at once: up to 21 KiB a wave and all of a launch's weights in
// flight together.  Under those loads the workgroup produces its activation rows in LDS, in fragment order --
// copied codes, or bf16 rows quantized here (PROD 1: a lane holds a whole 32-block, so its amax needs no exchange)
// -- and then multiplies, 16 rows at a time, the weights staying in their registers.  The wk partials of an
// n-tile meet in LDS and are summed in order.
//
// Grouped: blockIdx.y is an expert (or, with fewer routes than experts, the y-th that has any), so each expert's
// weights are read once whatever its rows.  SWIGLU (an expert's gate/up product): the workgroup's n-tiles are two
// of gate and the same two of up, and the epilogue quantizes the 32 columns' bf16(bf16(silu(g)) u) in place of
// storing gate and up.
// Cold weights: 1 x 2048 x 2048 3.9 us; w13 and w2 of 64 tokens, top 8 of 256 experts (K = 2048, I = 512) 52 and 24 us,
// 4.8 and 5.2 TB/s of weights, the rate of a large copy (5.2).
//
// kRoutes: a few routes as they come, their experts in row_index and route r's activation row r / row_div: no sort.
enum Fp4Unit : int { kExperts = 0, kHitExperts = 1, kRoutes = 2 };
struct Fp4Stream {
  int WN, WK;
  int E, unit;            // grouped: experts (0: dense), and what blockIdx.y counts (Fp4Unit)
  const uint16_t* x;      // PROD 1: bf16 rows, stride ldx
  int64_t ldx;
  uint32_t carry;         // the scale rule of PROD 1 and SWIGLU
  uint8_t* codes;         // SWIGLU: [rows, N / 4] and [rows, N / 64], N = 2 I
  uint8_t* scales;
};

constexpr int kFp4StreamCnt = 5, kFp4StreamWaves = 8;

template <int CNT, int PROD, bool SWIGLU>
__global__ __launch_bounds__(64 * kFp4StreamWaves) void fp4_stream_kernel(GemmParams p, Fp4Stream g) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), threads = blockDim.x;
  const int r = lane & 15, q = lane >> 4;
  const int T = (int)(p.K / 128), KT = (int)p.KT, WK = g.WK, wn = wv / WK, wk = wv - wn * WK;
  const int ntiles = (int)((p.N + 15) / 16);
  int64_t lo = 0, hi = p.M;
  int e = blockIdx.y;
  auto within = [&](int64_t row) -> int { return row < 0 ? 0 : row < p.M ? (int)row : (int)p.M; };
  if (g.E) {
    if (g.unit == kRoutes) {
      e = p.row_index[blockIdx.y];
      if (e < 0 || e >= g.E) return;
      lo = blockIdx.y;
      hi = lo + 1;
    } else if (g.unit == kHitExperts) {  // the blockIdx.y-th expert with rows: four experts a lane, whose offsets load together
      int left = blockIdx.y, found = -1;
      for (int e0 = 0; e0 < g.E && found < 0; e0 += 256) {
        const int x = e0 + 4 * lane;
        int64_t off[5];
#pragma unroll
        for (int j = 0; j < 5; ++j) off[j] = p.expert_offsets[x + j < g.E ? x + j : g.E];
        uint32_t some = 0;
        int before = 0, n = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool is = off[j + 1] > off[j];
          const uint64_t all = __ballot(is);
          some |= is ? 1u << j : 0u;
          before += __popcll(all & ((1ull << lane) - 1));
          n += __popcll(all);
        }
        if (left < n) {
          int k = left - before;
          const int who = __builtin_ctzll(__ballot(k >= 0 && k < __popc(some)));
          for (; k > 0 && some; --k) some &= some - 1;
          const int j = __builtin_ctz(some | 8u);
          int64_t first = off[0], end = off[1];
#pragma unroll
          for (int i = 1; i < 4; ++i) {
            first = j == i ? off[i] : first;
            end = j == i ? off[i + 1] : end;
          }
          found = __builtin_amdgcn_readlane(x + j, who);
          lo = __builtin_amdgcn_readlane(within(first), who);
          hi = __builtin_amdgcn_readlane(within(end), who);
        }
        left -= n;
      }
      if (found < 0) return;
      e = found;
    } else {
      lo = within(p.expert_offsets[e]);
      hi = within(p.expert_offsets[e + 1]);
    }
    if (lo >= hi) return;
  }
  // n-tile: SWIGLU's second half of the waves holds up
  int nt = blockIdx.x * g.WN + wn;
  if (SWIGLU) nt = blockIdx.x * 2 + (wn & 1) + (wn >> 1) * (ntiles / 2);
  const bool live = nt < ntiles;
  uint4 w[CNT][4];
  uint32_t sw[CNT];
  const int s0 = wk * CNT;
  if (live) {
    const uint8_t* wp = p.w + e * p.w_expert_stride + ((int64_t)nt * KT + s0) * 4096 + lane * 16;
    const uint8_t* sp = static_cast<const uint8_t*>(p.sw) + e * p.sw_expert_stride + ((int64_t)nt * KT + s0) * 256 + lane * 4;
#pragma unroll
    for (int i = 0; i < CNT; ++i)
      if (s0 + i < KT) {
        sw[i] = *reinterpret_cast<const uint32_t*>(sp + i * 256);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = *reinterpret_cast<const uint4*>(wp + i * 4096 + j * 1024);
      }
  }
  uint8_t* const ac = lds;                                       // codes: [T][64 lanes] x 16 bytes
  uint8_t* const as = ac + T * 1024;                            // scales: [KT][64 lanes] x 4 slices
  float* const red = reinterpret_cast<float*>(as + KT * 256);   // [WN][WK][64 lanes] x 4
  const int blocks = (int)(p.K / 32);

  for (int64_t row0 = lo; row0 < hi; row0 += 16) {
    const int rows = (int)(hi - row0 < 16 ? hi - row0 : 16), items = rows * blocks;
    if (row0 != lo) __syncthreads();  // the last block's reads of LDS
    // item: block b of row rr, rows fastest (at / rows by the reciprocal: at rows < 2^32); U of them a batch, so that
    // their loads wait together
    constexpr int U = 2;
    const uint32_t inv = rows > 1 ? (uint32_t)(0x100000000ull / (uint32_t)rows) + 1 : 0;
    uint4 v[U][PROD == 0 ? 1 : 4];
    uint32_t s[U];
    int rr[U], b[U];
    auto load = [&](int at0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        int at = at0 + u * threads + t;
        at = at < items ? at : items - 1;  // (past the end: the last again)
        b[u] = rows > 1 ? (int)__umulhi((uint32_t)at, inv) : at;
        rr[u] = at - b[u] * rows;
        int ar = (int)row0 + rr[u];  // (32-bit offsets, of codes in pieces of 16 bytes: the host admits no rows past them)
        if (g.E) {
          if (p.row_index) ar = (g.unit == kRoutes ? ar : p.row_index[ar]) / p.row_div;
          ar = ar < 0 ? 0 : ar < (int)p.a_rows ? ar : (int)p.a_rows - 1;
        }
        if constexpr (PROD == 0) {
          const uint32_t off = (uint32_t)ar * blocks + b[u];
          v[u][0] = reinterpret_cast<const uint4*>(p.a)[off];
          s[u] = static_cast<const uint8_t*>(p.sa)[off];
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            v[u][i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(g.x) +
                                                      ((uint32_t)ar * (uint32_t)(2 * g.ldx) + 64 * b[u] + 16 * i));
        }
      }
    };
    auto put = [&] {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint4 c = v[u][0];
        if constexpr (PROD == 1) {
          uint32_t d[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            d[4 * i] = v[u][i].x; d[4 * i + 1] = v[u][i].y; d[4 * i + 2] = v[u][i].z; d[4 * i + 3] = v[u][i].w;
          }
          s[u] = scale_e2m1(amax_bf16_bits<16, false>(d), g.carry);
          c = uint4{codes_e2m1(d, s[u]), codes_e2m1(d + 4, s[u]), codes_e2m1(d + 8, s[u]), codes_e2m1(d + 12, s[u])};
        }
        const int sl = b[u] >> 2, frag = rr[u] + 16 * (b[u] & 3);
        *reinterpret_cast<uint4*>(ac + (sl * 64 + frag) * 16) = c;
        as[((sl >> 2) * 64 + frag) * 4 + (sl & 3)] = (uint8_t)s[u];
      }
    };
    for (int at0 = 0; at0 < items; at0 += U * threads) {
      load(at0);
      put();
    }
    __syncthreads();
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    // (fragment lanes of rows past the last hold whatever LDS held: their outputs alone, not stored)
    if (live) {
#pragma unroll
      for (int i = 0; i < CNT; ++i)
        if (s0 + i < KT) {
          const uint32_t sa = *reinterpret_cast<const uint32_t*>(as + ((s0 + i) * 64 + lane) * 4);
          auto slice = [&](auto J) {
            constexpr int j = decltype(J)::value;
            const int sl = 4 * (s0 + i) + j;
            if (sl < T) acc = mfma_fp4<j, j>(w[i][j], *reinterpret_cast<const uint4*>(ac + (sl * 64 + lane) * 16), acc, sw[i], sa);
          };
          slice(std::integral_constant<int, 0>{});
          slice(std::integral_constant<int, 1>{});
          slice(std::integral_constant<int, 2>{});
          slice(std::integral_constant<int, 3>{});
        }
    }
    if (SWIGLU || WK > 1) {
      *reinterpret_cast<v4f*>(red + (wv * 64 + lane) * 4) = acc;
      __syncthreads();
    }
    // the sum of the partials of the workgroup's n-tile n, of fragment lane l
    auto total = [&](int n, int l) -> v4f {
      v4f v = *reinterpret_cast<const v4f*>(red + (n * WK * 64 + l) * 4);
      for (int k = 1; k < WK; ++k) {
        const v4f u = *reinterpret_cast<const v4f*>(red + ((n * WK + k) * 64 + l) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += u[i];
      }
      return v;
    };
    if constexpr (SWIGLU) {
      // thread: row rr, columns 8 sub .. + 7 of the 32
      const int rr = t >> 2, sub = t & 3;
      if (rr < 16) {  // (the first wave)
        float gate[8], up[8], v[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int l = 16 * (2 * (sub & 1) + h) + rr;
          const v4f a = total(sub >> 1, l), b = total(2 + (sub >> 1), l);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            gate[4 * h + i] = bf16_round(a[i]);
            up[4 * h + i] = bf16_round(b[i]);
          }
        }
        swiglu8<kFloorCarry175>(gate, up, v);
        uint32_t d[4], c;
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = cvt_pk_bf16(v[2 * i], v[2 * i + 1]);
        const uint32_t s = quant_e2m1_x4(d, g.carry, c);
        if (rr < rows) {
          const int64_t at = (row0 + rr) * (p.N / 64) + blockIdx.x;
          reinterpret_cast<uint32_t*>(g.codes)[at * 4 + sub] = c;
          if (sub == 0) g.scales[at] = (uint8_t)s;
        }
      }
    } else if (live && wk == 0) {
      const int64_t col = (int64_t)nt * 16 + 4 * q;
      const v4f v = WK > 1 ? total(wn, lane) : acc;
      if (r < rows) {
        uint16_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = out_bits_fp4(v[i], p.bias, col + i < p.N ? col + i : 0);
        uint16_t* dst = p.out + (row0 + r) * p.ldc + col;
        if (col + 4 <= p.N && p.ldc % 4 == 0 && ((uintptr_t)p.out & 7) == 0) {
          *reinterpret_cast<uint2*>(dst) = uint2{h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16};
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (col + i < p.N) dst[i] = h[i];
        }
      }
    }
  }
}

struct Fp4StreamPlan {
  int cnt, WK, WN, lds;
  int64_t groups;  // workgroups over the n-tiles
};

// The waves' share of K and of the n-tiles: as many super-tiles a wave as still leave two waves a CU, and about four
// waves a workgroup (graph-timed, us, super-tiles x n-tiles a workgroup: 1 x 2048 x 2048 1 x 1 3.8, 2 x 1 3.9, 4 x 4
// 4.9; 1 x 17408 x 5120 2 x 1 15.6, 3 x 1 13.9, 5 x 2 13.1, 5 x 4 17.5; 64 tokens of 256 experts of 1024 x 2048 1 x 2
// 52.0, 4 x 4 46.6, 4 x 6 50.9: a workgroup's waves wait for each other twice).  False where the activations do not
// fit in LDS or K is past what eight waves hold.
static bool fp4_stream_plan(int64_t N, int64_t K, int64_t units, bool swiglu, Fp4StreamPlan& pl) {
  const int64_t KT = (K + kTileK - 1) / kTileK, ntiles = (N + 15) / 16;
  const int waves_max = swiglu ? kFp4StreamWaves / 4 : kFp4StreamWaves;  // over K
  pl.WK = 0;
  for (int cnt = kFp4StreamCnt; cnt >= 1; --cnt) {
    const int64_t wk = (KT + cnt - 1) / cnt;
    if (wk > waves_max) break;
    pl.WK = (int)wk;
    if (ntiles * units * wk >= 2 * cu_count()) break;
  }
  if (pl.WK == 0) return false;
  pl.cnt = (int)((KT + pl.WK - 1) / pl.WK);
  pl.WN = swiglu || pl.WK == 1 ? 4 : pl.WK >= 4 ? 1 : 4 / pl.WK;
  pl.groups = swiglu ? N / 64 : (ntiles + pl.WN - 1) / pl.WN;
  const int64_t lds = K / 128 * 1024 + KT * 256 + (pl.WK > 1 || swiglu ? pl.WK * pl.WN * 1024 : 0);
  pl.lds = (int)lds;
  return lds <= 160 * 1024;
}

template <int PROD, bool SWIGLU>
static hipError_t launch_fp4_stream(const Fp4StreamPlan& pl, const GemmParams& p, Fp4Stream g, int64_t units, hipStream_t s) {
  g.WN = pl.WN;
  g.WK = pl.WK;
  const dim3 grid((unsigned)pl.groups, (unsigned)units), block(64 * pl.WK * pl.WN);
#define MXL_FP4_CNT(C_) \
  if (pl.cnt == C_) hipLaunchKernelGGL((fp4_stream_kernel<C_, PROD, SWIGLU>), grid, block, pl.lds, s, p, g);
  MXL_FP4_CNT(1)
  MXL_FP4_CNT(2)
  MXL_FP4_CNT(3)
  MXL_FP4_CNT(4)
  MXL_FP4_CNT(5)
#undef MXL_FP4_CNT
  return hipGetLastError();
}

// Dense rows that the streaming kernel takes, up to 16.  Each workgroup produces all of them, so that with
// quantization its cost grows with rows x K and with the workgroups a CU runs one after the other (us, fused | quantizer
// and product: 16 x 2048 x 2048 5.6 | 6.6, 4 x 2560 x 9216 8.8 | 9.2, 8 rows 10.6 | 9.9, 2 x 17408 x 5120 13.7 | 15.0, 4
// rows 16.2 | 15.1).  Of codes, weights of more than two workgroups a CU run better in tiles (16 x 17408 x 5120
// 18.1 | 13.5; 16 x 2560 x 9216 10.0 | 10.4).
constexpr int64_t kFp4StreamRows = 16;
static bool fp4_dense_streams(int64_t M, int64_t N, int64_t K, bool quant, Fp4StreamPlan& pl) {
  if (M > kFp4StreamRows || !fp4_stream_plan(N, K, 1, false, pl)) return false;
  const int64_t cus = cu_count();
  return quant ? M * K * ((pl.groups + cus - 1) / cus) <= 48 * 1024 : pl.groups <= 2 * cus;
}

// Grouped products of few rows an expert (routes / experts): 8, or 16 of a short K, whose rows cost less to produce
// (us, streamed | 128-row tiles, 256 experts, top 8: w13 of K = 2048 at 128 / 256 tokens 51.6 / 55.0 | 54.2 / 54.5; w2
// of K = 512 at 256 / 400 27.8 / 32.3 | 36.7 / 38.5).  With the quantization and the SwiGLU producer in the launch
// (which saves two, 6 us) w13 takes 55.9 / 61.6.
static bool fp4_grouped_streams(int64_t routed_rows, int64_t num_experts, int64_t N, int64_t K, bool swiglu,
                                Fp4StreamPlan& pl) {
  return routed_rows < (K <= 1024 && !swiglu ? 16 : 8) * num_experts &&
         fp4_stream_plan(N, K, std::min(routed_rows, num_experts), swiglu, pl);
}

// ------------------------------------------------------------ many experts, operands past 4 GiB

// The grouped product where neither the streaming kernel nor the tiles run (more than 1024 experts with many rows
// each, operands past their 32-bit offsets), with 64-bit offsets.  One wavefront: the 16 x 16 tile of output rows row0 .. (below row_hi) and n-tile nt, all of K.
// a_row(row): the activation row of an output row.
template <class Row>
__device__ __forceinline__ void fp4_tile(const GemmParams& p, const uint8_t* w, const uint8_t* sw, int64_t nt,
                                         int64_t row0, int64_t row_hi, int lane, Row&& a_row) {
  const int r = lane & 15, q = lane >> 4;
  const int64_t row = row0 + r < row_hi ? row0 + r : row_hi - 1, ar = a_row(row);
  const uint8_t* a = p.a + ar * p.lda + 16 * q;
  const uint8_t* sa = static_cast<const uint8_t*>(p.sa) + ar * (p.K / 32) + q;
  w += nt * p.KT * 4096 + lane * 16;
  sw += nt * p.KT * 256 + lane * 4;
  const int T = (int)(p.K / 128);
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int t = 0; t < T; ++t) {
    const uint4 wv = *reinterpret_cast<const uint4*>(w + t * 1024), av = *reinterpret_cast<const uint4*>(a + t * 64);
    const uint32_t s = *reinterpret_cast<const uint32_t*>(sw + (t >> 2) * 256) >> (8 * (t & 3));
    acc = mfma_fp4<0, 0>(wv, av, acc, s, sa[4 * t]);
  }
  if (row0 + r >= row_hi) return;
  const int64_t col = nt * 16 + 4 * q;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.N) p.out[row * p.ldc + col + e] = out_bits_fp4(acc[e], p.bias, col + e);
}

__global__ __launch_bounds__(256) void fp4_grouped_kernel(GemmParams p) {
  const int64_t nt = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), e = blockIdx.y;
  if (nt * 16 >= p.N) return;
  const int64_t lo = p.expert_offsets[e] > 0 ? p.expert_offsets[e] : 0;
  const int64_t hi = p.expert_offsets[e + 1] < p.M ? p.expert_offsets[e + 1] : p.M;
  for (int64_t row0 = lo; row0 < hi; row0 += 16)
    fp4_tile(p, p.w + e * p.w_expert_stride, static_cast<const uint8_t*>(p.sw) + e * p.sw_expert_stride, nt, row0, hi,
             threadIdx.x & 63,
             [&](int64_t row) {
               const int64_t at = p.row_index ? p.row_index[row] / p.row_div : row;
               return at < 0 ? 0 : at < p.a_rows ? at : p.a_rows - 1;
             });
}

}  // namespace mxl

// ------------------------------------------------------------------- C ABI

using namespace mxl;

extern "C" int64_t mxl_tiled_weight_bytes(int64_t N, int64_t K, int fmt);
extern "C" int64_t mxl_tiled_scale_bytes(int64_t N, int64_t K);

constexpr int kFp4MaxK = 1 << 22;

static int check_operands(const char* who, const void* a, const void* sa, const void* w, const void* sw, int64_t N,
                          int64_t K, const void* out) {
  MXL_CHECK_ARG(N > 0 && K > 0 && K % 128 == 0 && K <= kFp4MaxK, "%s: need N > 0, 0 < K <= %d, K %% 128 == 0 (N=%lld K=%lld)",
                who, kFp4MaxK, (long long)N, (long long)K);
  MXL_CHECK_ARG((((uintptr_t)a | (uintptr_t)w) & 15) == 0, "%s: a and w must be 16-byte aligned", who);
  MXL_CHECK_ARG((((uintptr_t)sa | (uintptr_t)sw) & 3) == 0, "%s: the scales must be 4-byte aligned", who);
  MXL_CHECK_ARG(((uintptr_t)out & 1) == 0, "%s: misaligned output", who);
  return MXL_OK;
}

// Whether bf16 rows [rows, K] of stride ldx lie within the 32-bit byte offsets of the streaming kernel's producer.
static bool fp4_rows_reach(int64_t rows, int64_t ldx, int64_t K) {
  return rows <= 1 || rows - 1 <= ((int64_t(1) << 31) - K) / ldx;
}

// A stage of the 2 x 2-wave tiles is 128 bytes of a row, whatever its format, and its two MFMAs of a K128 slice
// of MXFP4 take the time of one of 8-bit activations, so the plan is the time model's of K / 2 columns.  Its costs (and
// the hybrid's borders) are fitted to 8-bit stages, not to these: a 128 x 64 stage measures 0.41 us here (512 x 2560 x
// 9216, 36 stages whole-K in 19.8) and 0.289 there.  Splits end on 1024 columns, two super-tiles.
static WideConfig fp4_tiles_config(int64_t M, int64_t N, int64_t K) {
  const int64_t KT = (K + kTileK - 1) / kTileK;
  WideConfig c = wide_tiles_config(M, N, (K / 2 + 127) / 128 * 128, false);
  c.kt_per_split = 2 * c.kt_per_split < KT ? 2 * c.kt_per_split : KT;  // super-tiles of half the stages
  c.S = (int)((KT + c.kt_per_split - 1) / c.kt_per_split);
  if (c.dp_tiles > 0) {
    c.kt2 = 2 * c.kt2 < KT ? 2 * c.kt2 : KT;
    c.S2 = (int)((KT + c.kt2 - 1) / c.kt2);
  }
  return c;
}

// (the codes' offsets are those of K / 2 bytes a row; a weight's scales, 256 bytes a super-tile of 512 columns, are
// indexed in 32 bits)
static bool fp4_tiles_eligible(int64_t M, int64_t N, int64_t K) {
  return wide_tiles_eligible(M, N, K / 2, false) && ((N + 15) / 16) * ((K + kTileK - 1) / kTileK) <= (int64_t(1) << 24);
}

static GemmParams fp4_params(const void* a, const void* sa, const void* w, const void* sw, int64_t N, int64_t K,
                             void* out, int64_t ldc) {
  GemmParams p{};
  p.a = (const uint8_t*)a; p.sa = sa; p.w = (const uint8_t*)w; p.sw = sw; p.out = (uint16_t*)out;
  p.lda = K / 2; p.ldc = ldc; p.N = N; p.K = K; p.KT = (K + kTileK - 1) / kTileK;
  p.row_div = 1; p.S = 1;
  return p;
}

static int launch_status(hipError_t e, const char* who) {
  if (e == hipSuccess) return MXL_OK;
  set_error("%s: launch failed: %s", who, hipGetErrorString(e));
  return MXL_EHIP;
}

// Rows of one launch of the tiles: operands below 4 GiB, whole 256-row blocks.
static int64_t fp4_slab_rows(int64_t M, int64_t K) {
  const int64_t most = ((int64_t(1) << 32) / (K / 2) - 1) / 256 * 256;
  return M < most ? M : most;
}

extern "C" int64_t mxl_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  Fp4StreamPlan pl;
  if (M <= 0 || N <= 0 || K <= 0 || K % 128 || K > kFp4MaxK || fp4_dense_streams(M, N, K, false, pl)) return 0;
  const int64_t rows = fp4_slab_rows(M, K), rest = M % rows;
  const int64_t need = wide_workspace_bytes(fp4_tiles_config(rows, N, K), rows, N);
  return rest ? std::max(need, wide_workspace_bytes(fp4_tiles_config(rest, N, K), rest, N)) : need;
}

extern "C" int mxl_mxfp4_gemm(const void* a, const void* sa, int64_t M, const void* w_tiled, const void* sw_tiled,
                              int64_t N, int64_t K, const void* bias, void* out, int64_t ldc, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_mxfp4_gemm";
  const int rc = check_operands(who, a, sa, w_tiled, sw_tiled, N, K, out);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(M >= 0 && ldc >= N, "%s: need M >= 0 and ldc >= N (M=%lld ldc=%lld)", who, (long long)M, (long long)ldc);
  if (M == 0) return MXL_OK;
  hipStream_t s = (hipStream_t)stream;
  GemmParams p = fp4_params(a, sa, w_tiled, sw_tiled, N, K, out, ldc);
  p.bias = (const uint16_t*)bias;
  Fp4StreamPlan pl;
  if (fp4_dense_streams(M, N, K, false, pl)) {
    p.M = p.a_rows = M;
    return launch_status(launch_fp4_stream<0, false>(pl, p, Fp4Stream{}, 1, s), who);
  }
  MXL_CHECK_ARG(fp4_tiles_eligible(fp4_slab_rows(M, K), N, K), "%s: too large (N=%lld K=%lld)", who, (long long)N,
                (long long)K);
  const int64_t need = mxl_mxfp4_gemm_workspace_bytes(M, N, K);
  MXL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "%s: needs a 16-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  const int64_t slab = fp4_slab_rows(M, K);
  for (int64_t row = 0; row < M; row += slab) {
    GemmParams q = p;
    q.M = q.a_rows = std::min(slab, M - row);
    q.a = p.a + row * p.lda;
    q.sa = static_cast<const uint8_t*>(p.sa) + row * (K / 32);
    q.out = p.out + row * ldc;
    q.partial = (float*)workspace;
    const WideConfig c = fp4_tiles_config(q.M, N, K);
    q.S = c.S;
    const int st = launch_status(launch_gemm_wide(kE2M1, false, c, q, 0, s), who);
    if (st != MXL_OK) return st;
  }
  return MXL_OK;
}

extern "C" int mxl_mxfp4_quant_gemm_supported(int64_t M, int64_t N, int64_t K) {
  Fp4StreamPlan pl;
  return M > 0 && N > 0 && K > 0 && K % 128 == 0 && fp4_dense_streams(M, N, K, true, pl);
}

extern "C" int mxl_mxfp4_quant_gemm(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, const void* w_tiled,
                                    const void* sw_tiled, int64_t N, const void* bias, void* out, int64_t ldc,
                                    void* stream) {
  const char* who = "mxl_mxfp4_quant_gemm";
  const int rc = check_operands(who, x, nullptr, w_tiled, sw_tiled, N, K, out);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(M >= 0 && ldc >= N, "%s: need M >= 0 and ldc >= N (M=%lld ldc=%lld)", who, (long long)M, (long long)ldc);
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0, "%s: ldx must be >= K and a multiple of 8", who);
  MXL_CHECK_ARG(fp4_rule(rule), "%s: unknown rule %d", who, rule);
  if (M == 0) return MXL_OK;
  MXL_CHECK_ARG(fp4_rows_reach(M, ldx, K), "%s: the rows span more than 4 GiB", who);
  Fp4StreamPlan pl;
  if (!fp4_dense_streams(M, N, K, true, pl)) {
    set_error("%s: %lld rows of K = %lld do not run in one launch", who, (long long)M, (long long)K);
    return MXL_EUNSUPPORTED;
  }
  GemmParams p = fp4_params(nullptr, nullptr, w_tiled, sw_tiled, N, K, out, ldc);
  p.M = p.a_rows = M;
  p.bias = (const uint16_t*)bias;
  Fp4Stream g{};
  g.x = (const uint16_t*)x;
  g.ldx = ldx;
  g.carry = fp4_carry(rule);
  return launch_status(launch_fp4_stream<1, false>(pl, p, g, 1, (hipStream_t)stream), who);
}

static int check_grouped(const char* who, int64_t a_rows, int row_div, int64_t num_experts, int64_t routed_rows) {
  MXL_CHECK_ARG(num_experts > 0 && num_experts <= 0xFFFF && row_div >= 1 && a_rows >= 0 && routed_rows >= 0,
                "%s: need 0 < experts <= 65535, row_div >= 1 and row counts >= 0", who);
  MXL_CHECK_ARG(routed_rows == 0 || a_rows > 0, "%s: no activation rows", who);
  return MXL_OK;
}

extern "C" int mxl_mxfp4_grouped_swiglu_supported(int64_t routed_rows, int64_t num_experts, int64_t I, int64_t K) {
  Fp4StreamPlan pl;
  return routed_rows > 0 && num_experts > 0 && num_experts <= 0xFFFF && I > 0 && I % 32 == 0 && K > 0 && K % 128 == 0 &&
         fp4_grouped_streams(routed_rows, num_experts, 2 * I, K, true, pl);
}

extern "C" int mxl_mxfp4_grouped_swiglu(const void* x, int64_t a_rows, int64_t ldx, const int32_t* row_index, int row_div,
                                        const int64_t* expert_offsets, int64_t num_experts, int64_t routed_rows,
                                        const void* w_tiled, const void* sw_tiled, int64_t I, int64_t K, int rule,
                                        void* codes, void* scales, void* stream) {
  const char* who = "mxl_mxfp4_grouped_swiglu";
  int rc = check_operands(who, x, nullptr, w_tiled, sw_tiled, 2 * I, K, nullptr);
  if (rc == MXL_OK) rc = check_grouped(who, a_rows, row_div, num_experts, routed_rows);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(I % 32 == 0, "%s: need I %% 32 == 0 (I=%lld)", who, (long long)I);
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0, "%s: ldx must be >= K and a multiple of 8", who);
  MXL_CHECK_ARG(fp4_rule(rule), "%s: unknown rule %d", who, rule);
  MXL_CHECK_ARG(((uintptr_t)codes & 3) == 0, "%s: the codes must be 4-byte aligned", who);
  MXL_CHECK_ARG(fp4_rows_reach(a_rows, ldx, K), "%s: the rows span more than 4 GiB", who);
  if (routed_rows == 0) return MXL_OK;
  Fp4StreamPlan pl;
  if (!fp4_grouped_streams(routed_rows, num_experts, 2 * I, K, true, pl)) {
    set_error("%s: %lld rows of %lld experts of K = %lld do not run in one launch", who, (long long)routed_rows,
              (long long)num_experts, (long long)K);
    return MXL_EUNSUPPORTED;
  }
  GemmParams p = fp4_params(nullptr, nullptr, w_tiled, sw_tiled, 2 * I, K, nullptr, 2 * I);
  p.M = routed_rows; p.a_rows = a_rows; p.row_index = row_index; p.row_div = row_div; p.expert_offsets = expert_offsets;
  p.w_expert_stride = mxl_tiled_weight_bytes(2 * I, K, kE2M1);
  p.sw_expert_stride = mxl_tiled_scale_bytes(2 * I, K);
  Fp4Stream g{};
  g.E = (int)num_experts;
  g.unit = routed_rows < num_experts ? kHitExperts : kExperts;
  g.x = (const uint16_t*)x;
  g.ldx = ldx;
  g.carry = fp4_carry(rule);
  g.codes = (uint8_t*)codes;
  g.scales = (uint8_t*)scales;
  return launch_status(launch_fp4_stream<1, true>(pl, p, g, std::min(routed_rows, num_experts), (hipStream_t)stream), who);
}

extern "C" int mxl_mxfp4_grouped_gemm(const void* a, const void* sa, int64_t a_rows, const int32_t* row_index,
                                      int row_div, const int64_t* expert_offsets, int64_t num_experts,
                                      int64_t routed_rows, const void* w_tiled, const void* sw_tiled, int64_t N,
                                      int64_t K, void* out, void* stream) {
  const char* who = "mxl_mxfp4_grouped_gemm";
  int rc = check_operands(who, a, sa, w_tiled, sw_tiled, N, K, out);
  if (rc == MXL_OK) rc = check_grouped(who, a_rows, row_div, num_experts, routed_rows);
  if (rc != MXL_OK) return rc;
  if (routed_rows == 0) return MXL_OK;
  GemmParams p = fp4_params(a, sa, w_tiled, sw_tiled, N, K, out, N);
  p.M = routed_rows; p.a_rows = a_rows; p.row_index = row_index; p.row_div = row_div; p.expert_offsets = expert_offsets;
  p.w_expert_stride = mxl_tiled_weight_bytes(N, K, kE2M1);
  p.sw_expert_stride = mxl_tiled_scale_bytes(N, K);
  Fp4StreamPlan pl;
  // (the streaming kernel numbers the 16-byte pieces of A in 32 bits)
  if (a_rows <= (int64_t(1) << 32) / (K / 32) && fp4_grouped_streams(routed_rows, num_experts, N, K, false, pl)) {
    Fp4Stream g{};
    g.E = (int)num_experts;
    g.unit = routed_rows < num_experts ? kHitExperts : kExperts;
    return launch_status(launch_fp4_stream<0, false>(pl, p, g, std::min(routed_rows, num_experts), (hipStream_t)stream), who);
  }
  if (num_experts <= kWideGroupedMaxExperts && fp4_tiles_eligible(std::max(a_rows, routed_rows), N, K)) {
    // 128-row blocks whatever the rows an expert (64-row ones: 400 tokens of 256 experts 56.0 either way, 777 of 48
    // 27.3 against 23.8)
    WideConfig c{2, 1, p.KT};
    c.MT = 8;
    return launch_status(launch_gemm_wide(kE2M1, false, c, p, num_experts, (hipStream_t)stream), who);
  }
  fp4_grouped_kernel<<<dim3((unsigned)((N + 63) / 64), (unsigned)num_experts), 256, 0, (hipStream_t)stream>>>(p);
  MXL_CHECK_LAUNCH(who);
  return MXL_OK;
}

// Routes that an experts call of few tokens runs unsorted, each a unit of its own: the sort's launch costs
// more than weights that some share, which come from L2 the second time (256 experts, top 8, K = 2048, I = 512, graph-
// timed, us, unsorted | sorted: one token 14.5 | 18.9, four 21.4 | 26.2, four of the same experts 16.9 | 19.4, eight of
// the same 23.0 | 20.0).
constexpr int64_t kFp4DirectRoutes = 32;
static bool fp4_direct(int64_t routes, int64_t E, int64_t H, int64_t I) {
  Fp4StreamPlan pl;
  return routes <= kFp4DirectRoutes && E <= 0x7FFFFFFF && fp4_grouped_streams(routes, E, 2 * I, H, true, pl) &&
         fp4_grouped_streams(routes, E, H, I, false, pl);
}

// Both products of the unsorted routes: x bf16 [T, H] through w13 and the SwiGLU producer to codes and scales [routes,
// I], then through w2 to y [routes, H].  The plans are those of the sorted routes' units, min(routes, E): K is split over
// the same waves, so a layer has the same bits from ids and from a router's sorted routes.
static hipError_t fp4_direct_launch(const void* x, int64_t T, int64_t ldx, const int32_t* ids, int64_t topk, int64_t E,
                                    int64_t H, int64_t I, const void* w13, const void* sw13, const void* w2,
                                    const void* sw2, int rule, void* codes, void* scales, void* y, hipStream_t s) {
  const int64_t routes = T * topk;
  Fp4StreamPlan pl;
  Fp4Stream g{};
  g.E = (int)E;
  g.unit = kRoutes;
  GemmParams p = fp4_params(nullptr, nullptr, w13, sw13, 2 * I, H, nullptr, 2 * I);
  p.M = routes; p.a_rows = T; p.row_index = ids; p.row_div = (int)topk;
  p.w_expert_stride = mxl_tiled_weight_bytes(2 * I, H, kE2M1);
  p.sw_expert_stride = mxl_tiled_scale_bytes(2 * I, H);
  g.x = (const uint16_t*)x;
  g.ldx = ldx;
  g.carry = fp4_carry(rule);
  g.codes = (uint8_t*)codes;
  g.scales = (uint8_t*)scales;
  if (!fp4_stream_plan(2 * I, H, std::min(routes, E), true, pl)) return hipErrorInvalidValue;
  const hipError_t e = launch_fp4_stream<1, true>(pl, p, g, routes, s);
  if (e != hipSuccess) return e;
  GemmParams q = fp4_params(codes, scales, w2, sw2, H, I, y, H);
  q.M = q.a_rows = routes; q.row_index = ids; q.row_div = 1;
  q.w_expert_stride = mxl_tiled_weight_bytes(H, I, kE2M1);
  q.sw_expert_stride = mxl_tiled_scale_bytes(H, I);
  if (!fp4_stream_plan(H, I, std::min(routes, E), false, pl)) return hipErrorInvalidValue;
  return launch_fp4_stream<0, false>(pl, q, g, routes, s);
}

// Whether the gate/up product of an experts call (I % 128 == 0) runs in the tiles, whose epilogue then is the SwiGLU
// producer.
static bool fp4_swiglu_tiles(int64_t T, int64_t routed_rows, int64_t num_experts, int64_t I, int64_t K) {
  Fp4StreamPlan pl;
  return num_experts <= kWideGroupedMaxExperts &&
         !fp4_grouped_streams(routed_rows, num_experts, 2 * I, K, false, pl) &&
         fp4_tiles_eligible(std::max(T, routed_rows), 2 * I, K);
}

// Its launch: codes a / sa of T rows, MXFP4 SwiGLU codes [routed rows, I / 2] and scales [routed rows, I / 32] out.
static int fp4_swiglu_tiles_launch(const char* who, const void* a, const void* sa, int64_t T, const int32_t* row_index,
                                   int row_div, const int64_t* expert_offsets, int64_t num_experts, int64_t routed_rows,
                                   const void* w_tiled, const void* sw_tiled, int64_t I, int64_t K, int rule, void* codes,
                                   void* scales, hipStream_t s) {
  const int rc = check_operands(who, a, sa, w_tiled, sw_tiled, 2 * I, K, nullptr);
  if (rc != MXL_OK) return rc;
  GemmParams p = fp4_params(a, sa, w_tiled, sw_tiled, 2 * I, K, nullptr, 2 * I);
  p.M = routed_rows; p.a_rows = T; p.row_index = row_index; p.row_div = row_div; p.expert_offsets = expert_offsets;
  p.w_expert_stride = mxl_tiled_weight_bytes(2 * I, K, kE2M1);
  p.sw_expert_stride = mxl_tiled_scale_bytes(2 * I, K);
  p.mid_codes = (uint8_t*)codes; p.mid_scales = (uint8_t*)scales; p.mid_carry = fp4_carry(rule);
  WideConfig c{2, 1, p.KT};
  c.MT = 8;
  return launch_status(launch_gemm_wide(kE2M1, false, c, p, num_experts, s), who);
}

// ------------------------------------------------------------------ layers in one call

extern "C" int mxl_quantize_mxfp4(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes, void* scales,
                                  void* stream);
extern "C" int mxl_swiglu_mxfp4(const void* gate_up, int64_t M, int64_t K, int rule, void* codes, void* scales,
                                void* stream);
extern "C" int64_t mxl_moe_route_workspace_bytes(int64_t T, int64_t topk, int64_t E);
extern "C" int mxl_moe_route(const int32_t* topk_ids, int64_t T, int64_t topk, int64_t E, int32_t* sorted_routes,
                             int64_t* expert_offsets, int32_t* inverse, void* workspace, int64_t workspace_bytes,
                             void* stream);
extern "C" int mxl_moe_reduce(const void* routed_output, const float* topk_weights, const int32_t* inverse, int64_t T,
                              int64_t topk, int64_t H, void* out, void* stream);

namespace {

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

struct LinearScratch {
  void *codes, *scales, *gemm;
  int64_t gemm_bytes, bytes;
};
LinearScratch linear_scratch(uint8_t* base, int64_t M, int64_t N, int64_t K) {
  Pieces p{base};
  LinearScratch l;
  l.codes = p.take(M * (K / 2));
  l.scales = p.take(M * (K / 32));
  l.gemm_bytes = mxl_mxfp4_gemm_workspace_bytes(M, N, K);
  l.gemm = p.take(l.gemm_bytes);
  l.bytes = p.used;
  return l;
}

struct ExpertScratch {
  void *routes, *offsets, *inverse, *sort, *codes, *scales, *gate_up, *codes2, *scales2, *y;
  int64_t sort_bytes, bytes;
  bool direct;        // the routes unsorted
  bool fused, tiles;  // the SwiGLU producer in the gate/up product's launch: with the quantizer, or behind it
};
ExpertScratch expert_scratch(uint8_t* base, int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, bool sorted,
                             bool fuse) {
  const int64_t R = T * topk;
  Pieces p{base};
  ExpertScratch x{};
  x.direct = fuse && !sorted && fp4_direct(R, E, H, I);
  sorted |= x.direct;  // (no sort)
  x.sort_bytes = sorted ? 0 : mxl_moe_route_workspace_bytes(T, topk, E);
  x.fused = fuse && T <= (int64_t(1) << 31) / H && mxl_mxfp4_grouped_swiglu_supported(R, E, I, H);  // (32-bit offsets)
  x.tiles = fuse && !x.fused && fp4_swiglu_tiles(T, R, E, I, H);
  if (!sorted) {
    x.routes = p.take(R * 4);
    x.offsets = p.take((E + 1) * 8);
    x.inverse = p.take(R * 4);
    x.sort = p.take(x.sort_bytes);
  }
  if (!x.fused) {
    x.codes = p.take(T * (H / 2));
    x.scales = p.take(T * (H / 32));
    if (!x.tiles) x.gate_up = p.take(R * 2 * I * 2);
  }
  x.codes2 = p.take(R * (I / 2));
  x.scales2 = p.take(R * (I / 32));
  x.y = p.take(R * H * 2);
  x.bytes = p.used;
  return x;
}

}  // namespace

extern "C" int64_t mxl_mxfp4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int swiglu) {
  if (M <= 0 || N <= 0 || K <= 0 || K % 128 || K > kFp4MaxK) return 0;
  return !swiglu && mxl_mxfp4_quant_gemm_supported(M, N, K) ? 0 : linear_scratch(nullptr, M, N, K).bytes;
}

extern "C" int mxl_mxfp4_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int swiglu, int rule,
                                const void* w_tiled, const void* sw_tiled, int64_t N, const void* bias, void* out,
                                int64_t ldc, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_mxfp4_linear";
  const int rc = check_operands(who, x, nullptr, w_tiled, sw_tiled, N, K, out);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(!swiglu || ldx == 2 * K, "%s: gate/up rows are contiguous, ldx = 2 K", who);
  if (M > 0 && !swiglu && mxl_mxfp4_quant_gemm_supported(M, N, K))
    return mxl_mxfp4_quant_gemm(x, M, K, ldx, rule, w_tiled, sw_tiled, N, bias, out, ldc, stream);
  const int64_t need = mxl_mxfp4_linear_workspace_bytes(M, N, K, swiglu);
  MXL_CHECK_ARG(M <= 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0),
                "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  const LinearScratch l = linear_scratch((uint8_t*)workspace, M > 0 ? M : 0, N, K);
  const int st = swiglu ? mxl_swiglu_mxfp4(x, M, K, rule, l.codes, l.scales, stream)
                        : mxl_quantize_mxfp4(x, M, K, ldx, rule, l.codes, l.scales, stream);
  if (st != MXL_OK || M == 0) return st;
  return mxl_mxfp4_gemm(l.codes, l.scales, M, w_tiled, sw_tiled, N, K, bias, out, ldc, l.gemm, l.gemm_bytes, stream);
}

extern "C" int64_t mxl_mxfp4_experts_workspace_bytes(int64_t T, int64_t topk, int64_t E, int64_t H, int64_t I, int sorted,
                                                     int fuse) {
  if (T <= 0 || topk <= 0 || E <= 0 || H <= 0 || I <= 0) return 0;
  return expert_scratch(nullptr, T, topk, E, H, I, sorted != 0, fuse != 0).bytes;
}

extern "C" int mxl_mxfp4_experts(const void* x, int64_t T, int64_t ldx, const int32_t* topk_ids, const float* topk_weights,
                                 int64_t topk, const int32_t* sorted_routes, const int64_t* expert_offsets,
                                 const int32_t* inverse, int64_t E, int64_t H, int64_t I, const void* w13,
                                 const void* sw13, const void* w2, const void* sw2, int rule, int fuse, void* out,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_mxfp4_experts";
  const bool sorted = sorted_routes != nullptr;
  MXL_CHECK_ARG(T >= 0 && topk > 0 && E > 0, "%s: need T >= 0, topk > 0, E > 0", who);
  MXL_CHECK_ARG(H > 0 && I > 0 && H % 128 == 0 && I % 128 == 0, "%s: need H, I > 0, divisible by 128 (H=%lld I=%lld)", who,
                (long long)H, (long long)I);
  MXL_CHECK_ARG(sorted ? expert_offsets && inverse : topk_ids != nullptr, "%s: needs ids, or the routes sorted", who);
  MXL_CHECK_ARG(T <= 0x7FFFFFFF / topk, "%s: too many routes", who);
  if (T == 0) return MXL_OK;
  const int64_t R = T * topk, need = mxl_mxfp4_experts_workspace_bytes(T, topk, E, H, I, sorted, fuse);
  MXL_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
                "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  ExpertScratch s = expert_scratch((uint8_t*)workspace, T, topk, E, H, I, sorted, fuse != 0);
  int st = MXL_OK;
  if (s.direct) {
    MXL_CHECK_ARG(ldx >= H && ldx % 8 == 0 && fp4_rule(rule) && (((uintptr_t)x | (uintptr_t)w13 | (uintptr_t)w2) & 15) == 0 &&
                      (((uintptr_t)sw13 | (uintptr_t)sw2) & 3) == 0 && H <= kFp4MaxK && I <= kFp4MaxK,
                  "%s: bad stride, rule, alignment or size (ldx=%lld rule=%d H=%lld I=%lld)", who, (long long)ldx, rule,
                  (long long)H, (long long)I);
    MXL_CHECK_ARG(fp4_rows_reach(T, ldx, H), "%s: the rows span more than 4 GiB", who);
    st = launch_status(fp4_direct_launch(x, T, ldx, topk_ids, topk, E, H, I, w13, sw13, w2, sw2, rule, s.codes2, s.scales2,
                                         s.y, (hipStream_t)stream), who);
    return st != MXL_OK ? st : moe_reduce_by_route(who, s.y, topk_weights, topk_ids, T, topk, E, H, out, stream);
  }
  if (!sorted) {
    st = mxl_moe_route(topk_ids, T, topk, E, (int32_t*)s.routes, (int64_t*)s.offsets, (int32_t*)s.inverse, s.sort,
                       s.sort_bytes, stream);
    if (st != MXL_OK) return st;
    sorted_routes = (const int32_t*)s.routes;
    expert_offsets = (const int64_t*)s.offsets;
    inverse = (const int32_t*)s.inverse;
  }
  if (s.fused) {
    st = mxl_mxfp4_grouped_swiglu(x, T, ldx, sorted_routes, (int)topk, expert_offsets, E, R, w13, sw13, I, H, rule,
                                  s.codes2, s.scales2, stream);
  } else {
    st = mxl_quantize_mxfp4(x, T, H, ldx, rule, s.codes, s.scales, stream);
    if (st == MXL_OK)
      st = s.tiles ? fp4_swiglu_tiles_launch(who, s.codes, s.scales, T, sorted_routes, (int)topk, expert_offsets, E, R, w13,
                                             sw13, I, H, rule, s.codes2, s.scales2, (hipStream_t)stream)
                   : mxl_mxfp4_grouped_gemm(s.codes, s.scales, T, sorted_routes, (int)topk, expert_offsets, E, R, w13, sw13,
                                            2 * I, H, s.gate_up, stream);
    if (st == MXL_OK && !s.tiles) st = mxl_swiglu_mxfp4(s.gate_up, R, I, rule, s.codes2, s.scales2, stream);
  }
  if (st == MXL_OK)
    st = mxl_mxfp4_grouped_gemm(s.codes2, s.scales2, R, nullptr, 1, expert_offsets, E, R, w2, sw2, H, I, s.y, stream);
  if (st == MXL_OK) st = mxl_moe_reduce(s.y, topk_weights, inverse, T, topk, H, out, stream);
  return st;
}
