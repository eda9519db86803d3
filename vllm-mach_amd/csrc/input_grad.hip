// The input gradient of a frozen quantized linear layer on gfx950: dx = dy W, dy bf16 [M, N], W the layer's tiled codes
// [N, K] (MXFP8, MXFP6, MXFP4 with E8M0 scales per 32 of K; E4M3 with fp32 scales per 128 x 128), fp32 sums, bf16 out.
//
// The product runs over W's rows, across its scales, so the scaled MFMA cannot take the codes: they become bf16, which
// holds every code times a power of two exactly (within bf16's exponents), and the bf16 MFMA multiplies.  Block-FP8 codes
// are multiplied as they are, and each 128 rows' sum joins with its block's scale.
//
// A workgroup of 2 x 2 waves owns TM rows of dx by TK columns.  A stage is 64 rows of W: a wave decodes one tiled 16-row
// strip of it (scale and conversion are one instruction for a pair, or for 32 FP6 values) into LDS, row by row as W is,
// and the MFMA's operand, eight rows of one column a lane, comes out of LDS transposed (ds_read_b64_tr_b16).  W takes the
// A operand, so a lane holds four consecutive columns of a row of dx.
//
// Bound: the MFMAs at the clock that the power limit leaves, busy 65 % of the time (the rest: the stage's barrier and LDS
// issue).  2048 x 18432 x 2560 in 256 x 256 tiles: 184 us, 1.05 PFLOP/s, and 13 us for the join of the splits (as a library
// bf16 product of decoded weights 250 us).  Each workgroup decodes its strip of W anew: 256 rows share a decode.
#include <stdio.h>

#include <algorithm>
#include <type_traits>
#include <utility>

#include "adapters.h"
#include "gemm_wide.h"

namespace mxl {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x32_t __attribute__((ext_vector_type(32)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned int v6u_t __attribute__((ext_vector_type(6)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

constexpr int kGradStage = 64;  // rows of W

// f of 0 .. N - 1 as constants (register arrays are indexed by nothing else)
template <int N, class F>
__device__ __forceinline__ void for_n(F&& f) {
  if constexpr (N > 0) {
    for_n<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

struct GradParams {
  const uint16_t* dy;
  const uint8_t* w;
  const void* sw;  // tiled E8M0, or fp32 [ceil(N / 128), K / 128]
  uint16_t* out;
  float* partial;  // [S, M, K] when split
  int64_t M, N, K, KT, lddy, ldo;  // (N in whole pairs of stages)
  int S, strips;   // of 16 rows of W
  int64_t per;     // stages of a split, an even number
  uint32_t mblocks, kblocks, group_m;
  RowAdapters more;  // (ids null: none)
};

// The pieces of a stage that a thread moves from memory to LDS: NA 16-byte pieces of dy, and of its wave's strip of W
// (16 rows) the lane's codes of SL 128-column slices.
template <int FMT, int TM, int TK>
struct GradPieces {
  static constexpr int NA = TM / 32, SL = TK / 128;
  static constexpr int NC = FMT == kE4M3 ? 2 * SL : FMT == kE2M1 ? SL : SL == 2 ? 3 : 2;  // 16-byte pieces a lane
  static constexpr int UNITS = FMT == kE4M3 ? 2 * SL : SL;                              // decoded one by one
  u32x4 a[NA], c[NC];
  uint32_t s[2];
};

template <int FMT, int TM, int TK, bool BLOCK>
__global__ __launch_bounds__(256, (TM * TK > 128 * 128 ? 1 : 2)) void input_grad_kernel(GradParams p) {
  using Pieces = GradPieces<FMT, TM, TK>;
  constexpr int MI = TM / 64, KI = TK / 64, SL = Pieces::SL;  // 32 x 32 tiles of a wave; slices
  constexpr int RS = TK + 32;                                // elements of a row of W in LDS
  constexpr int A_BYTES = TM * 128, W_BYTES = kGradStage * RS * 2;
  constexpr int NA = Pieces::NA, NC = Pieces::NC;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [2] dy, [2] W
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wv >> 1, wk = wv & 1, r = lane & 15, q = lane >> 4;

  const uint32_t unit = wide_logical(blockIdx.x, gridDim.x), tiles = p.mblocks * p.kblocks;
  const uint32_t split = unit / tiles;
  uint32_t mb, kb;
  wide_coords(unit - split * tiles, p.mblocks, p.kblocks, p.group_m, mb, kb);
  const int64_t row0 = (int64_t)mb * TM;
  // the split's stages, an even number (dy has columns for all of them, zeros past W's last row)
  const int stages = (int)(p.N / kGradStage), s0 = (int)(split * p.per);
  const int s1 = s0 + (int)p.per < stages ? s0 + (int)p.per : stages;
  const int j0 = (int)(kb * SL) & 3;  // the first slice's place in its super-tile
  const int64_t kt = (int64_t)kb * SL >> 2;

  // dy: piece u of a thread is row t / 8 + 32 u, columns 8 (t % 8) of the stage; rows past M are the last again
  const uint8_t* const a_base = reinterpret_cast<const uint8_t*>(p.dy + row0 * p.lddy);
  const uint32_t ld = (uint32_t)p.lddy * 2, a_rows = (uint32_t)(p.M - row0 < TM ? p.M - row0 : TM);
  const uint32_t a_at = (uint32_t)(t >> 3) * ld + 16 * (t & 7), a_max = (a_rows - 1) * ld + 16 * (t & 7);
  Pieces x;
  auto load_a = [&](auto u, int s) {
    const uint32_t off = __builtin_elementwise_min(a_at + (uint32_t)(32 * u) * ld, a_max);
    x.a[u] = *reinterpret_cast<const u32x4*>(a_base + (int64_t)s * (2 * kGradStage) + off);
  };
  auto load_w = [&](int s) {  // (strips past the last: the last again, times zeros)
    const int nt = 4 * s + wv < p.strips ? 4 * s + wv : p.strips - 1;
    const int64_t tile = (int64_t)nt * p.KT + kt;
    const uint8_t* const w = p.w + tile * (FmtTraits<FMT>::CH * 1024) + lane * 16;
    const int c0 = FMT == kE4M3 ? 2 * j0 : FMT == kE2M1 ? j0 : (3 * j0) >> 1;
#pragma unroll
    for (int c = 0; c < NC; ++c) x.c[c] = *reinterpret_cast<const u32x4*>(w + (c0 + c) * 1024);
    if constexpr (!BLOCK) {
      const uint8_t* const sw = static_cast<const uint8_t*>(p.sw) + tile * 256;
      if constexpr (FMT == kE4M3) {  // pieces of 16 columns: half a block each, of lane groups q / 2 and 2 + q / 2
        x.s[0] = *reinterpret_cast<const uint32_t*>(sw + (16 * (q >> 1) + r) * 4);
        x.s[1] = *reinterpret_cast<const uint32_t*>(sw + (16 * (2 + (q >> 1)) + r) * 4);
      } else {
        x.s[0] = *reinterpret_cast<const uint32_t*>(sw + lane * 4);
      }
    }
  };
  // dy: piece i of row y sits at 16 (i ^ y / 2 % 8) of its 128 bytes: sixteen rows' same piece in all 64 banks
  uint8_t* const a_to = lds + (t >> 3) * 128 + 16 * ((t & 7) ^ ((t >> 4) & 7));
  auto store_a = [&](auto u, int buf) { *reinterpret_cast<u32x4*>(a_to + buf * A_BYTES + u * 4096) = x.a[u]; };
  // W: rows 64 bytes past a multiple of 256 apart, and of each 64 bytes of row y the pieces change places by y / 4 % 4:
  // sixteen rows' same piece, and four rows' 64 bytes, in all 64 banks.  A unit of the strip's row r: 16 (E4M3) or 32 columns
  uint8_t* const w_to = lds + 2 * A_BYTES + (16 * wv + r) * (RS * 2);
  const int w_swz = r >> 2;
  auto store_w = [&](auto U, int buf) {
    constexpr int un = decltype(U)::value, sl = FMT == kE4M3 ? un / 2 : un, h = FMT == kE4M3 ? un & 1 : 0;
    const float f = u2f(BLOCK ? 127u << 23 : __builtin_amdgcn_ubfe(x.s[h], 8 * (j0 + sl), 8) << 23);
    uint8_t* const base = w_to + buf * W_BYTES + (128 * sl + (FMT == kE4M3 ? 64 * h + 32 * (q >> 1) : 32 * q)) * 2;
    auto dst = [&](int i) -> u32x4& {  // piece i of the unit
      return *reinterpret_cast<u32x4*>(base + 16 * ((FMT == kE4M3 ? 2 * (q & 1) + i : i) ^ w_swz));
    };
    auto bits = [](auto v) { return __builtin_bit_cast(uint32_t, v); };
    if constexpr (FMT == kE4M3) {
      const u32x4 c = x.c[un];
      const uint32_t d[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        dst(i) = u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[2 * i], f, false)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[2 * i], f, true)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[2 * i + 1], f, false)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[2 * i + 1], f, true))};
    } else if constexpr (FMT == kE2M1) {
      const uint32_t d[4] = {x.c[un].x, x.c[un].y, x.c[un].z, x.c[un].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst(i) = u32x4{bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 0)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 1)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 2)),
                       bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 3))};
    } else {
      v6u_t d;  // six dwords, of an odd first slice from the first piece's middle
      const u32x4 y = x.c[un], z = x.c[un + 1];
      const bool odd = SL == 2 ? un == 1 : (j0 & 1) != 0;
      d[0] = odd ? y.z : y.x; d[1] = odd ? y.w : y.y; d[2] = odd ? z.x : y.z;
      d[3] = odd ? z.y : y.w; d[4] = odd ? z.z : z.x; d[5] = odd ? z.w : z.y;
      bf16x32_t v;
      if constexpr (FMT == kE2M3) v = __builtin_amdgcn_cvt_scalef32_pk32_bf16_fp6(d, f);
      else v = __builtin_amdgcn_cvt_scalef32_pk32_bf16_bf6(d, f);
      struct Q { u32x4 x[4]; };
      const Q o = __builtin_bit_cast(Q, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) dst(i) = o.x[i];
    }
  };

  v16f acc[MI][KI], raw[BLOCK ? MI : 1][BLOCK ? KI : 1];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int c = 0; c < KI; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[m][c][e] = 0.0f;
  if constexpr (BLOCK) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int c = 0; c < KI; ++c) raw[m][c] = acc[m][c];
  }
  // fragments of a slice of 16 rows of W: dy row lane % 32 and columns 8 (lane / 32), W column lane % 32 and those rows
  const int ah = lane >> 5;
  const uint8_t* const a_from = lds + (wm * (TM / 2) + (lane & 31)) * 128;
  const uint8_t* w_from[2];  // rows 0 .. 3 and 4 .. 7 of the lane's eight
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w_from[h] = lds + 2 * A_BYTES + (8 * (q >> 1) + 4 * h + (r >> 2)) * (RS * 2) + wk * TK +
                (16 * ((2 * (q & 1) + ((r & 3) >> 1)) ^ (2 * (q >> 1) + h)) + 8 * (r & 1));
  u32x4 af[2][MI];
  u32x2 wf[2][KI][2];
  constexpr int READS = MI + 2 * KI;
  auto read = [&](auto I, auto KK, int buf) {  // read I of slice KK
    constexpr int i = decltype(I)::value, kk = decltype(KK)::value;
    if constexpr (i < 2 * KI) {
      const uint8_t* const src = w_from[i & 1] + buf * W_BYTES + 16 * kk * (RS * 2) + (i >> 1) * 64;
      wf[kk & 1][i >> 1][i & 1] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)src));
    } else {
      af[kk & 1][i - 2 * KI] = *reinterpret_cast<const u32x4*>(a_from + buf * A_BYTES + (i - 2 * KI) * 4096 + 16 * ((2 * kk) ^ ah ^ ((lane >> 1) & 7)));
    }
  };
  auto mfma = [&](auto I, auto KK) {
    constexpr int i = decltype(I)::value, kk = decltype(KK)::value, m = i / KI, c = i % KI;
    v16f& sum = BLOCK ? raw[BLOCK ? m : 0][BLOCK ? c : 0] : acc[m][c];
    const u32x2 lo = wf[kk & 1][c][0], hi = wf[kk & 1][c][1];
    sum = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, u32x4{lo.x, lo.y, hi.x, hi.y}),
                                                 __builtin_bit_cast(bf16x8_t, af[kk & 1][m]), sum, 0, 0, 0);
  };
  auto fold = [&](int block_row) {  // 128 rows of W end: their sums by their block's scale
    if constexpr (BLOCK) {
      static_assert(TK == 128, "a scale a workgroup");
      const float f = static_cast<const float*>(p.sw)[block_row * (p.K / 128) + kb];
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int c = 0; c < KI; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            acc[m][c][e] = __builtin_fmaf(raw[m][c][e], f, acc[m][c][e]);
            raw[m][c][e] = 0.0f;
          }
    }
  };
  // this wave's LDS reads and writes are done, then the barrier (loads stay in flight)
  auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  if (s0 < s1) {
    // Stage s of four slices, MI KI MFMAs each.  Under them the next slice's fragments are read, the next stage's pieces
    // go from registers to LDS (slices 0 to 2) and those of the stage after it are requested.  Before the last slice
    // all waves meet: the next stage lies in LDS whole, and this one's fragments are all in registers, so the last
    // slice reads the next stage's first fragments and its buffer is free for the stage after.
    constexpr int S = MI * KI;
    auto stage = [&](auto BUF, int s) {
      constexpr int buf = decltype(BUF)::value;
      const int next = s + 2 < s1 ? s + 2 : s1 - 1;
      auto slice = [&](auto KK) {
        constexpr int kk = decltype(KK)::value, rk = (kk + 1) & 3, rb = kk == 3 ? buf ^ 1 : buf;
        if constexpr (kk == 3) meet();
        auto step = [&](auto I) {
          constexpr int i = decltype(I)::value;
          mfma(I, KK);
          // (the last quarter of a slice's steps reads nothing: its reads have landed when the next begins)
          constexpr int over = S - S / 4, first = i < over ? i * READS / over : READS, end = i < over ? (i + 1) * READS / over : READS;
          for_n<end - first>([&](auto n) {
            read(std::integral_constant<int, first + decltype(n)::value>{}, std::integral_constant<int, rk>{}, rb);
          });
          if constexpr (kk < 3) {
            // pieces to LDS: the strip's units, then dy's NA
            constexpr int ALL = NA + Pieces::UNITS, over = 3 * S - S / 2, at = kk * S + i;
            constexpr int lo = at < over ? at * ALL / over : ALL, hi = at < over ? (at + 1) * ALL / over : ALL;
            if constexpr (hi > lo) {
              static_assert(hi - lo == 1, "a piece a step");
              if constexpr (lo < Pieces::UNITS) {
                store_w(std::integral_constant<int, lo>{}, buf ^ 1);
                if constexpr (lo == Pieces::UNITS - 1) load_w(next);
              } else {
                store_a(std::integral_constant<int, lo - Pieces::UNITS>{}, buf ^ 1);
                load_a(std::integral_constant<int, lo - Pieces::UNITS>{}, next);
              }
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        };
        for_n<S>(step);
      };
      for_n<4>(slice);
      if constexpr (BLOCK && buf == 1) fold(s >> 1);
    };
    for_n<NA>([&](auto u) { load_a(u, s0); });
    load_w(s0);
    for_n<NA>([&](auto u) { store_a(u, 0); });
    for_n<Pieces::UNITS>([&](auto u) { store_w(u, 0); });
    for_n<NA>([&](auto u) { load_a(u, s0 + 1); });
    load_w(s0 + 1);
    meet();
    for_n<READS>([&](auto i) { read(i, std::integral_constant<int, 0>{}, 0); });
    for (int s = s0; s < s1; s += 2) {
      stage(std::integral_constant<int, 0>{}, s);
      stage(std::integral_constant<int, 1>{}, s + 1);
    }
  }

  bool odd = false;  // the wave left out values that are not finite
  if (p.more.ids && split == 0) {
    // The adapters of the tile's rows, in turn, 16 ranks at a time: A's rows take the place of W's (as they are), dv's
    // halves that of dy, zero in other adapters' rows.
    const RowAdapters& o = p.more;
    int own[MI], all[TM / 64];  // of the lane's row of each m-tile; of rows lane + 64 i of the tile
    auto id = [&](int64_t row) {
      const int x = row < p.M ? o.ids[row] : -1;
      return (uint32_t)x < (uint32_t)o.slots ? x : 0x7FFFFFFF;
    };
    for_n<MI>([&](auto m) { own[m] = id(row0 + wm * (TM / 2) + 32 * m + (lane & 31)); });
    for_n<TM / 64>([&](auto i) { all[i] = id(row0 + lane + 64 * i); });
    const int width = o.l.width(), groups = o.l.parts * o.l.groups;
    for (int last = -1;;) {
      int a = 0x7FFFFFFF;
      for_n<TM / 64>([&](auto i) { a = all[i] > last && all[i] < a ? all[i] : a; });
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int b = __shfl_xor(a, d, 64);
        a = b < a ? b : a;
      }
      a = last = __builtin_amdgcn_readfirstlane(a);
      if (a == 0x7FFFFFFF) break;
      for (int g = 0; g < groups; ++g) {
        const int part = g / o.l.groups, j0r = 16 * (g - part * o.l.groups);
        const uint16_t* const rows = o.mat + a * o.slot_stride + (int64_t)(part * o.l.rank + j0r) * o.ldm + (int64_t)kb * TK;
        u32x4 piece[TK / 128];
        for_n<TK / 128>([&](auto u) {  // row, columns 8 c ..
          const int at = t + 256 * u, y = at / (TK / 8), c = at % (TK / 8);
          piece[u] = u32x4{0, 0, 0, 0};
          if (j0r + y < o.l.rank && (int64_t)kb * TK + 8 * c < p.K) piece[u] = *reinterpret_cast<const u32x4*>(rows + y * o.ldm + 8 * c);
        });
        u32x4 vf[2][MI];
        for_n<MI>([&](auto m) {
          const int64_t row = row0 + wm * (TM / 2) + 32 * m + (lane & 31);
          const uint16_t* const v = o.v + (own[m] == a ? row : 0) * (2 * width) + 16 * g + 8 * ah;
          for_n<2>([&](auto h) {
            vf[h][m] = u32x4{0, 0, 0, 0};
            if (own[m] == a) vf[h][m] = *reinterpret_cast<const u32x4*>(v + h * width);
          });
        });
        meet();  // (the last reads of W's buffer)
        for_n<TK / 128>([&](auto u) {
          const int at = t + 256 * u, y = at / (TK / 8), c = at % (TK / 8);
          *reinterpret_cast<u32x4*>(lds + 2 * A_BYTES + y * (RS * 2) + 16 * (c ^ (y >> 2))) = piece[u];
        });
        meet();
        for_n<2 * KI>([&](auto i) { read(i, std::integral_constant<int, 0>{}, 0); });
        uint32_t top = 0;
        for_n<4 * KI>([&](auto i) { top = adapter_top(top, wf[0][i / 4][i / 2 % 2][i % 2]); });
        if (__builtin_amdgcn_ballot_w64(adapter_odd(top)) != 0) {
          odd = true;
          for_n<4 * KI>([&](auto i) { wf[0][i / 4][i / 2 % 2][i % 2] = adapter_finite(wf[0][i / 4][i / 2 % 2][i % 2]); });
        }
        for_n<2>([&](auto h) {
          for_n<MI * KI>([&](auto i) {
            constexpr int m = decltype(i)::value / KI, c = decltype(i)::value % KI;
            const u32x2 x0 = wf[0][c][0], x1 = wf[0][c][1];
            acc[m][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, u32x4{x0.x, x0.y, x1.x, x1.y}),
                                                               __builtin_bit_cast(bf16x8_t, vf[h][m]), acc[m][c], 0, 0, 0);
          });
        });
      }
    }
  }

  // (with all 256 accumulators live the compiler would first copy them to vector registers, more than there are)
  auto value = [&](auto m, auto c, auto e) -> float {
    if constexpr (MI * KI < 16) {
      return acc[m][c][decltype(e)::value];
    } else {
      float x;
      asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(acc[m][c][decltype(e)::value]));
      return x;
    }
  };
  // lane: row lane % 32, columns 8 g + 4 (lane / 32) .. + 3 of a 32 x 32 tile in registers 4 g ..
  for_n<MI>([&](auto m) {
    const int64_t row = row0 + wm * (TM / 2) + 32 * m + (lane & 31);
    for_n<KI>([&](auto c) {
      for_n<4>([&](auto g) {
        const int64_t col = (int64_t)kb * TK + wk * (TK / 2) + 32 * c + 8 * g + 4 * ah;
        v4f v;
        for_n<4>([&](auto e) {
          constexpr int i = decltype(e)::value;
          v[i] = value(m, c, std::integral_constant<int, 4 * decltype(g)::value + i>{});
        });
        if (row < p.M && col < p.K) {
          if (p.S > 1) {
            *reinterpret_cast<v4f*>(p.partial + (split * p.M + row) * p.K + col) = v;
          } else {
            const uint32_t h[4] = {f32_to_bf16(v[0]), f32_to_bf16(v[1]), f32_to_bf16(v[2]), f32_to_bf16(v[3])};
            *reinterpret_cast<u32x2*>(p.out + row * p.ldo + col) = u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    });
  });
  if (!odd) return;
  // The terms left out, with a value of A that is not finite: added to what the wave has stored.
  const RowAdapters& o = p.more;
  const int width = o.l.width();
  __threadfence();  // the wave's stores, before it loads them
#pragma unroll 1
  for (int c = lane; c < TK / 2; c += 64) {
    const int64_t col = (int64_t)kb * TK + wk * (TK / 2) + c;
    if (col >= p.K) continue;
    int seen = -1;  // an adapter of which the column's values are known to be finite
#pragma unroll 1
    for (int i = 0; i < TM / 2; ++i) {
      const int64_t row = row0 + wm * (TM / 2) + i;
      if (row >= p.M) break;
      const int a = o.ids[row];
      if ((uint32_t)a >= (uint32_t)o.slots || a == seen) continue;
      float sum = 0.0f;
      bool found = false;
#pragma unroll 1
      for (int part = 0; part < o.l.parts; ++part) {
        const uint16_t* const rows = o.mat + a * o.slot_stride + (int64_t)part * o.l.rank * o.ldm + col;
        const uint16_t* const v = o.v + row * (2 * width) + part * o.l.groups * 16;
#pragma unroll 8
        for (int j = 0; j < o.l.rank; ++j) {
          const uint16_t x = rows[j * o.ldm];
          if ((x & 0x7FFF) >= 0x7F80) sum += adapter_odd_term(x, v[j], v[width + j], found);
        }
      }
      if (!found) {
        seen = a;
      } else if (p.S > 1) {
        p.partial[row * p.K + col] += sum;
      } else {
        uint16_t& y = p.out[row * p.ldo + col];
        y = f32_to_bf16(bf16_to_f32(y) + sum);
      }
    }
  }
}

// out = the sum of the splits' partials [S, M, K], rounded; four columns a thread.
__global__ __launch_bounds__(256) void input_grad_join_kernel(const float* partial, int S, int64_t M, int64_t K,
                                                              uint16_t* out, int64_t ldo) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= M * K) return;
  v4f s = *reinterpret_cast<const v4f*>(partial + at);
  for (int k = 1; k < S; ++k) {
    const v4f x = *reinterpret_cast<const v4f*>(partial + k * M * K + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += x[e];
  }
  const int64_t row = at / K, col = at - row * K;
  const uint32_t h[4] = {f32_to_bf16(s[0]), f32_to_bf16(s[1]), f32_to_bf16(s[2]), f32_to_bf16(s[3])};
  *reinterpret_cast<uint2*>(out + row * ldo + col) = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
}

// dst [M, wide] = src [M, N] with zeros behind it; N and wide in eights.
__global__ __launch_bounds__(256) void input_grad_pad_kernel(const uint16_t* src, int64_t M, int64_t N, int64_t lds,
                                                             int64_t wide, uint16_t* dst) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / (wide / 8), col = 8 * (at - row * (wide / 8));
  if (row >= M) return;
  uint4 v = {0, 0, 0, 0};
  if (col < N) v = *reinterpret_cast<const uint4*>(src + row * lds + col);
  *reinterpret_cast<uint4*>(dst + row * wide + col) = v;
}

// out [N] = the column sums of dy [M, N], fp32 in a fixed order and one rounding: the bias' gradient.  A workgroup owns 64
// columns, a thread eight of them of every 128th row.  (A reduction that clears flags by a memory node would go wrong in
// replays of a captured backward.)  Bound: dy's bytes (2048 x 18432: 16.9 us, 4.5 TB/s), or for few columns the rounds of
// loads (16384 x 128, two workgroups of 16 rounds: 20.9).  `whole`: rows start on 16 bytes.
__global__ __launch_bounds__(1024) void column_sum_kernel(const uint16_t* dy, int64_t M, int64_t N, int64_t ld, bool whole,
                                                          uint16_t* out) {
  __shared__ float sums[16][64];
  const int t = threadIdx.x, lane = t & 63, wv = t >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + 8 * (t & 7);
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (whole && c + 8 <= N) {
    constexpr int U = 8;
    for (int64_t r0 = t >> 3; r0 < M; r0 += 128 * U) {
      u32x4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t r = r0 + 128 * u;
        x[u] = *reinterpret_cast<const u32x4*>(dy + (r < M ? r : r0) * ld + c);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r0 + 128 * u < M) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[2 * e] += u2f(x[u][e] << 16);
            s[2 * e + 1] += u2f(x[u][e] & 0xFFFF0000u);
          }
        }
    }
  } else {
    for (int64_t r = t >> 3; r < M; r += 128)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < N) s[e] += bf16_to_f32(dy[r * ld + c + e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int d = 8; d < 64; d <<= 1) s[e] += __shfl_xor(s[e], d, 64);
    if (lane < 8) sums[wv][8 * lane + e] = s[e];
  }
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * 64 + t;
  if (t >= 64 || col >= N) return;
  float sum = sums[0][t];
#pragma unroll
  for (int w = 1; w < 16; ++w) sum += sums[w][t];
  out[col] = f32_to_bf16(sum);
}

}  // namespace mxl

// ------------------------------------------------------------------- C ABI

using namespace mxl;

namespace {

struct GradPlan {
  int TM, TK, S;
  int64_t per;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile and split by a time model: us of a stage on a CU (of two workgroups where `resident`, and of one alone), in full
// launches at the clock that the power limit leaves; a split's partials make a round trip.  (513 x 5120 x 2688 takes 256 x
// 128 with a split, 28.4 + 5.1 us; 333 x 5120 x 2688 block-FP8 128 x 128, 24.7 + 4.2.)
struct GradCost {
  int TM, TK, resident;
  double stage, alone;
};
constexpr GradCost kGradCosts[] = {{256, 256, 1, 1.73, 1.73}, {256, 128, 1, 0.92, 0.92}, {128, 128, 2, 1.03, 0.62}};
constexpr double kGradFixed = 5.0, kGradJoin = 4.0, kGradBytesPerUs = 5.0e6;

GradPlan grad_plan(int64_t M, int64_t N, int64_t K, bool block) {
  const int64_t pairs = ceil_div(N, 2 * kGradStage), cus = cu_count();
  GradPlan best{};
  double best_us = 1e300;
  for (const GradCost& c : kGradCosts) {
    if (block && c.TM != 128) continue;  // (two sets of sums a lane; 128 x 256 tiles take 1.06 us a stage, never ahead of two of 128)
    const int64_t tiles = ceil_div(M, c.TM) * ceil_div(K, c.TK);
    for (int64_t s = 1; s <= 16 && s <= pairs; ++s) {
      const int64_t per = ceil_div(pairs, s);
      if (ceil_div(pairs, per) != s) continue;
      const int64_t n = ceil_div(tiles * s, cus);  // workgroups of the fullest CU
      double us = kGradFixed + 2 * per * (n / c.resident * c.stage + n % c.resident * c.alone);
      if (s > 1) us += kGradJoin + (8.0 * s + 2.0) * M * K / kGradBytesPerUs;
      if (us >= best_us) continue;
      best_us = us;
      best = GradPlan{c.TM, c.TK, (int)s, 2 * per};
    }
  }
  return best;
}

template <int FMT, bool BLOCK>
hipError_t launch_grad(const GradPlan& g, const GradParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.mblocks * p.kblocks * p.S));
#define MXL_GRAD(TM_, TK_)                                                                             \
  if (g.TM == TM_ && g.TK == TK_) {                                                                    \
    constexpr unsigned lds = 2 * (TM_ * 128 + kGradStage * (TK_ + 32) * 2);                            \
    static_assert(lds <= 160 * 1024, "LDS");                                                           \
    input_grad_kernel<FMT, TM_, TK_, BLOCK><<<grid, 256, lds, s>>>(p);                                 \
    return hipGetLastError();                                                                          \
  }
  if constexpr (!BLOCK) {
    MXL_GRAD(256, 256)
    MXL_GRAD(256, 128)
  }
  MXL_GRAD(128, 128)
#undef MXL_GRAD
  return hipErrorInvalidValue;
}

}  // namespace

// A dy whose columns end inside a pair of stages is copied with zeros behind them, ahead of the partials.
static int64_t pad_bytes(int64_t M, int64_t N) {
  const int64_t wide = ceil_div(N, 2 * kGradStage) * 2 * kGradStage;
  return wide == N ? 0 : ceil_div(M * wide * 2, 256) * 256;
}

int64_t mxl::input_grad_bytes(int64_t M, int64_t N, int64_t K, int block) {
  if (M <= 0 || M > 0x7FFFFFFF || N <= 0 || N > (1 << 22) || K <= 0 || K > (1 << 22)) return 0;
  const GradPlan g = grad_plan(M, N, K, block);
  return pad_bytes(M, N) + (g.S > 1 ? g.S * M * K * 4 : 0);
}

int mxl::input_grad(const char* who, const void* dy, int64_t M, int64_t N, int64_t lddy, const void* w, const void* sw,
                    int64_t K, int fmt, int block, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes,
                    const RowAdapters* more, void* stream) {
  MXL_CHECK_ARG(fmt == kE4M3 || fmt == kE2M3 || fmt == kE3M2 || fmt == kE2M1, "%s: unknown format %d", who, fmt);
  MXL_CHECK_ARG(!block || fmt == kE4M3, "%s: block-FP8 weights are E4M3", who);
  MXL_CHECK_ARG(M >= 0 && N > 0 && N % 8 == 0 && K > 0 && K % 128 == 0 && N <= (1 << 22) && K <= (1 << 22) && M <= 0x7FFFFFFF,
                "%s: need N > 0, N %% 8 == 0, K > 0, K %% 128 == 0, both at most 2^22 (M=%lld N=%lld K=%lld)", who,
                (long long)M, (long long)N, (long long)K);
  MXL_CHECK_ARG(lddy >= N && lddy % 8 == 0 && lddy <= (1 << 22) && ldo >= K && ldo % 4 == 0,
                "%s: need lddy >= N, a multiple of 8 up to 2^22, and ldo >= K, a multiple of 4", who);
  MXL_CHECK_ARG((((uintptr_t)dy | (uintptr_t)w) & 15) == 0 && ((uintptr_t)sw & 3) == 0 && ((uintptr_t)out & 7) == 0,
                "%s: misaligned operands", who);
  if (M == 0) return MXL_OK;
  const GradPlan g = grad_plan(M, N, K, block);
  const int64_t need = input_grad_bytes(M, N, K, block);
  MXL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "%s: needs a 16-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  GradParams p{};
  p.dy = (const uint16_t*)dy; p.w = (const uint8_t*)w; p.sw = sw; p.out = (uint16_t*)out;
  p.M = M; p.N = ceil_div(N, 2 * kGradStage) * 2 * kGradStage; p.K = K; p.KT = ceil_div(K, kTileK);
  p.lddy = lddy; p.ldo = ldo; p.S = g.S; p.per = g.per; p.strips = (int)ceil_div(N, 16);
  p.partial = (float*)((uint8_t*)workspace + pad_bytes(M, N));
  if (more) p.more = *more;
  MXL_CHECK_ARG(ceil_div(M, g.TM) * ceil_div(K, g.TK) * g.S <= 0x7FFFFFFF, "%s: too large", who);
  p.mblocks = (uint32_t)ceil_div(M, g.TM);
  p.kblocks = (uint32_t)ceil_div(K, g.TK);
  p.group_m = std::min<uint32_t>(p.mblocks, 1024 / g.TM);
  hipStream_t s = (hipStream_t)stream;
  if (p.N != N) {
    input_grad_pad_kernel<<<dim3((unsigned)ceil_div(M * p.N / 8, 256)), 256, 0, s>>>(p.dy, M, N, lddy, p.N, (uint16_t*)workspace);
    MXL_CHECK_LAUNCH(who);
    p.dy = (const uint16_t*)workspace;
    p.lddy = p.N;
  }
  const hipError_t e = block          ? launch_grad<kE4M3, true>(g, p, s)
                       : fmt == kE4M3 ? launch_grad<kE4M3, false>(g, p, s)
                       : fmt == kE2M3 ? launch_grad<kE2M3, false>(g, p, s)
                       : fmt == kE3M2 ? launch_grad<kE3M2, false>(g, p, s)
                                      : launch_grad<kE2M1, false>(g, p, s);
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", who, hipGetErrorString(e));
    return MXL_EHIP;
  }
  if (g.S > 1) {
    input_grad_join_kernel<<<dim3((unsigned)ceil_div(M * K, 1024)), 256, 0, s>>>(p.partial, g.S, M, K, p.out, ldo);
    MXL_CHECK_LAUNCH(who);
  }
  return MXL_OK;
}

extern "C" int mxl_bias_grad(const void* dy, int64_t M, int64_t N, int64_t lddy, void* out, void* stream) {
  const char* who = "mxl_bias_grad";
  MXL_CHECK_ARG(M >= 0 && N > 0 && N <= (1 << 22), "%s: need M >= 0 and 0 < N <= 2^22 (M=%lld N=%lld)", who, (long long)M,
                (long long)N);
  MXL_CHECK_ARG(lddy >= N && (((uintptr_t)dy | (uintptr_t)out) & 1) == 0, "%s: need lddy >= N", who);
  const bool whole = lddy % 8 == 0 && ((uintptr_t)dy & 15) == 0;
  column_sum_kernel<<<dim3((unsigned)ceil_div(N, 64)), 1024, 0, (hipStream_t)stream>>>((const uint16_t*)dy, M, N, lddy,
                                                                                     whole, (uint16_t*)out);
  MXL_CHECK_LAUNCH(who);
  return MXL_OK;
}

extern "C" int64_t mxl_input_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int block) {
  return input_grad_bytes(M, N, K, block);
}

extern "C" int mxl_input_grad_plan_name(int64_t M, int64_t N, int64_t K, int fmt, int block, char* buf, int64_t len) {
  MXL_CHECK_ARG(M > 0 && M <= 0x7FFFFFFF && N > 0 && N <= (1 << 22) && K > 0 && K <= (1 << 22) && K % 128 == 0 && buf,
                "mxl_input_grad_plan_name: bad shape");
  const GradPlan g = grad_plan(M, N, K, block != 0);
  const int n = snprintf(buf, len > 0 ? (size_t)len : 0, "input_grad_kernel<%d,%d,%d,%s>%s", fmt, g.TM, g.TK,
                         block ? "true" : "false", g.S > 1 ? " + input_grad_join_kernel" : "");
  MXL_CHECK_ARG(n < len, "plan name needs %d bytes", n + 1);
  return MXL_OK;
}

extern "C" int mxl_input_grad(const void* dy, int64_t M, int64_t N, int64_t lddy, const void* w_tiled, const void* sw,
                              int64_t K, int fmt, int block, void* out, int64_t ldo, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  return input_grad("mxl_input_grad", dy, M, N, lddy, w_tiled, sw, K, fmt, block, out, ldo, workspace, workspace_bytes,
                    nullptr, stream);
}
