// One output tile of the 2 x 2-wave GEMM on gfx950 (MX and block-FP8 weights): the device
// body of the dense kernels of gemm_tile.hip and the grouped ones of gemm_tile_grouped.hip.
// A stage is 128 bytes of an activation row: K128 of 8-bit activations, or K256 of MXFP4 ones
// (E2M1 weights take E2M1 activations), whose two K128 slices are an MFMA each, at half the time.
//
// What bounds it.  At 128 x 128 tiles per workgroup every K128 stage moves as many LDS
// bytes as the LDS serves in the time of its MFMAs, so the wide kernel (gemm_wide.hip)
// stays near a fifth of the MFMA peak however its copies are scheduled.  Here four waves
// in a 2 x 2 arrangement own 16 MTW x 16 NTW outputs each (128 x 128 at MTW = NTW = 8, a
// 256 x 256 workgroup tile): per stage the LDS moves 128 KiB of fragment reads and 64 KiB
// of copies (1536 cycles at 128 bytes per cycle) under 2048 cycles of MFMAs, and each
// byte from L2 feeds twice the flops.
//
// Pipeline.  The operands of a stage arrive as four units, the upper and lower half of
// every wave's rows (A0, A1) and columns (B0, B1), each in its own LDS slot, two to four
// stages deep: as many as the workgroups of a CU leave room for, since the copies in flight are
// what a launch with cold weights waits on.  A stage is four quadrants of (MTW / 2) (NTW / 2) MFMAs, walked so
// that consecutive quadrants share one half:
//   even stages (A0,B0) (A0,B1) (A1,B1) (A1,B0), odd stages (A0,B1) (A0,B0) (A1,B0) (A1,B1)
// so one register copy of each half suffices: the unit a quadrant needs next is read from
// LDS while the previous quadrant's MFMAs run, into registers whose last use is behind it.
// Twice per stage a barrier hands over two units and frees the two slots read before it,
// into which the copies of `depth` stages ahead are issued (vmcnt counts them: loads complete
// in issue order), so all but half a stage of the ring is in flight.
//
// Measured, weights rotated out of the caches (us, the tiles of waves side by side or, where
// they do not run, the generic kernel before): W6A8 4096 x 17408 x 5120 665 -> 302 (2.4 PFLOP/s),
// 1024 x 17408 x 5120 150 -> 95, 48 x 17408 x 5120 51 -> 23.4 (2.9 TB/s of weights); block-FP8 512
// x 18432 x 2560 55.5 -> 36.2, 32 x 18432 x 2560 29.3 -> 13.5 (3.5 TB/s); MXFP8 512 x 2560 x 9216
// 27.9 -> 25.8.  The 256 x 256 tile is bound by its MFMAs at the clock that the power limit leaves (W6A8
// 4096 x 17408 x 5120: MFMAs busy 58 % of the cycles, 0.6 LDS reads each), the smaller ones by their LDS
// traffic (1.3 to 1.7 reads per MFMA; 8-byte FP6 reads with bank conflicts) and, in the last round, the
// epilogue.
//
// The weights take the MFMA's A operand and the activations its B operand, so a lane holds
// four consecutive output columns of one row (8-byte stores), and in block-FP8 its four
// sums share one activation scale.
#pragma once

#include <stdio.h>

#include "adapters.h"
#include "fp4.h"
#include "gate_act.h"
#include "gemm_wide.h"

// the copies set M0 (the LDS base of a global->LDS load) themselves
#pragma clang diagnostic ignored "-Winline-asm"

namespace mxl {

typedef __attribute__((address_space(3))) uint8_t tile_lds_u8;

__device__ __forceinline__ uint32_t tile_lds(const uint8_t* p) { return (uint32_t)(uintptr_t)(const tile_lds_u8*)p; }

// Lane i copies 16 (4) bytes from base + voff to LDS [lds + 16 i] ([lds + 4 i]); base and
// lds are wave-uniform.
__device__ __forceinline__ void tile_copy16(const uint8_t* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "m0");
}
__device__ __forceinline__ void tile_copy4(const uint8_t* base, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(voff), "s"(base) : "m0");
}

// All but the newest N copies of this wave have landed and its LDS reads are done, then the
// barrier (no memory fence: it would drain the copies in flight).
template <int N>
__device__ __forceinline__ void tile_wait() {
  static_assert(N >= 0 && N <= 63, "vmcnt immediate");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}
// Piece permutation of row r (0..15) of an m-tile stored as whole 128-byte rows: piece p
// sits at 128 (r % 8) + 16 (p ^ tile_swz(r)) of its 1 KiB chunk, so that the fragment reads
// (lane 16 q + r: row r, pieces q and 4 + q) are free of bank conflicts.
__device__ __forceinline__ int tile_swz(int r) { return ((r >> 1) ^ ((r & 1) << 2)) & 7; }

template <int J>
struct Slice { static constexpr int value = J; };

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v6i __attribute__((ext_vector_type(6)));
template <int FMT>
struct TileB { typedef v8i type; };
template <>
struct TileB<kE2M3> { typedef v6i type; };
template <>
struct TileB<kE3M2> { typedef v6i type; };
// MXFP4, weights and activations alike: a lane's operands of the stage's two slices
struct TileFp4 { v4i half[2]; };
template <>
struct TileB<kE2M1> { typedef TileFp4 type; };
template <int FMT>
struct TileA { typedef v8i type; };
template <>
struct TileA<kE2M1> { typedef TileFp4 type; };

// c += W A^T for one 16 x 16 tile over a K128 slice, J the slice's byte of the packed E8M0
// operands.  Written as assembly so that the accumulator is updated in place: with 256
// accumulator registers live the compiler's allocator finds no room to rename one, and moves
// whole tiles between register files instead (measured on its output: several hundred moves
// and spills per stage).  The caller keeps two instructions between a VALU write of an
// operand and its use, and waits out the last MFMA before it or the compiler reads an accumulator
// (tests/test_mfma_hazards_host.py scans the built code for both).
template <int FMT, int J>
__device__ __forceinline__ void tile_mfma(v4f& c, const typename TileB<FMT>::type& w, const v8i& a, uint32_t sw,
                                          uint32_t sa) {
#define MXL_TILE_MFMA(SEL_, FMT_)                                                                                   \
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " SEL_ FMT_                                \
               : "+a"(c) : "v"(w), "v"(a), "v"(sw), "v"(sa))
#define MXL_TILE_MFMA_J(FMT_)                                                              \
  if constexpr (J == 0) MXL_TILE_MFMA("op_sel_hi:[0,0,0]", FMT_);                          \
  else if constexpr (J == 1) MXL_TILE_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]", FMT_);      \
  else if constexpr (J == 2) MXL_TILE_MFMA("op_sel_hi:[1,1,0]", FMT_);                     \
  else MXL_TILE_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]", FMT_)
  if constexpr (FMT == kE4M3) { MXL_TILE_MFMA_J(""); }
  else if constexpr (FMT == kE2M3) { MXL_TILE_MFMA_J(" cbsz:2"); }
  else { MXL_TILE_MFMA_J(" cbsz:3"); }
}
template <int J>
__device__ __forceinline__ void tile_mfma_fp4(v4f& c, const v4i& w, const v4i& a, uint32_t sw, uint32_t sa) {
  MXL_TILE_MFMA_J(" cbsz:4 blgp:4");
}
#undef MXL_TILE_MFMA_J
#undef MXL_TILE_MFMA

// An accumulator's values, read where they are used (left to the compiler, all of them are
// copied to vector registers at the end of the loop, more than there are)
__device__ __forceinline__ v4f tile_values(const v4f& c) {
  v4f v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(x) : "a"(c[e]));
    v[e] = x;
  }
  return v;
}

template <int MTW, int NTW>
struct TileShape {
  static constexpr int BM = 32 * MTW, BN = 32 * NTW;  // workgroup tile
  static constexpr int AU = MTW * 2048, BU = NTW * 2048;  // bytes of an A / B unit
  static constexpr int CA = MTW / 2, CB = NTW / 2;    // copies per wave of a unit (1 KiB each)
  static constexpr int HALF = CA + CB;                // copies per wave of half a stage (one A and one B unit)
};

// Stages of the LDS ring.  SHARED: of the workgroups that share a CU (RESIDENT of them); LONE:
// where the launch has too few for that, four, so that they keep as much in flight.
template <int MT, int NT>
struct TileDepth {
  static constexpr int RESIDENT = MT * NT > 16 ? 1 : MT * NT > 4 ? 2 : 4;
  static constexpr int SHARED = MT * NT > 32 || MT * NT == 16 || MT * NT == 4 ? 2 : 3;
  static constexpr int LONE = MT * NT > 16 ? SHARED : 4;
  // most workgroups per CU that still leave room for LONE stages each
  static constexpr int LONE_MAX = MT * NT == 4 ? 2 : 1;
  // of a tile's quarters, in the LDS of the launch
  static constexpr int QUARTER = 4;
};

// Of a launch of `grid` workgroups on `cus` CUs: the stages of its ring, and " (depth D)" or " (depth D, quarters)" for the
// name of its plan.
inline int tile_depth(const WideConfig& c, int64_t grid, int64_t cus) {
#define MXL_DEPTH(MT_, NT_) \
  if (c.MT == MT_ && c.NT == NT_) return grid <= TileDepth<MT_, NT_>::LONE_MAX * cus ? TileDepth<MT_, NT_>::LONE : TileDepth<MT_, NT_>::SHARED;
  MXL_DEPTH(16, 4) MXL_DEPTH(8, 4) MXL_DEPTH(8, 2) MXL_DEPTH(8, 1) MXL_DEPTH(4, 2) MXL_DEPTH(4, 1)
#undef MXL_DEPTH
  return 0;
}
inline int tile_plan_name(const char* kernel, const char* last, const WideConfig& c, const WideGrid& g, int64_t grid, int fmt,
                          char* buf, int64_t len) {
  const int n = snprintf(buf, len > 0 ? (size_t)len : 0, "%s<%d,%d,%d,%s> (depth %d%s)", kernel, fmt, c.MT, c.NT, last,
                         tile_depth(c, grid, cu_count()), grid > g.tail0 ? ", quarters" : "");
  MXL_CHECK_ARG(n < len, "plan name needs %d bytes", n + 1);
  return MXL_OK;
}

// What a tile's epilogue does with its sums.  All but the first pair columns of a merged gate/up weight (W = gate rows
// then up rows, I of each): half of a wave's n-tiles are gate columns, half the up columns of the same.
//   kEpiSwigluFp4  MXFP4 codes and scales of bf16(bf16(silu(gate)) up) (p.mid_codes, p.mid_scales), I % 64 == 0
//   kEpiGated      act(gate) up, rounded once to bf16 (p.out [M, I]), I % 16 == 0
//   kEpiGatedGrad  with dh [M, I] of that output, dh up act'(gate) and dh act(gate) (p.out [M, 2 I])
enum TileEpi : int { kEpiStore = 0, kEpiSwigluFp4 = 1, kEpiGated = 2, kEpiGatedGrad = 3 };
struct TileGate {
  int act = 0;                   // kActSilu, kActGeluTanh
  const uint16_t* dh = nullptr;  // rows of lddh
  int64_t lddh = 0;
};

// What a workgroup computes: rows row0 .. row_hi - 1 (at most BM of them stored) by n-block
// nb, super-tiles kb .. ke - 1.  part: instead of output elements the tile's fp32 partials as
// one block in MFMA fragment order: fragment f = m-tile * (BN / 16) + n-tile is 64 lanes x 4
// floats, lane (q, r) holding columns 4 q .. 4 q + 3 of row r.
struct TileWork {
  int row0, row_hi, nb, kb, ke;
  const uint8_t* w;
  const uint8_t* sw;
  float* part;
};

// LDS of a tile, from its base: the scale slots of two super-tiles (MX: the rows' E8M0 and the
// n-tiles' tiled E8M0 dwords; block-FP8: the rows' fp32 scales [4][BM] and the weight block
// scales of the K range), then `depth` stages of the four units A0, A1, B0, B1.
template <int MTW, int NTW, bool BLOCK>
struct TileLds {
  using S = TileShape<MTW, NTW>;
  static constexpr int SA = 0;
  static constexpr int SB = 2 * S::BM * 16;
  static constexpr int RING = SB + (BLOCK ? (S::BN + 127) / 128 * kWideBlockStages * 4 : 2 * S::BN * 16);
  static constexpr int STAGE = 2 * S::AU + 2 * S::BU;
  static constexpr int bytes(int depth) { return RING + depth * STAGE; }
};

// a_row(row): the activation row of output row `row` (rows past the last: any valid one).
// ADD (whole K): to the sums of rows with an adapter its low-rank part is added, ahead of any rounding; the kernel's third
// argument, a RowAdapters behind GemmParams and WideGrid, says what.  Returns whether the wave left out values that are not
// finite (add_odd adds them).
constexpr int kAddOffset = (sizeof(GemmParams) + 7) / 8 * 8 + (sizeof(WideGrid) + 7) / 8 * 8;
template <int FMT, int MTW, int NTW, bool BLOCK, int DEPTH, int EPI = kEpiStore, bool ADD = false, class Row>
__device__ __forceinline__ bool tile_gemm(const GemmParams& p, const TileWork& w, uint8_t* lds, Row&& a_row,
                                          const TileGate& gate = TileGate()) {
  constexpr bool SWIGLU = EPI == kEpiSwigluFp4, GATED = EPI == kEpiGated || EPI == kEpiGatedGrad;
  static_assert(!GATED || !BLOCK, "gate and up columns have block scales of their own");
  static_assert(!BLOCK || FMT == kE4M3, "block-FP8 weights are E4M3");
  using S = TileShape<MTW, NTW>;
  using L = TileLds<MTW, NTW, BLOCK>;
  constexpr int MH = MTW / 2, NH = NTW / 2, CH = FmtTraits<FMT>::CH;
  constexpr bool FP4 = FMT == kE2M1;
  constexpr int SPT = FP4 ? 2 : 4;  // stages of a 512-wide super-tile
  static_assert(!SWIGLU || (FP4 && NH == 2), "a wave's gate columns are a block of 32");
  // A stage's copies take the slots of the stage DEPTH before it in the order those fall free.
  // At an odd depth that stage reads its B units in the other order, so the B unit this stage
  // needs first is copied second, and the barrier that hands it over waits for CB copies more.
  constexpr int ODD = DEPTH & 1 ? S::CB : 0;
  const int t = threadIdx.x, lane = t & 63;
  const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wv >> 1, wn = wv & 1;
  const int r = lane & 15, q = lane >> 4;

  // stage and tile indices in 32 bits (the host bounds the operands below 4 GiB)
  const int slices = (int)(p.K / 128), T = FP4 ? (slices + 1) / 2 : slices;  // K128 slices, stages
  const int KT = (int)p.KT, ntiles = (int)((p.N + 15) / 16), kb = w.kb, ke = w.ke;
  // stages SPT kb .. te - 1; an odd count runs one more (end), whose weights (past K) are zero
  const int te = SPT * ke < T ? SPT * ke : T, end = (te + 1) & ~1;
  const int nt_base = w.nb * (S::BN / (EPI != kEpiStore ? 32 : 16)), up = ntiles / 2;
  // n-tile k of half h of wave column c
  auto n_tile = [&](int c, int h, int k) -> int {
    if constexpr (SWIGLU) {
      return nt_base + c * NH + k + h * up;
    } else if constexpr (GATED) {
      const int nt = nt_base + c * NH + k;
      return (nt < up ? nt : up - 1) + h * up;
    } else {
      const int nt = nt_base + c * NTW + h * NH + k;
      return nt < ntiles ? nt : ntiles - 1;
    }
  };

  // copy sources.  A unit h: chunk c = CA wv + u holds rows 8 (c % 2) .. + 7 of the unit's
  // m-tile e = c / 2 (wave row e / MH, its m-tile h MH + e % MH); rows past M re-read the last
  uint32_t a_off[2][S::CA];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int u = 0; u < S::CA; ++u) {
      const int c = S::CA * wv + u, e = c >> 1, cr = 8 * (c & 1) + (lane >> 3);
      const int row = a_row(w.row0 + ((e / MH) * MTW + h * MH + e % MH) * 16 + cr);
      a_off[h][u] = (uint32_t)row * (uint32_t)p.lda + 16 * ((lane & 7) ^ tile_swz(cr));
    }
  // MXFP4: the last of an odd number of slices is half a stage, whose other half is the next row's first
  // bytes (the weights there are zero, and E2M1 has no NaN) or, past the last row, its last 16 again
  const uint32_t a_last = FP4 ? (uint32_t)(p.a_rows * p.lda - 16) : 0;
  // B unit h: chunk c = CB wv + u is chunk c % 2 of the unit's n-tile e = c / 2
  const uint8_t* b_src[2][(S::CB + 1) / 2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int u = 0; u < S::CB; u += 2) {
      const int e = (S::CB * wv + u) >> 1;
      const int nt = n_tile(e / NH, h, e % NH);
      b_src[h][u / 2] = w.w + (int64_t)nt * KT * (CH * 1024) + (S::CB == 1 ? (wv & 1) * 1024 : 0);
    }
  const uint32_t lane16 = (uint32_t)lane * 16;
  const uint32_t lds_a = tile_lds(lds + L::RING) + S::CA * wv * 1024;
  const uint32_t lds_b = tile_lds(lds + L::RING) + 2 * S::AU + S::CB * wv * 1024;
  // copies of stage tt into the slot at `slot`
  auto copy_a = [&](int h, int u, int tt, int slot) {
    const int tc = tt < te ? tt : te - 1;  // an odd count's last stage: a valid one again
    uint32_t off = a_off[h][u];
    if constexpr (FP4) off = __builtin_elementwise_min(off, a_last - (uint32_t)tc * 128);
    tile_copy16(p.a + (uint32_t)tc * 128, off, lds_a + slot + h * S::AU + u * 1024);
  };
  auto copy_b = [&](int h, int u, int tt, int slot) {
    const int j = tt & (SPT - 1), c0 = FMT == kE4M3 || FP4 ? 2 * j : (3 * j) >> 1;
    tile_copy16(b_src[h][u >> 1] + (uint32_t)((tt >> (FP4 ? 1 : 2)) * CH + c0 + (u & 1)) * 1024, lane16,
                lds_b + slot + h * S::BU + u * 1024);
  };
  // MX: scales of super-tile kt, 64 rows (16 bytes each) and four n-tiles per wave (where the
  // tile has fewer, several waves copy the same).  A row's window of a part super-tile ends
  // with the row.  Swizzled scales, and rows shorter than a window: dword by dword, 16 rows a
  // copy, clamped to the last slice.  Block-FP8: the four groups' fp32 scales of the rows, one
  // group per wave.
  const bool dwords = !BLOCK && ((!FP4 && p.sa_swz) || p.K < kTileK);  // (MXFP4 scales are logical)
  const uint32_t srow = (uint32_t)(p.K / 32);
  const int swa = wv % (S::BM / 64), swb = wv % (S::BN / 64);
  uint32_t sa_off[BLOCK ? S::BM / 64 : 1];
  if constexpr (BLOCK) {
#pragma unroll
    for (int c = 0; c < S::BM / 64; ++c) sa_off[c] = (uint32_t)a_row(w.row0 + 64 * c + lane) * 4;
  } else {
    sa_off[0] = (uint32_t)a_row(w.row0 + 64 * swa + lane) * srow;
  }
  const int sc = 4 * swb + (lane >> 4), snt = n_tile(sc / NTW, sc % NTW / NH, sc % NH);
  const uint32_t sb_off = (uint32_t)snt * (uint32_t)KT * 256 + 16 * (lane & 15);
  const uint32_t lds_sa = tile_lds(lds + L::SA) + (BLOCK ? wv * S::BM * 4 : 64 * swa * 16);
  const uint32_t lds_sb = tile_lds(lds + L::SB) + 4 * swb * 256;
  // (FIRST: of the range's first super-tile; MXFP4's others belong to rows of a window and more)
  auto copy_scales = [&](int kt, auto FIRST) {
    const int st = kt & 1;
    const int kc = kt < ke ? kt : ke - 1;
    if constexpr (BLOCK) {
      const int g = 4 * kc + wv < T ? 4 * kc + wv : T - 1;
#pragma unroll
      for (int c = 0; c < S::BM / 64; ++c)
        tile_copy4(static_cast<const uint8_t*>(p.sa) + (int64_t)g * p.M * 4, sa_off[c],
                   lds_sa + st * (S::BM * 16) + 256 * c);
    } else {
      if (dwords && (!FP4 || decltype(FIRST)::value)) {
        const int slice = 4 * kc + (lane & 3) < slices ? 4 * kc + (lane & 3) : slices - 1;
#pragma unroll
        for (int u = 0; u < S::BM / 64; ++u) {
          const int c = wv + 4 * u, row = a_row(w.row0 + 16 * c + (lane >> 2));
          tile_copy4(static_cast<const uint8_t*>(p.sa),
                     FP4 ? (uint32_t)row * srow + 4 * slice : (uint32_t)(sa_row_offset(p, row) + slice * (int)p.sa_ss),
                     tile_lds(lds + L::SA) + st * (S::BM * 16) + 256 * c);
        }
      } else {
        const uint32_t win = 16 * kc + 16 <= (int)srow ? 16 * kc : srow - 16;
        tile_copy16(static_cast<const uint8_t*>(p.sa) + win, sa_off[0], lds_sa + st * (S::BM * 16));
      }
      tile_copy16(w.sw + (uint32_t)kc * 256, sb_off, lds_sb + st * (S::BN * 16));
    }
  };
  const int tb = SPT * kb;
  if constexpr (BLOCK) {
    // the weight block scales of the split's stages, one LDS row per 128 columns (read in the
    // loop from global memory they would be compiler-counted loads, whose waits drain the copies)
#pragma unroll
    for (int c = 0; c < (S::BN + 127) / 128; ++c) {
      const int64_t blocks = (p.N + 127) / 128, want = (int64_t)w.nb * S::BN / 128 + c;
      const uint8_t* src = w.sw + ((want < blocks ? want : blocks - 1) * T + tb) * 4;
      for (int k = 64 * wv; k < te - tb; k += 256) {
        const int at = k + lane < te - tb ? k + lane : te - tb - 1;
        tile_copy4(src, (uint32_t)at * 4, tile_lds(lds + L::SB) + (c * kWideBlockStages + k) * 4);
      }
    }
  }

  v4f acc[MTW][NTW];
#pragma unroll
  for (int i = 0; i < MTW; ++i)
#pragma unroll
    for (int n = 0; n < NTW; ++n) acc[i][n] = v4f{0.f, 0.f, 0.f, 0.f};
  typename TileA<FMT>::type a[2][MH];
  typename TileB<FMT>::type b[2][NH];
  uint32_t sa[MTW], sb[NTW];         // MX: packed E8M0 bytes of the super-tile's slices
  float fa[BLOCK ? MTW : 1][4], fb[4];  // block-FP8: the super-tile's activation and weight scales

  // fragment reads: two LDS reads each
  const int sw = tile_swz(r);
  const int ra = wm * MH * 2048 + (r >> 3) * 1024 + (r & 7) * 128;
  const int ra_lo = ra + 16 * (q ^ sw), ra_hi = ra + 16 * ((q + 4) ^ sw);
  const int rb = wn * NH * 2048 + lane * 16;
  auto read_a = [&](int h, int i, int half, int slot) {  // K 16 q .. (half 0) or 64 + 16 q .. (half 1)
    const uint8_t* src = lds + L::RING + slot + (half ? ra_hi : ra_lo) + h * S::AU + i * 2048;
    if constexpr (FP4) {  // (slice 0 or 1 of the stage, K 32 q .. of it)
      a[h][i].half[half] = *reinterpret_cast<const v4i*>(src);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(src);
      a[h][i][4 * half] = (int)v.x; a[h][i][4 * half + 1] = (int)v.y;
      a[h][i][4 * half + 2] = (int)v.z; a[h][i][4 * half + 3] = (int)v.w;
    }
  };
  auto read_b = [&](int h, int n, int half, int slot, int odd) {  // odd: the parity of the stage's slice
    const uint8_t* src = lds + L::RING + 2 * S::AU + slot + rb + h * S::BU + n * 2048;
    auto& x = b[h][n];
    if constexpr (FP4) {
      x.half[half] = *reinterpret_cast<const v4i*>(src + 1024 * half);
    } else if constexpr (FMT == kE4M3) {
      const uint4 v = *reinterpret_cast<const uint4*>(src + 1024 * half);
      x[4 * half] = (int)v.x; x[4 * half + 1] = (int)v.y; x[4 * half + 2] = (int)v.z; x[4 * half + 3] = (int)v.w;
    } else if (!odd) {  // even slice: the first chunk and 8 bytes of the second
      if (half == 0) {
        const uint4 v = *reinterpret_cast<const uint4*>(src);
        x[0] = (int)v.x; x[1] = (int)v.y; x[2] = (int)v.z; x[3] = (int)v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(src + 1024);
        x[4] = (int)v.x; x[5] = (int)v.y;
      }
    } else {
      if (half == 0) {
        const uint2 v = *reinterpret_cast<const uint2*>(src + 8);
        x[0] = (int)v.x; x[1] = (int)v.y;
      } else {
        const uint4 v = *reinterpret_cast<const uint4*>(src + 1024);
        x[2] = (int)v.x; x[3] = (int)v.y; x[4] = (int)v.z; x[5] = (int)v.w;
      }
    }
  };
  // the lane's E8M0 bytes of a super-tile: byte j of sa[i] is block 4 j + q of its row
  const uint32_t sel_lo = 0x0c0c0400u + 0x0101u * q, sel_hi = 0x04000c0cu + 0x01010000u * q;
  auto read_scales = [&](int kt) {
    const int st = kt & 1;
    if constexpr (BLOCK) {
#pragma unroll
      for (int i = 0; i < MTW; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          fa[i][j] = *reinterpret_cast<const float*>(lds + L::SA + st * (S::BM * 16) +
                                                     (j * S::BM + (wm * MTW + i) * 16 + r) * 4);
      const v4f f = *reinterpret_cast<const v4f*>(lds + L::SB +
                                                  ((S::BN > 128 ? wn : 0) * kWideBlockStages + 4 * kt - tb) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) fb[j] = f[j];
      if (4 * kt + 4 > T) {  // the stage past an odd count adds 0 * 0, whatever the last scales are
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          fb[j] = 4 * kt + j < T ? fb[j] : 0.0f;
#pragma unroll
          for (int i = 0; i < MTW; ++i) fa[i][j] = 4 * kt + j < T ? fa[i][j] : 0.0f;
        }
      }
    } else {
      // a part super-tile's window ends with the row: its first byte moves to byte 0
      const int shift = 4 * kt + 4 <= slices || dwords ? 0 : 8 * (4 * kt + 4 - slices);
#pragma unroll
      for (int i = 0; i < MTW; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(lds + L::SA + st * (S::BM * 16) + ((wm * MTW + i) * 16 + r) * 16);
        sa[i] = (__builtin_amdgcn_perm(x.y, x.x, sel_lo) | __builtin_amdgcn_perm(x.w, x.z, sel_hi)) >> shift;
      }
#pragma unroll
      for (int n = 0; n < NTW; ++n)
        sb[n] = *reinterpret_cast<const uint32_t*>(lds + L::SB + st * (S::BN * 16) + (wn * NTW + n) * 256 + lane * 4);
    }
  };

  // Stage tt (slice J of its pair) from the slot at `cur`, the next stage's at `nxt`: four
  // quadrants of Q MFMAs, after each MFMA its share of the reads of the next unit and of the
  // copies of DEPTH stages ahead (into the slots that this stage frees).  LEFT: the stages left,
  // this one included, at the end (0: more than four); then copies would lie past it, and fewer
  // half-stages of copies may stay in flight at a barrier (those after the units it hands over).
  auto stage = [&](auto J, auto LEFT, int tt, int cur, int nxt) {
    constexpr int st = decltype(J)::value & 1, x = st, y = 1 - st, left = decltype(LEFT)::value;
    constexpr bool ahead = left == 0 || left > DEPTH;
    constexpr int full = 2 * DEPTH - 2;
    constexpr int Q = MH * NH;
    v4f raw[3];
    float f[BLOCK ? MTW : 1];
    if constexpr (BLOCK) {
#pragma unroll
      for (int i = 0; i < MTW; ++i) f[i] = fa[i][st] * fb[st];
    }
    // block-FP8: acc = fma(raw, sa sb, acc) of the stage's g-th MFMA, two MFMAs after it
    auto fold = [&](int g) {
      const int s = g / Q, k = g % Q, i = (s >> 1) * MH + k / NH, n = (s == 0 || s == 3 ? x : y) * NH + k % NH;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][n][e] = __builtin_fmaf(raw[g % 3][e], f[BLOCK ? i : 0], acc[i][n][e]);
    };
    auto quad = [&](auto QI, auto&& between) {
      constexpr int s = decltype(QI)::value, ah = s >> 1, bh = s == 0 || s == 3 ? x : y;
      if constexpr (FP4) {  // the first slice's Q MFMAs, then the second's: a share after every two
        auto slice = [&](auto H) {
          constexpr int hf = decltype(H)::value;
#pragma unroll
          for (int i = 0; i < MH; ++i)
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              tile_mfma_fp4<2 * st + hf>(acc[ah * MH + i][bh * NH + n], b[bh][n].half[hf], a[ah][i].half[hf],
                                        sb[bh * NH + n], sa[ah * MH + i]);
              const int m = hf * Q + i * NH + n;
              if (m & 1) between(m >> 1);
            }
        };
        slice(Slice<0>{});
        slice(Slice<1>{});
        return;
      }
#pragma unroll
      for (int i = 0; i < MH; ++i)
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const int k = i * NH + n, g = s * Q + k;
          if constexpr (FP4) {
          } else if constexpr (BLOCK) {
            const v4f z = {0.f, 0.f, 0.f, 0.f};
            raw[g % 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[bh][n], a[ah][i], z, kE4M3, kE4M3, 0, 127, 0,
                                                                          127);
            if (g >= 2) fold(g - 2);
          } else {
            tile_mfma<FMT, decltype(J)::value>(acc[ah * MH + i][bh * NH + n], b[bh][n], a[ah][i], sb[bh * NH + n],
                                               sa[ah * MH + i]);
          }
          between(k);
          if constexpr (BLOCK) __builtin_amdgcn_sched_barrier(0);
        }
    };
    // a unit's `total` reads or copies spread over the Q MFMAs: the share of MFMA k
    auto reads_a = [&](int k, int h, int slot) {
      constexpr int R = (2 * MH + Q - 1) / Q;
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (k * R + u < 2 * MH) read_a(h, (k * R + u) >> 1, (k * R + u) & 1, slot);
    };
    auto reads_b = [&](int k, int h, int slot, int odd) {
      constexpr int R = (2 * NH + Q - 1) / Q;
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (k * R + u < 2 * NH) read_b(h, (k * R + u) >> 1, (k * R + u) & 1, slot, odd);
    };
    auto copies_a = [&](int k, int h) {
      if constexpr (!ahead) {
      } else if constexpr (Q >= S::CA) {
        if (k % (Q / S::CA) == Q / S::CA - 1) copy_a(h, k / (Q / S::CA), tt + DEPTH, cur);
      } else {
#pragma unroll
        for (int u = 0; u < S::CA / Q; ++u) copy_a(h, k * (S::CA / Q) + u, tt + DEPTH, cur);
      }
    };
    auto copies_b = [&](int k, int h) {
      if constexpr (!ahead) {
      } else if constexpr (Q >= S::CB) {
        if (k % (Q / S::CB) == Q / S::CB - 1) copy_b(h, k / (Q / S::CB), tt + DEPTH, cur);
      } else {
#pragma unroll
        for (int u = 0; u < S::CB / Q; ++u) copy_b(h, k * (S::CB / Q) + u, tt + DEPTH, cur);
      }
    };
    tile_wait<S::HALF * (left && 2 * left - 2 < full ? 2 * left - 2 : full)>();
    if constexpr (FP4 && st == 0) {
      // every wave has read this super-tile's scales: their slot takes those of the one after the next.  (A
      // super-tile is two stages, which a copy into the other slot one ahead could outlast: seven half-stages of
      // copies follow it before the wait ahead of its read, which leaves at most six in flight.)
      if ((tt >> 1) + 2 < ke) copy_scales((tt >> 1) + 2, Slice<0>{});
    }
    quad(Slice<0>{}, [&](int k) { reads_b(k, y, cur, st); copies_a(k, 0); });
    quad(Slice<1>{}, [&](int k) { reads_a(k, 1, cur); copies_b(k, x); });
    if constexpr (left != 1) tile_wait<S::HALF * (ahead ? full : 2 * left - 3) - ODD>();
    quad(Slice<2>{}, [&](int k) { reads_a(k, 0, nxt); copies_b(k, y); });
    quad(Slice<3>{}, [&](int k) { reads_b(k, y, nxt, 1 - st); copies_a(k, 1); });
    if constexpr (BLOCK) {
      fold(4 * Q - 2);
      fold(4 * Q - 1);
    }
  };

  typedef const __attribute__((address_space(4))) uint8_t* kernarg_t;
  if constexpr (ADD) {  // the rows' adapters, behind the ring, for the end
    const kernarg_t at = (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr() + kAddOffset;
    const int32_t* const ids = ((const __attribute__((address_space(4))) RowAdapters*)at)->ids;
    const int wr = 64 * (wv % (S::BM / 64));
    tile_copy4(reinterpret_cast<const uint8_t*>(ids + w.row0), 4 * (uint32_t)(a_row(w.row0 + wr + lane) - w.row0),
               tile_lds(lds + L::bytes(DEPTH)) + 4 * wr);
  }
  copy_scales(kb, Slice<1>{});
  if (FP4 && kb + 1 < ke) copy_scales(kb + 1, Slice<0>{});
  const int count = end - tb;  // stages: an even number
#pragma unroll
  for (int k = 0; k < DEPTH; ++k) {  // units in the order the loop copies them
    if (k >= 2 && k >= count) break;
    const int x = (k + DEPTH) & 1;
#pragma unroll
    for (int u = 0; u < S::CA; ++u) copy_a(0, u, tb + k, k * L::STAGE);
#pragma unroll
    for (int u = 0; u < S::CB; ++u) copy_b(x, u, tb + k, k * L::STAGE);
#pragma unroll
    for (int u = 0; u < S::CB; ++u) copy_b(1 - x, u, tb + k, k * L::STAGE);
#pragma unroll
    for (int u = 0; u < S::CA; ++u) copy_a(1, u, tb + k, k * L::STAGE);
  }
  if (DEPTH > 2 && count == 2) tile_wait<S::HALF * 3 - ODD>();
  else tile_wait<S::HALF * (2 * DEPTH - 1) - ODD>();
#pragma unroll
  for (int i = 0; i < MH; ++i) { read_a(0, i, 0, 0); read_a(0, i, 1, 0); }
#pragma unroll
  for (int n = 0; n < NH; ++n) { read_b(0, n, 0, 0, 0); read_b(0, n, 1, 0, 0); }

  // two stages per iteration, byte pairs 0, 1 then 2, 3 of the packed scales
  int cur = 0;  // the slot of the pair's first stage
  auto pair = [&](auto LEFT, int pr) {  // LEFT: the stages left at the pair's first, 0 for many
    const int kt = FP4 ? pr : pr >> 1;
    if (FP4 || (pr & 1) == 0) {
      if (!FP4 && kt + 1 < ke) copy_scales(kt + 1, Slice<0>{});
      read_scales(kt);  // landed: the copies of the stages before this one were issued after them
    } else if constexpr (BLOCK) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        fb[j] = fb[j + 2];
#pragma unroll
        for (int i = 0; i < MTW; ++i) fa[i][j] = fa[i][j + 2];
      }
    } else {
#pragma unroll
      for (int i = 0; i < MTW; ++i) sa[i] >>= 16;
#pragma unroll
      for (int n = 0; n < NTW; ++n) sb[n] >>= 16;
    }
    if constexpr (!BLOCK) {  // (the empty statements keep the operands' last writes ahead of the s_nop)
#pragma unroll
      for (int i = 0; i < MTW; ++i)
#pragma unroll
        for (int n = 0; n < NTW; ++n) asm volatile("" : "+a"(acc[i][n]));
#pragma unroll
      for (int i = 0; i < MTW; ++i) asm volatile("" : "+v"(sa[i]));
#pragma unroll
      for (int n = 0; n < NTW; ++n) asm volatile("" : "+v"(sb[n]));
      asm volatile("s_nop 1");
    }
    constexpr int left = decltype(LEFT)::value;
    constexpr int ring = DEPTH * L::STAGE;
    const int one = cur + L::STAGE < ring ? cur + L::STAGE : 0, two = one + L::STAGE < ring ? one + L::STAGE : 0;
    stage(Slice<0>{}, Slice<left>{}, 2 * pr, cur, one);
    stage(Slice<1>{}, Slice<left ? left - 1 : 0>{}, 2 * pr + 1, one, two);
    // 64 x 64 tiles, gated ones and those with adapters: the compiler moves the accumulators after the loop, 17 states
    // and more after the last MFMA whose result takes 20
    if constexpr (!BLOCK && (GATED || ADD)) asm volatile("s_nop 4");
    else if constexpr (!BLOCK && MTW * NTW == 4) asm volatile("s_nop 2");
    cur = two;
  };
  const int last = end >> 1;  // pairs 2 kb .. last - 1; the copies end in the final one or two
  int pr = FP4 ? kb : 2 * kb;
  for (; pr + (DEPTH > 2 ? 2 : 1) < last; ++pr) pair(Slice<0>{}, pr);
  if (DEPTH > 2 && pr + 1 < last) pair(Slice<4>{}, pr++);
  pair(Slice<2>{}, pr);

  bool odd = false;
  if constexpr (ADD) {
    {
      // After the last MFMAs' results: 16 ranks an MFMA, v's halves in its two halves of K, zero in the rows of other
      // adapters than the one at hand (and B in columns of other parts).  Adapters, parts and ranks go one after the
      // other; what it costs is the wait for each one's first bytes (some 4 us on a 256 x 256 tile), not the loads: laid out
      // so that every load met whole lines, 2048 x 18432 x 2560 took 119 us against 112.
      // The arguments are read here (through a pointer that the compiler cannot see through): held in scalar registers
      // over the main loop they would spill.
      typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
      typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
      kernarg_t at = (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr() + kAddOffset;
      asm volatile("" : "+s"(at));
      const auto* const add = (const __attribute__((address_space(4))) RowAdapters*)at;
      auto pin = [&] {
#pragma unroll
        for (int i = 0; i < MTW; ++i)
#pragma unroll
          for (int n = 0; n < NTW; ++n) {
            if constexpr (BLOCK) asm volatile("" : "+v"(acc[i][n]));
            else asm volatile("" : "+a"(acc[i][n]));
          }
      };
      if constexpr (!BLOCK) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
      pin();
      int own[MTW];
#pragma unroll
      for (int i = 0; i < MTW; ++i) {
        const int row = (wm * MTW + i) * 16 + r;
        const int x = *reinterpret_cast<const int32_t*>(lds + L::bytes(DEPTH) + 4 * row);
        own[i] = w.row0 + row < w.row_hi && (uint32_t)x < (uint32_t)add->slots ? x : 0x7FFFFFFF;
      }
      // the part of a column
      auto part_of = [&](int col) {
        int of = 0;
        for (int k = 1; k < add->l.parts; ++k) of += col >= (int)add->l.cols[k] ? 1 : 0;
        return of;
      };
      // the smallest adapter past `last` of the wave's rows
      auto next = [&](int last) {
        int a = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < MTW; ++i) a = own[i] > last && own[i] < a ? own[i] : a;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
          const int b = __shfl_xor(a, d, 64);
          a = b < a ? b : a;
        }
        return __builtin_amdgcn_readfirstlane(a);
      };
      const int first = part_of(16 * n_tile(wn, 0, 0)), end = part_of(16 * n_tile(wn, 1, NH - 1));
      int a = next(-1), part = first, g = 0;
      while (a != 0x7FFFFFFF) {  // (one loop: nested ones would move the accumulators)
        asm volatile("" : "+s"(at));
        const auto* const o = (const __attribute__((address_space(4))) RowAdapters*)at;
        const int parts = o->l.parts, rank = o->l.rank, groups = o->l.groups, width = 16 * groups * parts;
        const int lo = (int)o->l.cols[part], hi = part + 1 < parts ? (int)o->l.cols[part + 1] : (int)p.N;
        const uint8_t* const mat = reinterpret_cast<const uint8_t*>(o->mat + a * o->slot_stride) + 32 * g;
        const uint8_t* const v = reinterpret_cast<const uint8_t*>(o->v) + 32 * (part * groups + g);
        const bool in = 16 * g + 8 * (q & 1) < rank;  // (ranks come in eights)
        // every lane loads, from a valid place; what does not count becomes zero
        u32x4 xv[MTW], xb[NTW];
        const uint32_t vrow = (uint32_t)(w.row0 + wm * MTW * 16 + r) * (uint32_t)(4 * width) + (q >> 1) * 2 * width + 16 * (q & 1);
#pragma unroll
        for (int i = 0; i < MTW; ++i)
          xv[i] = *reinterpret_cast<const u32x4*>(v + (own[i] == a ? vrow + (uint32_t)(64 * i) * (uint32_t)width : 0u));
#pragma unroll
        for (int n = 0; n < NTW; ++n) {
          const int col = 16 * n_tile(wn, n / NH, n % NH) + r, from = col < lo ? lo : col < hi ? col : hi - 1;
          xb[n] = *reinterpret_cast<const u32x4*>(mat + ((uint32_t)from * (uint32_t)(2 * o->ldm) + (in ? 16 * (q & 1) : 0)));
        }
#pragma unroll
        for (int i = 0; i < MTW; ++i) {
          const uint32_t m = own[i] == a ? 0xFFFFFFFFu : 0u;
          xv[i] &= u32x4{m, m, m, m};
          asm volatile("" : "+v"(xv[i]));
        }
#pragma unroll
        for (int n = 0; n < NTW; ++n) {
          const int col = 16 * n_tile(wn, n / NH, n % NH) + r;
          const uint32_t m = in && col >= lo && col < hi ? 0xFFFFFFFFu : 0u;
          xb[n] &= u32x4{m, m, m, m};
          asm volatile("" : "+v"(xb[n]));
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < MTW; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = adapter_top(top, xv[i][e]);
#pragma unroll
        for (int n = 0; n < NTW; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = adapter_top(top, xb[n][e]);
        if (__builtin_amdgcn_ballot_w64(adapter_odd(top)) != 0) {
          odd = true;
#pragma unroll
          for (int i = 0; i < MTW; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) xv[i][e] = adapter_finite(xv[i][e]);
#pragma unroll
          for (int n = 0; n < NTW; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) xb[n][e] = adapter_finite(xb[n][e]);
        }
        if (++g == groups) {
          g = 0;
          if (++part > end) {
            part = first;
            a = next(a);
          }
        }
        if constexpr (!BLOCK) asm volatile("s_nop 1");
#pragma unroll
        for (int n = 0; n < NTW; ++n)
#pragma unroll
          for (int i = 0; i < MTW; ++i) {
            if constexpr (BLOCK)
              acc[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xb[n]),
                                                                 __builtin_bit_cast(bf16x8, xv[i]), acc[i][n], 0, 0, 0);
            else
              asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[i][n]) : "v"(xb[n]), "v"(xv[i]));
          }
        if constexpr (!BLOCK) asm volatile("s_nop 15");  // (the next ranks' sums start from these results)
      }
      pin();
    }
  }
  auto values = [&](int i, int n) -> v4f {
    if constexpr (BLOCK) return acc[i][n];
    else return tile_values(acc[i][n]);
  };
  if constexpr (!BLOCK) asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");  // the last MFMAs' results
  // lane (q, r): columns 4 q .. 4 q + 3 of row r of every 16 x 16 tile
  if constexpr (SWIGLU) {
    // Against a launch of its own (us, 777 tokens top 6 of 48 experts of 1280 x 1920: product and producer 24.0 + 5.2,
    // here 22.9; 2048 top 8 of 256 of 1024 x 2048: 66 + 9.2, here 69.5).
    // The activations of bf16 gates come from the 16 KiB table (silu_math.h), staged where the ring was (arithmetic for
    // gates outside it): exp and a division take 30 instructions of each of a lane's values.
    const uint16_t* const tab = reinterpret_cast<const uint16_t*>(lds + L::RING);
    static_assert(kSiluEntries * 2 == 16 * 1024 && 2 * L::STAGE >= 16 * 1024, "four copies a wave, within the ring");
    tile_wait<0>();
#pragma unroll
    for (int u = 0; u < 4; ++u)
      tile_copy16(reinterpret_cast<const uint8_t*>(kSiluAct) + (4 * wv + u) * 1024, lane16,
                  tile_lds(lds + L::RING) + (4 * wv + u) * 1024);
    tile_wait<0>();
    auto pack = [](float x, float y) -> uint32_t {
      uint32_t d = cvt_pk_bf16(x, y);
      d = x != x ? (d & 0xFFFF0000u) | 0x7FC0u : d;
      return y != y ? (d & 0x0000FFFFu) | 0x7FC00000u : d;
    };
    const int blk = w.nb * (NTW / 2) + wn, blocks = up / 2;
#pragma unroll
    for (int i = 0; i < MTW; ++i) {
      uint32_t gd[4], ud[4], d[4];  // pairs: columns 4 q .. + 3 of the block's first 16, then of the others
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const v4f g = values(i, n), u = values(i, NH + n);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          gd[2 * n + e] = pack(g[2 * e], g[2 * e + 1]);
          ud[2 * n + e] = pack(u[2 * e], u[2 * e + 1]);
        }
      }
      if (__builtin_amdgcn_ballot_w64(!silu_in_table(uint4{gd[0], gd[1], gd[2], gd[3]})) == 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t o = silu_offsets(gd[e]) + ((gd[e] >> 3) & 0x10001000u);
          const float a0 = u2f((uint32_t)tab[o & 0xFFFFu] << 16), a1 = u2f((uint32_t)tab[o >> 16] << 16);
          d[e] = cvt_pk_bf16(a0 * u2f(ud[e] << 16), a1 * u2f(ud[e] & 0xFFFF0000u));
        }
      } else {
        float g[8], u[8], v[8];
        bf16x8_to_f32(uint4{gd[0], gd[1], gd[2], gd[3]}, g);
        bf16x8_to_f32(uint4{ud[0], ud[1], ud[2], ud[3]}, u);
        swiglu8<kFloorCarry175>(g, u, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = cvt_pk_bf16(v[2 * e], v[2 * e + 1]);
      }
      uint32_t amax = amax_bf16_bits<4, false>(d);
      amax = __builtin_elementwise_max(amax, (uint32_t)__shfl_xor((int)amax, 16, 64));
      amax = __builtin_elementwise_max(amax, (uint32_t)__shfl_xor((int)amax, 32, 64));
      const uint32_t s = scale_e2m1(amax, p.mid_carry), c = codes_e2m1(d, s);
      // lanes q and q ^ 1 make eight columns of the first half and eight of the second
      const uint32_t other = (uint32_t)__shfl_xor((int)c, 16, 64);
      const uint32_t word = q & 1 ? other >> 16 | (c & 0xFFFF0000u) : (c & 0xFFFFu) | other << 16;
      const int row = w.row0 + (wm * MTW + i) * 16 + r;
      if (row < w.row_hi) {
        const int64_t at = (int64_t)row * blocks + blk;
        reinterpret_cast<uint32_t*>(p.mid_codes)[at * 4 + (q & 1) * 2 + (q >> 1)] = word;
        if (q == 0) p.mid_scales[at] = (uint8_t)s;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    return odd;
  }
  if constexpr (GATED) {
    // Lane: four columns of one row of gate and of up, side by side in its registers.  Of two n-tiles every other 16
    // lanes change places, after which a lane stores eight columns of one of them (as the wide stores below).  dh's rows
    // are loaded a row of n-tiles ahead.
    typedef unsigned int u4 __attribute__((ext_vector_type(4)));
    const int I = 16 * up, col0 = 16 * (nt_base + wn * NH);
    auto rows = [&](auto ACT) {
      uint2 dh[2][EPI == kEpiGatedGrad ? NH : 1];
      auto load = [&](int i) {
        if constexpr (EPI == kEpiGatedGrad) {
          const int row = w.row0 + (wm * MTW + i) * 16 + r;
          const uint16_t* const src = gate.dh + (int64_t)(row < w.row_hi ? row : w.row_hi - 1) * gate.lddh;
#pragma unroll
          for (int n = 0; n < NH; ++n)
            dh[i & 1][n] = *reinterpret_cast<const uint2*>(src + (col0 + 16 * n < I ? col0 + 16 * n + 4 * q : 0));
        }
      };
      load(0);
#pragma unroll
      for (int i = 0; i < MTW; ++i) {
        const int row = w.row0 + (wm * MTW + i) * 16 + r;
        uint16_t* const out = p.out + (int64_t)row * p.ldc;
        if (i + 1 < MTW) load(i + 1);
        uint32_t even[2][2];
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          const v4f g = values(i, n), u = values(i, NH + n);
          float x[2][4];  // the output, or the gradients of gate and of up
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float slope;
            const float act = gate_act<decltype(ACT)::value>(g[e], slope);
            if constexpr (EPI == kEpiGated) {
              x[0][e] = act * u[e];
            } else {
              const uint2 d2 = dh[i & 1][n];
              const uint32_t pair = e < 2 ? d2.x : d2.y;
              const float d = u2f(e & 1 ? pair & 0xFFFF0000u : pair << 16);
              x[0][e] = d * u[e] * slope;
              x[1][e] = d * act;
            }
          }
#pragma unroll
          for (int h = 0; h < (EPI == kEpiGated ? 1 : 2); ++h) {
            uint32_t b[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) b[k] = f32_to_bf16(x[h][2 * k]) | (uint32_t)f32_to_bf16(x[h][2 * k + 1]) << 16;
            if constexpr (NH == 1) {
              const int col = col0 + 4 * q;
              if (row < w.row_hi && col < I) *reinterpret_cast<uint2*>(out + h * I + col) = uint2{b[0], b[1]};
            } else if (n & 1) {
              u4 o;
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const auto y = __builtin_amdgcn_permlane16_swap(even[h][k], b[k], false, false);
                o[k] = y[0];
                o[2 + k] = y[1];
              }
              const int col = col0 + 16 * (n - 1) + 16 * (q & 1) + 8 * (q >> 1);
              if (row < w.row_hi && col < I) *reinterpret_cast<u4*>(out + h * I + col) = o;
            } else {
              even[h][0] = b[0];
              even[h][1] = b[1];
            }
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if (gate.act == kActSilu) rows(Slice<kActSilu>{});
    else rows(Slice<kActGeluTanh>{});
    return odd;
  }
  if (w.part) {
#pragma unroll
    for (int i = 0; i < MTW; ++i)
#pragma unroll
      for (int n = 0; n < NTW; ++n) {
        const int f = (wm * MTW + i) * (S::BN / 16) + wn * NTW + n;
        *reinterpret_cast<v4f*>(w.part + (f * 64 + lane) * 4) = values(i, n);
        __builtin_amdgcn_sched_barrier(0);
      }
  } else if (p.N % 4 == 0 && p.ldc % 4 == 0 && p.ldc < (1 << 22) && ((uintptr_t)p.out & 7) == 0 && !p.out_f16 &&
             p.alpha == 1.0f) {
    // Buffer stores drop what lies past the last row (the buffer ends with it) or column (an
    // offset past the buffer), so the accumulators leave without a branch each.
    typedef unsigned int u2 __attribute__((ext_vector_type(2)));
    typedef unsigned int u4 __attribute__((ext_vector_type(4)));
    uint16_t* const base = p.out + (int64_t)w.row0 * p.ldc;
    const int rows = w.row_hi - w.row0 < S::BM ? w.row_hi - w.row0 : S::BM, ld = (int)p.ldc;
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)base, (short)0, ((rows - 1) * ld + (int)p.N) * 2, 0x00020000);
    const int r0 = wm * MTW * 16 + r, c0 = w.nb * S::BN + wn * NTW * 16 + 4 * q;
    // two bf16 of two fp32 (NaNs quiet)
    auto pack = [](float x, float y) -> uint32_t {
      uint32_t d = cvt_pk_bf16(x, y);
      d = x != x ? (d & 0xFFFF0000u) | 0x7FC0u : d;
      return y != y ? (d & 0x0000FFFFu) | 0x7FC00000u : d;
    };
    // BIAS: one is added to the rounded output (MXFP8 2048 x 18432 x 2560 135 us with a pass of its
    // own, 104 here, 222 through the LDS below), to MXFP4's sums ahead of the rounding.  WIDE (MXFP4, rows of
    // whole 16-byte pieces): of two n-tiles side by side every other 16 lanes change places, after which a lane holds
    // eight consecutive columns of one of them: half the stores, of 64 bytes of a row each (4096 x 17408 x 5120
    // 206 -> 198 us).
    auto store = [&](auto BIAS, auto WIDE) {
      constexpr bool wide = decltype(WIDE)::value;
      u2 bias[NTW];
      if constexpr (decltype(BIAS)::value) {
#pragma unroll
        for (int n = 0; n < NTW; ++n) {
          const uint16_t* const src = p.bias + (c0 + 16 * n < (int)p.N ? c0 + 16 * n : 0);
#pragma unroll
          for (int e = 0; e < 2; ++e) bias[n][e] = src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
        }
      }
      const int cw = c0 - 4 * q + 16 * (q & 1) + 8 * (q >> 1);  // the wide store's columns
#pragma unroll
      for (int i = 0; i < MTW; ++i) {
        u2 even;
#pragma unroll
        for (int n = 0; n < NTW; ++n) {
          const v4f v = values(i, n);
          u2 h;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float lo = v[2 * e], hi = v[2 * e + 1];
            if constexpr (decltype(BIAS)::value) {
              if constexpr (!FP4) {
                h[e] = pack(lo, hi);
                lo = u2f(h[e] << 16);
                hi = u2f(h[e] & 0xFFFF0000u);
              }
              lo = lo + u2f(bias[n][e] << 16);
              hi = hi + u2f(bias[n][e] & 0xFFFF0000u);
            }
            h[e] = pack(lo, hi);
          }
          if constexpr (!wide) {
            const uint32_t off = c0 + 16 * n < (int)p.N ? (uint32_t)((r0 + 16 * i) * ld + c0 + 16 * n) * 2 : 0xFFFFFFF0u;
            __builtin_amdgcn_raw_buffer_store_b64(h, rs, (int)off, 0, 0);
          } else if (n & 1) {
            u4 o;  // columns 0 .. 3 then 4 .. 7 of the lane's eight
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const auto x = __builtin_amdgcn_permlane16_swap(even[e], h[e], false, false);
              o[e] = x[0];
              o[2 + e] = x[1];
            }
            const int col = cw + 16 * (n - 1);
            const uint32_t off = col < (int)p.N ? (uint32_t)((r0 + 16 * i) * ld + col) * 2 : 0xFFFFFFE0u;
            __builtin_amdgcn_raw_buffer_store_b128(o, rs, (int)off, 0, 0);
          } else {
            even = h;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    if constexpr (FP4) {  // (elsewhere the second form's scalar registers spill)
      if (p.N % 8 == 0 && p.ldc % 8 == 0 && ((uintptr_t)p.out & 15) == 0) {
        if (p.bias) store(Slice<1>{}, Slice<1>{});
        else store(Slice<0>{}, Slice<1>{});
        return odd;
      }
    }
    if (p.bias) store(Slice<1>{}, Slice<0>{});
    else store(Slice<0>{}, Slice<0>{});
  } else {
    // other output formats and alignments: 16 rows at a time through the wave's own
    // part of the ring, once every wave is past its last read of it
    constexpr int TW = 16 * NTW;
    static_assert(4 * 16 * TW * 4 <= 2 * L::STAGE, "the staged rows fit the ring");
    float* const stage_out = reinterpret_cast<float*>(lds + L::RING) + wv * 16 * TW;
    tile_wait<0>();
#pragma unroll
    for (int i = 0; i < MTW; ++i) {
#pragma unroll
      for (int n = 0; n < NTW; ++n) *reinterpret_cast<v4f*>(stage_out + r * TW + 16 * n + 4 * q) = values(i, n);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll 1
      for (int c = lane; c < 16 * TW; c += 64) {
        const int64_t row = w.row0 + (wm * MTW + i) * 16 + c / TW, col = (int64_t)w.nb * S::BN + wn * TW + c % TW;
        const float v = stage_out[c];
        if (row < w.row_hi && col < p.N) p.out[row * p.ldc + col] = FP4 ? out_bits_fp4(v, p.bias, col) : out_bits(p, v, col);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  return odd;
}

// What a wave of an ADD tile left out: the terms with a value of B or v that is not finite, added to its outputs as they are
// stored (with such a term an output is an infinity or NaN, whatever its rounding).  It reads the kernel's arguments anew:
// kept in scalar registers over the tile they would spill.
template <int MTW, int NTW>
__device__ __forceinline__ void add_odd(int row0, int nb) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  auto at = (const __attribute__((address_space(4))) uint8_t*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(at));
  const auto& p = *(const __attribute__((address_space(4))) GemmParams*)at;
  const auto& add = *(const __attribute__((address_space(4))) RowAdapters*)(at + kAddOffset);
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rank = add.l.rank, groups = add.l.groups, parts = add.l.parts, width = parts * groups * 16;
  const int M = (int)p.M, N = (int)p.N;
  __threadfence();  // the wave's stores, before it loads them
#pragma unroll 1
  for (int c = lane; c < 16 * NTW; c += 64) {
    const int col = nb * (32 * NTW) + (wv & 1) * 16 * NTW + c;
    if (col >= N) continue;
    int part = 0;
    for (int k = 1; k < parts; ++k) part += col >= (int)add.l.cols[k] ? 1 : 0;
#pragma unroll 1
    for (int i = 0; i < 16 * MTW; ++i) {
      const int row = row0 + (wv >> 1) * 16 * MTW + i;
      if (row >= M) break;
      const int a = add.ids[row];
      if ((uint32_t)a >= (uint32_t)add.slots) continue;
      const uint16_t* const b = add.mat + a * add.slot_stride + (int64_t)col * add.ldm;
      const uint16_t* const v = add.v + (int64_t)row * (2 * width) + part * groups * 16;
      float sum = 0.0f;
      bool odd = false;
#pragma unroll 2
      for (int j = 0; j < rank; j += 8) {
        const u16x8 x = *reinterpret_cast<const u16x8*>(b + j), y = *reinterpret_cast<const u16x8*>(v + j),
                    z = *reinterpret_cast<const u16x8*>(v + width + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += adapter_odd_term(x[e], y[e], z[e], odd);
      }
      uint16_t& y = p.out[(int64_t)row * p.ldc + col];
      if (odd) y = f32_to_bf16(bf16_to_f32(y) + sum);
    }
  }
}

}  // namespace mxl
