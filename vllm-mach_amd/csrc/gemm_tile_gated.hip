// Gated blocks of MX weights: act(x Wg^T) (x Wu^T) of a merged gate/up layer in one launch of the 2 x 2-wave tiles
// (gemm_tile.h), and the gradients of both products from that of the output, gate and up computed again.
//
// A tile's columns are half gate, half the up columns of the same, so both sums of an output meet in one lane's
// registers, and neither is written nor rounded.  What bounds the launch is the product (gemm_tile.h); the epilogue's
// exponentials run in the last round only.  The products' gradients are rounded to bf16 on their way to the input gradient,
// whose MFMA takes no more (against 64 bits dx is off by 0.0023, relative, with fp32 there by 0.0017).  4096 x 18432 x 2560
// MXFP8 172 us (2.25 PFLOP/s); 2048 x 18432 x 2560 MXFP4 67 us, with the gradient's epilogue 87 (14 more with 4-byte stores and
// dh loaded where it is used).  1 x 18432 x 2560 MXFP8 10.5 us, 4.6 TB/s of weights.
#include <algorithm>

#include "gemm_tile.h"

namespace mxl {

template <int FMT, int MT, int NT, int EPI>
__global__ __launch_bounds__(256, (WidePerCu<MT, NT, false, 2>::value)) void gated_tile_kernel(GemmParams p, WideGrid g,
                                                                                              TileGate gate) {
  constexpr int MTW = MT / 2, NTW = 2 * NT, BM = 16 * MT, TC = 32 * NT;  // (output columns of a tile)
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // TileLds::bytes(g.depth)
  const int M = (int)p.M, KT = (int)p.KT;
  auto a_row = [&](int row) { return row < M ? row : M - 1; };
  const uint8_t* const sw = static_cast<const uint8_t*>(p.sw);
  const uint32_t L = blockIdx.x, tail0 = (uint32_t)g.tail0;
  const uint32_t mblocks = (uint32_t)g.mblocks, nblocks = (uint32_t)g.nblocks, group_m = (uint32_t)g.group_m;
  uint32_t mb, nb;
  if constexpr (MT >= 8 && NT >= 2) {
    if (L >= tail0) {  // quarters of the last tiles
      const uint32_t unit = wide_logical(L - tail0, (uint32_t)gridDim.x - tail0);
      wide_coords(tail0 + (unit >> 2), mblocks, nblocks, group_m, mb, nb);
      const int row0 = (int)(mb * BM + (unit & 1) * (BM / 2)), qn = (int)(2 * nb + (unit >> 1 & 1));
      if (row0 >= M || (int64_t)qn * TC >= p.N) return;  // (N = 2 I)
      const TileWork w{row0, M, qn, 0, KT, p.w, sw, nullptr};
      tile_gemm<FMT, MTW / 2, NTW / 2, false, TileDepth<MT, NT>::QUARTER, EPI>(p, w, lds, a_row, gate);
      return;
    }
  }
  wide_coords(wide_logical(L, tail0), mblocks, nblocks, group_m, mb, nb);
  const TileWork w{(int)(mb * BM), M, (int)nb, 0, KT, p.w, sw, nullptr};
  using D = TileDepth<MT, NT>;
  if (D::LONE != D::SHARED && g.depth == D::LONE) tile_gemm<FMT, MTW, NTW, false, D::LONE, EPI>(p, w, lds, a_row, gate);
  else tile_gemm<FMT, MTW, NTW, false, D::SHARED, EPI>(p, w, lds, a_row, gate);
}

template <int FMT, int EPI>
static hipError_t launch_gated_fmt(const WideConfig& c, const GemmParams& p, const WideGrid& g0, const TileGate& gate,
                                   int64_t grid, hipStream_t s) {
  WideGrid g = g0;
#define MXL_GATED(MT_, NT_)                                                                                         \
  if (c.MT == MT_ && c.NT == NT_) {                                                                                 \
    using D = TileDepth<MT_, NT_>;                                                                                  \
    using L = TileLds<MT_ / 2, 2 * NT_, false>;                                                                     \
    g.depth = grid <= (int64_t)D::LONE_MAX * cu_count() ? D::LONE : D::SHARED;                                      \
    hipLaunchKernelGGL((gated_tile_kernel<FMT, MT_, NT_, EPI>), dim3((unsigned)grid), dim3(256),                    \
                       (unsigned)L::bytes(g.depth), s, p, g, gate);                                                 \
    return hipGetLastError();                                                                                       \
  }
  MXL_GATED(16, 4)
  MXL_GATED(8, 4)
  MXL_GATED(8, 2)
  MXL_GATED(8, 1)
  MXL_GATED(4, 2)
  MXL_GATED(4, 1)
#undef MXL_GATED
  return hipErrorInvalidValue;
}

#ifndef MXL_GATED_EPI
#define MXL_GATED_EPI kEpiGated
#define MXL_GATED_NAME launch_gated_tiles
#endif

hipError_t MXL_GATED_NAME(int fmt, const WideConfig& c, const GemmParams& p, const WideGrid& g, const TileGate& gate,
                          int64_t grid, hipStream_t s) {
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  if (fmt == kE4M3) return launch_gated_fmt<kE4M3, MXL_GATED_EPI>(c, p, g, gate, grid, s);
  if (fmt == kE2M3) return launch_gated_fmt<kE2M3, MXL_GATED_EPI>(c, p, g, gate, grid, s);
  if (fmt == kE3M2) return launch_gated_fmt<kE3M2, MXL_GATED_EPI>(c, p, g, gate, grid, s);
  if (fmt == kE2M1) return launch_gated_fmt<kE2M1, MXL_GATED_EPI>(c, p, g, gate, grid, s);
  return hipErrorInvalidValue;
}

}  // namespace mxl
