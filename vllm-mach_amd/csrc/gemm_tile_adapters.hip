// Linear layers with the low-rank adapters of their rows added in the product's launch: the 2 x 2-wave tiles
// (gemm_tile.h, ADD), the activations' quantization, and the adapters' first half (adapters.hip) ahead of them.
//
// Bound: the product, and some 4 us a tile and adapter in waits for v's and B's first bytes.  2048 x 18432 x 2560 MXFP8, rank
// 16: 108 us at its best, the product alone 95; 4096 x 17408 x 5120, 8 adapters of rank 64: 351 at its best, alone 300.
#include <algorithm>

#include "gemm_tile.h"

namespace mxl {

// Whole tiles and, past them, quarters (the gated kernels' grid; a K split's workgroups beside the adapters' operands
// would run out of scalar registers).  So few tiles of a long K, where the layer's own product splits K, are slower here than
// apart (figures at rows_add, adapters.h).
template <int FMT, int MT, int NT, bool BLOCK>
__global__ __launch_bounds__(256, (WidePerCu<MT, NT, false, 2>::value)) void adapter_tile_kernel(GemmParams p, WideGrid g,
                                                                                                RowAdapters add) {
  static_assert(alignof(GemmParams) == 8 && alignof(WideGrid) == 8 && alignof(RowAdapters) == 8, "the arguments' offsets");
  constexpr int MTW = MT / 2, NTW = 2 * NT, BM = 16 * MT, TW = 64 * NT;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // TileLds::bytes(g.depth)
  const int M = (int)p.M, KT = (int)p.KT;
  auto a_row = [&](int row) { return row < M ? row : M - 1; };
  const uint8_t* const sw = static_cast<const uint8_t*>(p.sw);
  const uint32_t L = blockIdx.x, tail0 = (uint32_t)g.tail0;
  const uint32_t mblocks = (uint32_t)g.mblocks, nblocks = (uint32_t)g.nblocks, group_m = (uint32_t)g.group_m;
  uint32_t mb, nb;
  if constexpr (MT >= 8 && NT >= 2) {
    if (L >= tail0) {
      const uint32_t unit = wide_logical(L - tail0, (uint32_t)gridDim.x - tail0);
      wide_coords(tail0 + (unit >> 2), mblocks, nblocks, group_m, mb, nb);
      const int row0 = (int)(mb * BM + (unit & 1) * (BM / 2)), qn = (int)(2 * nb + (unit >> 1 & 1));
      if (row0 >= M || (int64_t)qn * (TW / 2) >= p.N) return;
      const TileWork w{row0, M, qn, 0, KT, p.w, sw, nullptr};
      if (tile_gemm<FMT, MTW / 2, NTW / 2, BLOCK, TileDepth<MT, NT>::QUARTER, kEpiStore, true>(p, w, lds, a_row))
        add_odd<MTW / 2, NTW / 2>(row0, qn);
      return;
    }
  }
  wide_coords(wide_logical(L, tail0), mblocks, nblocks, group_m, mb, nb);
  const TileWork w{(int)(mb * BM), M, (int)nb, 0, KT, p.w, sw, nullptr};
  using D = TileDepth<MT, NT>;
  const bool odd = D::LONE != D::SHARED && g.depth == D::LONE
                       ? tile_gemm<FMT, MTW, NTW, BLOCK, D::LONE, kEpiStore, true>(p, w, lds, a_row)
                       : tile_gemm<FMT, MTW, NTW, BLOCK, D::SHARED, kEpiStore, true>(p, w, lds, a_row);
  if (odd) add_odd<MTW, NTW>(w.row0, w.nb);
}

template <int FMT, bool BLOCK>
static hipError_t launch_adapter_fmt(const WideConfig& c, const GemmParams& p, const WideGrid& g0, const RowAdapters& add,
                                     int64_t grid, hipStream_t s) {
  WideGrid g = g0;
#define MXL_ADAPTER_TILES(MT_, NT_)                                                                            \
  if (c.MT == MT_ && c.NT == NT_) {                                                                            \
    using D = TileDepth<MT_, NT_>;                                                                             \
    using L = TileLds<MT_ / 2, 2 * NT_, BLOCK>;                                                                \
    static_assert(L::bytes(D::LONE) + 1024 <= 160 * 1024 && L::bytes(D::SHARED) + 1024 <= 160 * 1024, "LDS"); \
    g.depth = grid <= (int64_t)D::LONE_MAX * cu_count() ? D::LONE : D::SHARED;                                 \
    hipLaunchKernelGGL((adapter_tile_kernel<FMT, MT_, NT_, BLOCK>), dim3((unsigned)grid), dim3(256),           \
                       (unsigned)L::bytes(g.depth) + 1024, s, p, g, add); /* (the rows' ids) */                \
    return hipGetLastError();                                                                                  \
  }
  if constexpr (!BLOCK) {
    MXL_ADAPTER_TILES(16, 4)
    MXL_ADAPTER_TILES(8, 4)
  }
  MXL_ADAPTER_TILES(8, 2)
  MXL_ADAPTER_TILES(8, 1)
  MXL_ADAPTER_TILES(4, 2)
  MXL_ADAPTER_TILES(4, 1)
#undef MXL_ADAPTER_TILES
  return hipErrorInvalidValue;
}

hipError_t launch_adapter_tiles(int fmt, bool block, const WideConfig& c, const GemmParams& p, const WideGrid& g,
                                const RowAdapters& add, int64_t grid, hipStream_t s) {
  if (grid > 0x7FFFFFFF || c.WM != 2) return hipErrorInvalidValue;
  if (block) return fmt == kE4M3 ? launch_adapter_fmt<kE4M3, true>(c, p, g, add, grid, s) : hipErrorInvalidValue;
  if (fmt == kE4M3) return launch_adapter_fmt<kE4M3, false>(c, p, g, add, grid, s);
  if (fmt == kE2M3) return launch_adapter_fmt<kE2M3, false>(c, p, g, add, grid, s);
  if (fmt == kE3M2) return launch_adapter_fmt<kE3M2, false>(c, p, g, add, grid, s);
  if (fmt == kE2M1) return launch_adapter_fmt<kE2M1, false>(c, p, g, add, grid, s);
  return hipErrorInvalidValue;
}

}  // namespace mxl

using namespace mxl;

extern "C" int mxl_adapter_linear_supported(int64_t M, int64_t N, int64_t K, int fmt, int block, int64_t slots,
                                            int64_t parts, int64_t rank);

extern "C" int mxl_adapter_linear_plan_name(int64_t M, int64_t N, int64_t K, int fmt, int block, char* buf, int64_t len) {
  MXL_CHECK_ARG(buf && mxl_adapter_linear_supported(M, N, K, fmt, block, 1, 1, 8), "mxl_adapter_linear_plan_name: bad shape");
  WideGrid g{};
  int64_t grid;
  const WideConfig c = wide_tiles_whole(M, N, K, fmt, block != 0, g, grid);
  return tile_plan_name("adapter_tile_kernel", block ? "true" : "false", c, g, grid, fmt, buf, len);
}
