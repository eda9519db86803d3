// C ABI of the gated blocks: the activations' quantization and the tiles of gemm_tile_gated.hip.
#include <algorithm>

#include "fp4.h"
#include "gate_act.h"
#include "gemm_tile.h"

namespace mxl {
hipError_t launch_gated_tiles(int fmt, const WideConfig& c, const GemmParams& p, const WideGrid& g, const TileGate& gate,
                              int64_t grid, hipStream_t s);
hipError_t launch_gated_grad_tiles(int fmt, const WideConfig& c, const GemmParams& p, const WideGrid& g,
                                   const TileGate& gate, int64_t grid, hipStream_t s);
}  // namespace mxl

using namespace mxl;

extern "C" int mxl_quantize_mxfp8(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes, void* scales,
                                  void* stream);
extern "C" int mxl_quantize_mxfp4(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes, void* scales,
                                  void* stream);

namespace {

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }
int64_t row_bytes(int64_t K, int fmt) { return fmt == kE2M1 ? K / 2 : K; }

// Rows of one launch: 32-bit operand offsets, whole 256-row blocks.
int64_t slab_rows(int64_t M, int64_t K, int fmt) {
  const int64_t most = ((int64_t(1) << 32) / row_bytes(K, fmt) - 1) / 256 * 256;
  return std::min(M, most);
}

int64_t workspace_bytes(int64_t M, int64_t K, int fmt) { return round256(M * row_bytes(K, fmt)) + round256(M * (K / 32)); }

int run(const char* who, const void* x, int64_t M, int64_t K, int64_t ldx, int rule, const void* w, const void* sw,
        int64_t I, int fmt, int act, const void* dh, int64_t lddh, void* out, int64_t ldo, void* workspace,
        int64_t bytes, void* stream) {
  const int64_t wide = dh ? 2 * I : I;
  MXL_CHECK_ARG(fmt == kE4M3 || fmt == kE2M3 || fmt == kE3M2 || fmt == kE2M1, "%s: unknown format %d", who, fmt);
  MXL_CHECK_ARG(act == kActSilu || act == kActGeluTanh, "%s: unknown activation %d", who, act);
  MXL_CHECK_ARG(fmt != kE2M1 || fp4_rule(rule), "%s: unknown rule %d", who, rule);
  MXL_CHECK_ARG(M >= 0 && M <= 0x7FFFFFFF - 256 && I > 0 && I % 16 == 0 && K > 0 && K % 128 == 0 && K <= (1 << 22),
                "%s: need I > 0, I %% 16 == 0, 0 < K <= 2^22, K %% 128 == 0 (M=%lld I=%lld K=%lld)", who, (long long)M,
                (long long)I, (long long)K);
  MXL_CHECK_ARG(2 * I / 16 * ((K + kTileK - 1) / kTileK) < (1 << 24), "%s: too large (I=%lld K=%lld)", who, (long long)I,
                (long long)K);
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0 && ldo >= wide && ldo % 8 == 0 && (!dh || (lddh >= I && lddh % 4 == 0)),
                "%s: bad row stride (ldx=%lld ldo=%lld lddh=%lld)", who, (long long)ldx, (long long)ldo, (long long)lddh);
  MXL_CHECK_ARG((((uintptr_t)x | (uintptr_t)w) & 15) == 0 && ((uintptr_t)sw & 3) == 0 &&
                    ((uintptr_t)out & 15) == 0 && ((uintptr_t)dh & 7) == 0, "%s: misaligned operands", who);
  if (M == 0) return MXL_OK;
  MXL_CHECK_ARG(workspace && bytes >= workspace_bytes(M, K, fmt) && ((uintptr_t)workspace & 255) == 0,
                "%s: needs a 256-byte aligned workspace of %lld bytes (have %lld)", who,
                (long long)workspace_bytes(M, K, fmt), (long long)bytes);
  uint8_t* const codes = (uint8_t*)workspace;
  uint8_t* const scales = codes + round256(M * row_bytes(K, fmt));
  const int st = fmt == kE2M1 ? mxl_quantize_mxfp4(x, M, K, ldx, rule, codes, scales, stream)
                              : mxl_quantize_mxfp8(x, M, K, ldx, rule, codes, scales, stream);
  if (st != MXL_OK) return st;
  const int64_t slab = slab_rows(M, K, fmt);
  for (int64_t row = 0; row < M; row += slab) {
    GemmParams p{};
    p.M = p.a_rows = std::min(slab, M - row);
    p.N = 2 * I; p.K = K; p.KT = (K + kTileK - 1) / kTileK;
    p.a = codes + row * row_bytes(K, fmt); p.sa = scales + row * (K / 32); p.lda = row_bytes(K, fmt);
    p.w = (const uint8_t*)w; p.sw = sw; p.out = (uint16_t*)out + row * ldo; p.ldc = ldo;
    p.row_div = 1; p.S = 1;
    TileGate gate;
    gate.act = act;
    gate.dh = dh ? (const uint16_t*)dh + row * lddh : nullptr;
    gate.lddh = lddh;
    WideGrid g{};
    int64_t grid;
    const WideConfig c = wide_tiles_whole(p.M, p.N, K, fmt, false, g, grid);
    const hipError_t e = (dh ? launch_gated_grad_tiles : launch_gated_tiles)(fmt, c, p, g, gate, grid, (hipStream_t)stream);
    if (e != hipSuccess) {
      set_error("%s: launch failed: %s", who, hipGetErrorString(e));
      return MXL_EHIP;
    }
  }
  return MXL_OK;
}

}  // namespace

extern "C" int64_t mxl_gated_workspace_bytes(int64_t M, int64_t K, int fmt) {
  return M <= 0 || M > 0x7FFFFFFF || K <= 0 || K > (1 << 22) ? 0 : workspace_bytes(M, K, fmt);
}

extern "C" int mxl_gated_plan_name(int64_t M, int64_t I, int64_t K, int fmt, int grad, char* buf, int64_t len) {
  MXL_CHECK_ARG(M > 0 && M <= 0x7FFFFFFF && I > 0 && I <= (1 << 22) && I % 16 == 0 && K > 0 && K <= (1 << 22) && K % 128 == 0 && buf,
                "mxl_gated_plan_name: bad shape");
  WideGrid g{};
  int64_t grid;
  const WideConfig c = wide_tiles_whole(slab_rows(M, K, fmt), 2 * I, K, fmt, false, g, grid);
  return tile_plan_name("gated_tile_kernel", grad ? "3" : "2", c, g, grid, fmt, buf, len);
}

extern "C" int mxl_gated_linear(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, const void* w_tiled,
                                const void* sw_tiled, int64_t I, int fmt, int act, void* out, int64_t ldo,
                                void* workspace, int64_t workspace_bytes, void* stream) {
  return run("mxl_gated_linear", x, M, K, ldx, rule, w_tiled, sw_tiled, I, fmt, act, nullptr, 0, out, ldo, workspace,
             workspace_bytes, stream);
}

extern "C" int mxl_gated_grad(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, const void* w_tiled,
                              const void* sw_tiled, int64_t I, int fmt, int act, const void* dh, int64_t lddh, void* out,
                              int64_t ldo, void* workspace, int64_t workspace_bytes, void* stream) {
  MXL_CHECK_ARG(dh || M == 0, "mxl_gated_grad: needs dh");
  if (M == 0) return MXL_OK;
  return run("mxl_gated_grad", x, M, K, ldx, rule, w_tiled, sw_tiled, I, fmt, act, dh, lddh, out, ldo, workspace,
             workspace_bytes, stream);
}
