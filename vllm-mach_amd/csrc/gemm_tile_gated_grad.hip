// The gradient epilogue's tiles, compiled apart for the build's time.
#define MXL_GATED_EPI kEpiGatedGrad
#define MXL_GATED_NAME launch_gated_grad_tiles
#include "gemm_tile_gated.hip"
