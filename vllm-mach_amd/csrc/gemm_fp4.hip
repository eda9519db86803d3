// Products of MXFP4 activations and weights on gfx950, dense and MoE-grouped: y = A W^T with E2M1
// codes and E8M0 scales per 32 on both sides, fp32 sums, bf16 out.
//
// The scaled MFMA multiplies 16 x 16 x 128 with a scale byte per lane and operand: lane 16 q + r supplies
// the 16 bytes of K [32 q, + 32) -- one scale block -- of row r of either operand.  The weights take its
// A operand and the activations its B operand, so a lane holds four consecutive output columns of one row.
#include "gemm_common.h"

namespace mxl {

// c += W A^T over a K128 slice: sw holds the slice's scale in byte J, sa in byte 0.
template <int J>
__device__ __forceinline__ v4f mfma_fp4(const uint4& w, const uint4& a, v4f c, uint32_t sw, uint32_t sa) {
  const v8i x = {(int)w.x, (int)w.y, (int)w.z, (int)w.w, 0, 0, 0, 0};
  const v8i y = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, kE2M1, kE2M1, J, (int)sw, 0, (int)sa);
}

// One wavefront: the 16 x 16 tile of output rows row0 .. (below row_hi) and n-tile nt, all of K.
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
    acc = mfma_fp4<0>(wv, av, acc, s, sa[4 * t]);
  }
  if (row0 + r >= row_hi) return;
  const int64_t col = nt * 16 + 4 * q;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < p.N) p.out[row * p.ldc + col + e] = out_bits(p, acc[e], col + e);
}

__global__ __launch_bounds__(256) void fp4_gemm_kernel(GemmParams p) {
  const int64_t nt = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (nt * 16 >= p.N) return;
  fp4_tile(p, p.w, static_cast<const uint8_t*>(p.sw), nt, (int64_t)blockIdx.y * 16, p.M, threadIdx.x & 63,
           [](int64_t row) { return row; });
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

static int check_operands(const char* who, const void* a, const void* sa, const void* w, const void* sw, int64_t N,
                          int64_t K, const void* out) {
  MXL_CHECK_ARG(N > 0 && K > 0 && K % 128 == 0, "%s: need N > 0, K > 0, K %% 128 == 0 (N=%lld K=%lld)", who,
                (long long)N, (long long)K);
  MXL_CHECK_ARG((((uintptr_t)a | (uintptr_t)w) & 15) == 0, "%s: a and w must be 16-byte aligned", who);
  MXL_CHECK_ARG((((uintptr_t)sa | (uintptr_t)sw) & 3) == 0, "%s: the scales must be 4-byte aligned", who);
  MXL_CHECK_ARG(((uintptr_t)out & 1) == 0, "%s: misaligned output", who);
  return MXL_OK;
}

// A stage of the 2 x 2-wave tiles is 128 bytes of a row, whatever its format, and takes two MFMAs of a K128
// slice of MXFP4 the time of one of 8-bit activations: the time model of K / 2 bytes holds.
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

static bool fp4_tiles_eligible(int64_t M, int64_t N, int64_t K) { return wide_tiles_eligible(M, N, K / 2, false); }

static GemmParams fp4_params(const void* a, const void* sa, const void* w, const void* sw, int64_t N, int64_t K,
                             void* out, int64_t ldc) {
  GemmParams p{};
  p.a = (const uint8_t*)a; p.sa = sa; p.w = (const uint8_t*)w; p.sw = sw; p.out = (uint16_t*)out;
  p.lda = K / 2; p.ldc = ldc; p.N = N; p.K = K; p.KT = (K + kTileK - 1) / kTileK;
  p.row_div = 1; p.S = 1;
  return p;
}

extern "C" int64_t mxl_mxfp4_gemm_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 16 || N <= 0 || K <= 0 || K % 128 || !fp4_tiles_eligible(M, N, K)) return 0;
  return wide_workspace_bytes(fp4_tiles_config(M, N, K), M, N);
}

extern "C" int mxl_mxfp4_gemm(const void* a, const void* sa, int64_t M, const void* w_tiled, const void* sw_tiled,
                              int64_t N, int64_t K, const void* bias, void* out, int64_t ldc, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_mxfp4_gemm";
  const int rc = check_operands(who, a, sa, w_tiled, sw_tiled, N, K, out);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(M >= 0 && ldc >= N, "%s: need M >= 0 and ldc >= N (M=%lld ldc=%lld)", who, (long long)M, (long long)ldc);
  if (M == 0) return MXL_OK;
  GemmParams p = fp4_params(a, sa, w_tiled, sw_tiled, N, K, out, ldc);
  p.M = p.a_rows = M;
  p.bias = (const uint16_t*)bias;
  if (M > 16 && fp4_tiles_eligible(M, N, K)) {
    const WideConfig c = fp4_tiles_config(M, N, K);
    const int64_t need = wide_workspace_bytes(c, M, N);
    MXL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                  "%s: needs a 16-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                  (long long)workspace_bytes);
    p.S = c.S;
    p.partial = (float*)workspace;
    const hipError_t e = launch_gemm_wide(kE2M1, false, c, p, 0, (hipStream_t)stream);
    if (e != hipSuccess) {
      set_error("%s: launch failed: %s", who, hipGetErrorString(e));
      return MXL_EHIP;
    }
    return MXL_OK;
  }
  fp4_gemm_kernel<<<dim3((unsigned)((N + 63) / 64), (unsigned)((M + 15) / 16)), 256, 0, (hipStream_t)stream>>>(p);
  MXL_CHECK_LAUNCH(who);
  return MXL_OK;
}

extern "C" int mxl_mxfp4_grouped_gemm(const void* a, const void* sa, int64_t a_rows, const int32_t* row_index,
                                      int row_div, const int64_t* expert_offsets, int64_t num_experts,
                                      int64_t routed_rows, const void* w_tiled, const void* sw_tiled, int64_t N,
                                      int64_t K, void* out, void* stream) {
  const char* who = "mxl_mxfp4_grouped_gemm";
  const int rc = check_operands(who, a, sa, w_tiled, sw_tiled, N, K, out);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(num_experts > 0 && num_experts <= 0xFFFF && row_div >= 1 && a_rows >= 0 && routed_rows >= 0,
                "%s: need 0 < experts <= 65535, row_div >= 1 and row counts >= 0", who);
  if (routed_rows == 0) return MXL_OK;
  GemmParams p = fp4_params(a, sa, w_tiled, sw_tiled, N, K, out, N);
  p.M = routed_rows; p.a_rows = a_rows; p.row_index = row_index; p.row_div = row_div; p.expert_offsets = expert_offsets;
  p.w_expert_stride = mxl_tiled_weight_bytes(N, K, kE2M1);
  p.sw_expert_stride = mxl_tiled_scale_bytes(N, K);
  if (routed_rows >= 16 * num_experts && num_experts <= kWideGroupedMaxExperts && a_rows > 0 &&
      fp4_tiles_eligible(a_rows, N, K)) {
    WideConfig c{2, 1, p.KT};
    c.MT = routed_rows >= 48 * num_experts ? 8 : 4;
    const hipError_t e = launch_gemm_wide(kE2M1, false, c, p, num_experts, (hipStream_t)stream);
    if (e != hipSuccess) {
      set_error("%s: launch failed: %s", who, hipGetErrorString(e));
      return MXL_EHIP;
    }
    return MXL_OK;
  }
  fp4_grouped_kernel<<<dim3((unsigned)((N + 63) / 64), (unsigned)num_experts), 256, 0, (hipStream_t)stream>>>(p);
  MXL_CHECK_LAUNCH(who);
  return MXL_OK;
}
