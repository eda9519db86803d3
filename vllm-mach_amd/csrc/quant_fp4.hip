// MXFP4 producers for gfx950: the activation (and weight) quantizer and SwiGLU -> MXFP4.
//
// Both are passes over memory: the quantizer moves 2 + 17/32 bytes a value, the producer 4 + 17/32 (4096 x 5120 12.5 us,
// 4.2 TB/s).
// Four lanes own a 32-element block, each with the 16 bytes of one load per input and a 4-byte store of
// its eight codes, so that every access of a wavefront is one contiguous span; the amax is an
// xor-shuffle maximum over the four lanes.
#include <algorithm>

#include "fp4.h"

namespace mxl {

__global__ __launch_bounds__(256) void quant_mxfp4_kernel(const uint16_t* __restrict__ x, int64_t ldx,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          uint32_t blocks_per_row, uint32_t blocks, uint32_t carry) {
  // (32-bit lane indices: the host bounds the block count; lanes past the end shadow the last block)
  const uint32_t t = blockIdx.x * blockDim.x + threadIdx.x, sub = t & 3;
  const bool live = t / 4 < blocks;
  const uint32_t id = live ? t / 4 : blocks - 1, row = id / blocks_per_row, blk = id - row * blocks_per_row;
  const uint4 v = *reinterpret_cast<const uint4*>(x + (int64_t)row * ldx + blk * 32 + sub * 8);
  const uint32_t d[4] = {v.x, v.y, v.z, v.w};
  uint32_t c;
  const uint32_t s = quant_e2m1_x4(d, carry, c);
  if (!live) return;
  reinterpret_cast<uint32_t*>(codes)[(int64_t)id * 4 + sub] = c;
  if (sub == 0) scales[id] = (uint8_t)s;
}

// v = bf16(bf16(silu(g)) u) of the MXFP8 producer (rules 0 and 1 there), then the quantization.  TABLE: the workgroup
// first stages the 16 KiB table of bf16(silu(g)) in LDS, and a wavefront whose gates all lie in it reads the
// activations there: exp and the division are three quarters of the instructions that bound the pass without it.
// 512 rows of 9216: 7.4 us, 9.5 without; 16384 of 512: 9.2, 12.5.  Few items do not pay the staging.  The 7.4 are 21.6 MB
// (4.1 at a large copy's rate) behind a launch and, in every workgroup, the table: 69 % of the waves' time is waits.
constexpr int64_t kFp4TableItemsPerCu = 512;
int cu_count();  // compute units of the current device (gemm_stream.hip)
template <bool TABLE>
__global__ __launch_bounds__(TABLE ? 512 : 256) void swiglu_mxfp4_kernel(const uint16_t* __restrict__ gate_up,
                                                                         uint8_t* __restrict__ codes,
                                                                         uint8_t* __restrict__ scales,
                                                                         uint32_t blocks_per_row, uint32_t blocks,
                                                                         uint32_t carry) {
  __shared__ __attribute__((aligned(16))) uint16_t tab[TABLE ? kSiluEntries : 8];
  if (TABLE) {
    for (uint32_t i = threadIdx.x; i < kSiluEntries / 8; i += blockDim.x)
      reinterpret_cast<uint4*>(tab)[i] = reinterpret_cast<const uint4*>(kSiluAct)[i];
    __syncthreads();
  }
  // (whole blocks: lanes past the end shadow the last one)
  for (uint32_t base = blockIdx.x * (blockDim.x / 4); base < blocks; base += gridDim.x * (blockDim.x / 4)) {
    const uint32_t own = base + threadIdx.x / 4, sub = threadIdx.x & 3;
    const bool live = own < blocks;
    const uint32_t id = live ? own : blocks - 1, row = id / blocks_per_row, blk = id - row * blocks_per_row;
    const int64_t K = (int64_t)blocks_per_row * 32, at = row * 2 * K + blk * 32 + sub * 8;
    const uint4 graw = *reinterpret_cast<const uint4*>(gate_up + at);
    const uint4 uraw = *reinterpret_cast<const uint4*>(gate_up + at + K);
    uint32_t d[4];
    if (TABLE && __builtin_amdgcn_ballot_w64(!silu_in_table(graw)) == 0) {
      const uint32_t gd[4] = {graw.x, graw.y, graw.z, graw.w}, ud[4] = {uraw.x, uraw.y, uraw.z, uraw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t o = silu_offsets(gd[i]) + ((gd[i] >> 3) & 0x10001000u);
        const float a0 = u2f((uint32_t)tab[o & 0xFFFFu] << 16), a1 = u2f((uint32_t)tab[o >> 16] << 16);
        d[i] = cvt_pk_bf16(a0 * u2f(ud[i] << 16), a1 * u2f(ud[i] & 0xFFFF0000u));
      }
    } else {
      float g[8], u[8], v[8];
      bf16x8_to_f32(graw, g);
      bf16x8_to_f32(uraw, u);
      swiglu8<kFloorCarry175>(g, u, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = cvt_pk_bf16(v[2 * i], v[2 * i + 1]);  // (bf16 values already)
    }
    uint32_t c;
    const uint32_t s = quant_e2m1_x4(d, carry, c);
    if (!live) continue;
    reinterpret_cast<uint32_t*>(codes)[(int64_t)id * 4 + sub] = c;
    if (sub == 0) scales[id] = (uint8_t)s;
  }
}

}  // namespace mxl

using namespace mxl;

static int check_quant(const char* who, const void* in, int64_t M, int64_t K, int rule, const void* codes) {
  MXL_CHECK_ARG(M >= 0 && K > 0 && K % 32 == 0, "%s: need M >= 0, K > 0, K %% 32 == 0 (M=%lld K=%lld)", who,
                (long long)M, (long long)K);
  MXL_CHECK_ARG(fp4_rule(rule), "%s: unknown rule %d", who, rule);
  MXL_CHECK_ARG(((uintptr_t)in & 15) == 0 && ((uintptr_t)codes & 3) == 0,
                "%s: the input must be 16-byte aligned, the codes 4-byte aligned", who);
  // lanes are indexed in 32 bits
  MXL_CHECK_ARG(K <= 0x7FFFFFFF && M <= (int64_t)0x7FFFFF00 / 4 / (K / 32), "%s: too large (M=%lld, K=%lld)", who,
                (long long)M, (long long)K);
  return MXL_OK;
}

extern "C" int mxl_quantize_mxfp4(const void* x, int64_t M, int64_t K, int64_t ldx, int rule, void* codes,
                                  void* scales, void* stream) {
  const int rc = check_quant("mxl_quantize_mxfp4", x, M, K, rule, codes);
  if (rc != MXL_OK) return rc;
  MXL_CHECK_ARG(ldx >= K && ldx % 8 == 0, "mxl_quantize_mxfp4: ldx must be >= K and a multiple of 8");
  if (M == 0) return MXL_OK;
  const int64_t blocks = M * (K / 32);
  const dim3 grid((unsigned)((blocks * 4 + 255) / 256));
  hipStream_t s = (hipStream_t)stream;
  const uint32_t per = (uint32_t)(K / 32), n = (uint32_t)blocks;
  quant_mxfp4_kernel<<<grid, 256, 0, s>>>((const uint16_t*)x, ldx, (uint8_t*)codes, (uint8_t*)scales, per, n,
                                          fp4_carry(rule));
  MXL_CHECK_LAUNCH("mxl_quantize_mxfp4");
  return MXL_OK;
}

extern "C" int mxl_swiglu_mxfp4(const void* gate_up, int64_t M, int64_t K, int rule, void* codes, void* scales,
                                void* stream) {
  const int rc = check_quant("mxl_swiglu_mxfp4", gate_up, M, K, rule, codes);
  if (rc != MXL_OK) return rc;
  if (M == 0) return MXL_OK;
  const int64_t blocks = M * (K / 32);
  hipStream_t s = (hipStream_t)stream;
  const uint32_t per = (uint32_t)(K / 32), n = (uint32_t)blocks, carry = fp4_carry(rule);
  const uint16_t* in = (const uint16_t*)gate_up;
  uint8_t *c = (uint8_t*)codes, *sc = (uint8_t*)scales;
  if (blocks * 4 >= kFp4TableItemsPerCu * cu_count()) {  // four workgroups a CU at most
    const dim3 grid((unsigned)std::min<int64_t>((blocks + 127) / 128, 4 * (int64_t)cu_count()));
    swiglu_mxfp4_kernel<true><<<grid, 512, 0, s>>>(in, c, sc, per, n, carry);
  } else {
    swiglu_mxfp4_kernel<false><<<dim3((unsigned)((blocks + 63) / 64)), 256, 0, s>>>(in, c, sc, per, n, carry);
  }
  MXL_CHECK_LAUNCH("mxl_swiglu_mxfp4");
  return MXL_OK;
}
