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
#include <algorithm>

#include "gemm_wide.h"

namespace mxl {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x32_t __attribute__((ext_vector_type(32)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned int v6u_t __attribute__((ext_vector_type(6)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4;

constexpr int kGradStage = 64;  // rows of W

struct GradParams {
  const uint16_t* dy;
  const uint8_t* w;
  const void* sw;  // tiled E8M0, or fp32 [ceil(N / 128), K / 128]
  uint16_t* out;
  float* partial;  // [S, M, K] when split
  int64_t M, N, K, KT, lddy, ldo;
  int S;
  int64_t per;     // stages of a split, an even number
  uint32_t mblocks, kblocks, group_m;
};

template <int FMT, int TK>
struct GradW {
  static constexpr int SL = TK / 128;  // 128-column slices of a wave's strip
  static constexpr int NC = FMT == kE4M3 ? 2 * SL : FMT == kE2M1 ? SL : SL == 2 ? 3 : 2;  // 16-byte pieces a lane
  uint4 c[NC];
  uint32_t s[2];
};

template <int FMT, int TM, int TK, bool BLOCK>
__global__ __launch_bounds__(256) void input_grad_kernel(GradParams p) {
  constexpr int MI = TM / 64, KI = TK / 64, SL = TK / 128;  // 32 x 32 tiles of a wave; slices
  constexpr int RS = TK + 32;                              // elements of a row of W in LDS
  constexpr int A_BYTES = TM * 128, W_BYTES = kGradStage * RS * 2;
  constexpr int NA = TM / 32;                              // 16-byte pieces of dy a thread
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];  // [2] dy, [2] W
  const int t = threadIdx.x, lane = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wv >> 1, wk = wv & 1, r = lane & 15, q = lane >> 4;

  const uint32_t unit = wide_logical(blockIdx.x, gridDim.x), tiles = p.mblocks * p.kblocks;
  const uint32_t split = unit / tiles;
  uint32_t mb, kb;
  wide_coords(unit - split * tiles, p.mblocks, p.kblocks, p.group_m, mb, kb);
  const int64_t row0 = (int64_t)mb * TM;
  const int stages = (int)((p.N + kGradStage - 1) / kGradStage);
  const int s0 = (int)(split * p.per), s1 = s0 + (int)p.per < stages ? s0 + (int)p.per : stages;
  const int ntiles = (int)((p.N + 15) / 16), j0 = (int)(kb * SL) & 3;  // the first slice's place in its super-tile
  const int64_t kt = (int64_t)kb * SL >> 2;

  // dy: piece u of a thread is row t / 8 + 32 u, columns 8 (t % 8) of the stage
  const uint16_t* const a_base = p.dy + row0 * p.lddy;
  uint32_t a_off[NA];
#pragma unroll
  for (int u = 0; u < NA; ++u) {
    const int64_t row = row0 + (t >> 3) + 32 * u < p.M ? (t >> 3) + 32 * u : p.M - 1 - row0;
    a_off[u] = (uint32_t)(row * p.lddy) + 8 * (t & 7);
  }
  uint4 av[NA];
  GradW<FMT, TK> wr;
  auto load = [&](int s) {
    const int64_t n0 = (int64_t)s * kGradStage;
    const bool in = n0 + 8 * (t & 7) < p.N;  // (N comes in eights)
#pragma unroll
    for (int u = 0; u < NA; ++u) {
      av[u] = *reinterpret_cast<const uint4*>(a_base + (in ? n0 : -8 * (t & 7)) + a_off[u]);
      if (!in) av[u] = uint4{0, 0, 0, 0};
    }
    const int nt = s * 4 + wv < ntiles ? s * 4 + wv : ntiles - 1;  // (of strips past the last, zeros below)
    const int64_t tile = (int64_t)nt * p.KT + kt;
    const uint8_t* const w = p.w + tile * (FmtTraits<FMT>::CH * 1024) + lane * 16;
    const int c0 = FMT == kE4M3 ? 2 * j0 : FMT == kE2M1 ? j0 : (3 * j0) >> 1;
#pragma unroll
    for (int c = 0; c < GradW<FMT, TK>::NC; ++c) wr.c[c] = *reinterpret_cast<const uint4*>(w + (c0 + c) * 1024);
    if constexpr (!BLOCK) {
      const uint8_t* const sw = static_cast<const uint8_t*>(p.sw) + tile * 256;
      if constexpr (FMT == kE4M3) {  // pieces of 16 columns: half a block each, of lane groups q / 2 and 2 + q / 2
        wr.s[0] = *reinterpret_cast<const uint32_t*>(sw + (16 * (q >> 1) + r) * 4) >> (8 * j0);
        wr.s[1] = *reinterpret_cast<const uint32_t*>(sw + (16 * (2 + (q >> 1)) + r) * 4) >> (8 * j0);
      } else {
        wr.s[0] = *reinterpret_cast<const uint32_t*>(sw + lane * 4) >> (8 * j0);
      }
    }
    if (s * 4 + wv >= ntiles) {
#pragma unroll
      for (int c = 0; c < GradW<FMT, TK>::NC; ++c) wr.c[c] = uint4{0, 0, 0, 0};
      wr.s[0] = wr.s[1] = 0x7F7F7F7Fu;
    }
  };
  // dy: piece p of row x sits at 16 (p ^ x % 8) of its 128 bytes
  const uint32_t a_to = (t >> 3) * 128 + 16 * ((t & 7) ^ ((t >> 3) & 7));
  auto store = [&](int buf) {
    uint8_t* const a = lds + buf * A_BYTES;
#pragma unroll
    for (int u = 0; u < NA; ++u) *reinterpret_cast<uint4*>(a + a_to + u * 4096) = av[u];
    uint8_t* const w = lds + 2 * A_BYTES + buf * W_BYTES + (16 * wv + r) * (RS * 2);
    auto scale = [&](int i, int sl) { return u2f(BLOCK ? 127u << 23 : ((wr.s[i] >> (8 * sl)) & 0xFFu) << 23); };
#pragma unroll
    for (int sl = 0; sl < SL; ++sl) {
      if constexpr (FMT == kE4M3) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {  // columns 64 h + 16 q of the slice
          const uint4 c = wr.c[2 * sl + h];
          const uint32_t d[4] = {c.x, c.y, c.z, c.w};
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[i], scale(h, sl), false));
            o[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(d[i], scale(h, sl), true));
          }
          uint4* const to = reinterpret_cast<uint4*>(w + (128 * sl + 64 * h + 16 * q) * 2);
          to[0] = uint4{o[0], o[1], o[2], o[3]};
          to[1] = uint4{o[4], o[5], o[6], o[7]};
        }
      } else {  // columns 32 q of the slice
        uint4* const to = reinterpret_cast<uint4*>(w + (128 * sl + 32 * q) * 2);
        if constexpr (FMT == kE2M1) {
          const uint32_t d[4] = {wr.c[sl].x, wr.c[sl].y, wr.c[sl].z, wr.c[sl].w};
          const float f = scale(0, sl);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            to[i] = uint4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 0)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 1)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 2)),
                          __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d[i], f, 3))};
        } else {
          v6u_t d;  // six dwords, of an odd first slice from the first piece's middle
          const uint4 x = wr.c[sl], y = wr.c[sl + 1];
          const bool odd = SL == 2 ? sl == 1 : (j0 & 1) != 0;
          d[0] = odd ? x.z : x.x; d[1] = odd ? x.w : x.y; d[2] = odd ? y.x : x.z;
          d[3] = odd ? y.y : x.w; d[4] = odd ? y.z : y.x; d[5] = odd ? y.w : y.y;
          bf16x32_t v;
          if constexpr (FMT == kE2M3) v = __builtin_amdgcn_cvt_scalef32_pk32_bf16_fp6(d, scale(0, sl));
          else v = __builtin_amdgcn_cvt_scalef32_pk32_bf16_bf6(d, scale(0, sl));
          struct Q { uint4 x[4]; };
          const Q o = __builtin_bit_cast(Q, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i] = o.x[i];
        }
      }
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
  // fragments: dy row lane % 32 and columns 16 kk + 8 (lane / 32); W column lane % 32 and those rows
  const int ah = lane >> 5, ax = lane & 7;
  const uint32_t a_from = (wm * (TM / 2) + (lane & 31)) * 128;
  const uint32_t w_from = (8 * (q >> 1) + (r >> 2)) * (RS * 2) + (wk * (TK / 2) + 16 * (q & 1) + 4 * (r & 3)) * 2;
  auto compute = [&](int buf) {
    const uint8_t* const a = lds + buf * A_BYTES + a_from;
    const uint8_t* const w = lds + 2 * A_BYTES + buf * W_BYTES + w_from;
#pragma unroll
    for (int kk = 0; kk < kGradStage / 16; ++kk) {
      uint4 af[MI], wf[KI];
#pragma unroll
      for (int m = 0; m < MI; ++m) af[m] = *reinterpret_cast<const uint4*>(a + m * 4096 + 16 * ((2 * kk + ah) ^ ax));
#pragma unroll
      for (int c = 0; c < KI; ++c) {
        const s16x4_t x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(w + 16 * kk * (RS * 2) + c * 64));
        const s16x4_t x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(w + (16 * kk + 4) * (RS * 2) + c * 64));
        const uint2 y0 = __builtin_bit_cast(uint2, x0), y1 = __builtin_bit_cast(uint2, x1);
        wf[c] = uint4{y0.x, y0.y, y1.x, y1.y};
      }
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int c = 0; c < KI; ++c) {
          v16f& to = BLOCK ? raw[BLOCK ? m : 0][BLOCK ? c : 0] : acc[m][c];
          to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, wf[c]),
                                                       __builtin_bit_cast(bf16x8_t, af[m]), to, 0, 0, 0);
        }
    }
  };

  if (s0 < s1) {
    load(s0);
    store(0);
    if (s0 + 1 < s1) load(s0 + 1);
    __syncthreads();
    for (int s = s0; s < s1; ++s) {
      const int buf = (s - s0) & 1;
      if (s + 1 < s1) store(buf ^ 1);
      if (s + 2 < s1) load(s + 2);
      compute(buf);
      if constexpr (BLOCK) {
        if ((s & 1) || s + 1 == s1) {  // a block of 128 rows ends
          const float f = static_cast<const float*>(p.sw)[(int64_t)(s >> 1) * (p.K / 128) +
                                                          std::min<int64_t>(kb * SL + (SL == 2 ? wk : 0), p.K / 128 - 1)];
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
      }
      __syncthreads();
    }
  }

  // lane: row lane % 32, columns 8 g + 4 (lane / 32) .. + 3 of a 32 x 32 tile in registers 4 g ..
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int64_t row = row0 + wm * (TM / 2) + 32 * m + (lane & 31);
    if (row >= p.M) continue;
#pragma unroll
    for (int c = 0; c < KI; ++c)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int64_t col = (int64_t)kb * TK + wk * (TK / 2) + 32 * c + 8 * g + 4 * ah;
        if (col >= p.K) continue;
        const v4f v = {acc[m][c][4 * g], acc[m][c][4 * g + 1], acc[m][c][4 * g + 2], acc[m][c][4 * g + 3]};
        if (p.S > 1) {
          *reinterpret_cast<v4f*>(p.partial + (split * p.M + row) * p.K + col) = v;
        } else {
          const uint32_t h[4] = {f32_to_bf16(v[0]), f32_to_bf16(v[1]), f32_to_bf16(v[2]), f32_to_bf16(v[3])};
          *reinterpret_cast<uint2*>(p.out + row * p.ldo + col) = uint2{h[0] | h[1] << 16, h[2] | h[3] << 16};
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

}  // namespace mxl

// ------------------------------------------------------------------- C ABI

using namespace mxl;

namespace {

struct GradPlan {
  int TM, TK, S;
  int64_t per;
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

GradPlan grad_plan(int64_t M, int64_t N, int64_t K) {
  GradPlan g{128, 128, 1, 0};
  const int64_t tiles = ceil_div(M, g.TM) * ceil_div(K, g.TK), pairs = ceil_div(N, 2 * kGradStage);
  g.S = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)cu_count() / tiles, pairs / 4, 16}));
  g.per = ceil_div(pairs, g.S) * 2;
  g.S = (int)ceil_div(2 * pairs, g.per);
  return g;
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
  MXL_GRAD(128, 128)
#undef MXL_GRAD
  return hipErrorInvalidValue;
}

}  // namespace

extern "C" int64_t mxl_input_grad_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const GradPlan g = grad_plan(M, N, K);
  return g.S > 1 ? g.S * M * K * 4 : 0;
}

extern "C" int mxl_input_grad(const void* dy, int64_t M, int64_t N, int64_t lddy, const void* w_tiled, const void* sw,
                              int64_t K, int fmt, int block, void* out, int64_t ldo, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  const char* who = "mxl_input_grad";
  MXL_CHECK_ARG(fmt == kE4M3 || fmt == kE2M3 || fmt == kE3M2 || fmt == kE2M1, "%s: unknown format %d", who, fmt);
  MXL_CHECK_ARG(!block || fmt == kE4M3, "%s: block-FP8 weights are E4M3", who);
  MXL_CHECK_ARG(M >= 0 && N > 0 && N % 8 == 0 && K > 0 && K % 128 == 0 && N <= (1 << 22) && K <= (1 << 22) && M <= 0x7FFFFFFF,
                "%s: need N > 0, N %% 8 == 0, K > 0, K %% 128 == 0, both at most 2^22 (M=%lld N=%lld K=%lld)", who,
                (long long)M, (long long)N, (long long)K);
  MXL_CHECK_ARG(lddy >= N && lddy % 8 == 0 && lddy <= (1 << 22) && ldo >= K && ldo % 4 == 0,
                "%s: need lddy >= N, a multiple of 8 up to 2^22, and ldo >= K, a multiple of 4", who);
  MXL_CHECK_ARG((((uintptr_t)dy | (uintptr_t)w_tiled) & 15) == 0 && ((uintptr_t)sw & 3) == 0 && ((uintptr_t)out & 7) == 0,
                "%s: misaligned operands", who);
  if (M == 0) return MXL_OK;
  const GradPlan g = grad_plan(M, N, K);
  const int64_t need = mxl_input_grad_workspace_bytes(M, N, K);
  MXL_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
                "%s: needs a 16-byte aligned workspace of %lld bytes (have %lld)", who, (long long)need,
                (long long)workspace_bytes);
  GradParams p{};
  p.dy = (const uint16_t*)dy; p.w = (const uint8_t*)w_tiled; p.sw = sw; p.out = (uint16_t*)out; p.partial = (float*)workspace;
  p.M = M; p.N = N; p.K = K; p.KT = ceil_div(K, kTileK); p.lddy = lddy; p.ldo = ldo; p.S = g.S; p.per = g.per;
  MXL_CHECK_ARG(ceil_div(M, g.TM) * ceil_div(K, g.TK) * g.S <= 0x7FFFFFFF, "%s: too large", who);
  p.mblocks = (uint32_t)ceil_div(M, g.TM);
  p.kblocks = (uint32_t)ceil_div(K, g.TK);
  p.group_m = std::min<uint32_t>(p.mblocks, 1024 / g.TM);
  hipStream_t s = (hipStream_t)stream;
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
