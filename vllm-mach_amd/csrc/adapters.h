// What the adapters' kernels (adapters.hip) and the products that add them (gemm_tile.h, input_grad.hip) share.
#pragma once

#include "mx_common.h"

namespace mxl {

constexpr int kMaxParts = 8, kMaxRank = 256, kMaxSlots = 2048, kAdapterTile = 16;

// Tokens sorted by adapter: positions [offsets[a], offsets[a + 1]) of order are adapter a's, in tiles of 16 positions:
// tile i is (adapter, first position, end, 0), adapter -1 past the last.
struct AdapterBatch {
  const int32_t* order;
  const int64_t* offsets;
  const int32_t* tiles;
  int num_tiles;
  int64_t M;
};

// v of a token: its parts' ranks, each part padded to groups of 16, as bf16 [2][width]: the values, then what bf16 left of
// them.  A token without an adapter has none (its v is never written).
struct LowRank {
  int parts, rank, groups;  // groups: of 16 ranks of a part
  int64_t cols[kMaxParts + 1];
  __host__ __device__ int width() const { return parts * groups * 16; }
};

// What a product adds of a batch's adapters to its sums, ahead of their rounding: for a row t of adapter ids[t] (outside
// [0, slots): none) the products of v[t] with mat, B [N, ldm] for y += B v (of a column's part), or A [R, ldm] for
// dx += A^T dv (of all parts).  slot_stride: of mat's adapters.
struct RowAdapters {
  const int32_t* ids = nullptr;
  int slots = 0;
  const uint16_t* v = nullptr;
  const uint16_t* mat = nullptr;
  int64_t slot_stride = 0, ldm = 0;
  LowRank l{};
};

// Whether a product adds the adapters of its rows itself: it walks the adapters of a tile's rows one after the other (some
// 4 us each on the largest tile, waits for memory), so that few rows an adapter, and rows of many adapters, are better added
// by a launch of their own (adapter_expand_kernel).  MXFP8 layers with ranks of 16 or (17408 x 5120, 8 adapters) 64, us in
// one product / apart, tokens in runs of an adapter and, the worst case, mixed at random:
//   256 x 5120 x 2560, 8 adapters: 23 / 25, mixed 28 / 26       2048 x 17408 x 5120, 8 adapters: 207 / 276, mixed 296 / 288
//   1024 x 5120 x 2560, 32: 36 / 40, mixed 56 / 42              2048 x 17408 x 5120, 64: 194 / 210, mixed 374 / 215
// The rule has no N or K in it, and few tiles of a long K lose by that, one adapter each 32 rows or more: 64 x 2560 x 17408, 2
// adapters, 64 / 28; 256 x 2560 x 17408, 8: 68 / 39; 64 x 512 x 5120, 2: 23 / 17; even at 64 x 17408 x 5120, 2: 32 / 30.
inline bool rows_add(int64_t M, int64_t slots) { return slots <= 16 && M >= 32 * slots; }

// A product multiplies an adapter's values with zeros too, in rows of other adapters and columns of other parts, where an
// infinity or NaN must not count.  So it multiplies the finite ones only (adapter_odd finds a wave's others, which
// adapter_finite takes out), and a wave that met others adds their terms to what it has stored (adapter_odd_term).  Looking
// for them takes two instructions a register of values: 4096 x 17408 x 5120 with ranks of 64 371 -> 376 us, the training step
// of 2048 x 18432 x 2560 365 -> 367.
// Whether one of the lane's bf16 values is an infinity or NaN: `top`, the largest of the packed magnitudes.
typedef unsigned short adapter_u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t adapter_top(uint32_t top, uint32_t pair) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(adapter_u16x2, top),
                                                                __builtin_bit_cast(adapter_u16x2, pair & 0x7FFF7FFFu)));
}
__device__ __forceinline__ bool adapter_odd(uint32_t top) { return (top & 0xFFFFu) >= 0x7F80u || top >= 0x7F800000u; }
__device__ __forceinline__ uint32_t adapter_finite(uint32_t pair) {
  const uint32_t h = pair & 0x7FFF7FFFu;
  return pair & ((h & 0xFFFFu) >= 0x7F80u ? 0xFFFF0000u : 0xFFFFFFFFu) & (h >= 0x7F800000u ? 0x0000FFFFu : 0xFFFFFFFFu);
}
// mat v of bf16 values where one of them is not finite (v as its value and what bf16 left of it); `odd`: there was one.
__device__ __forceinline__ float adapter_odd_term(uint16_t mat, uint16_t v, uint16_t rest, bool& odd) {
  if ((mat & 0x7FFF) < 0x7F80 && (v & 0x7FFF) < 0x7F80) return 0.0f;
  odd = true;
  return bf16_to_f32(mat) * (bf16_to_f32(v) + bf16_to_f32(rest));
}

// dx = dy W (input_grad.hip), with `more` the adapters' dx as well.
int64_t input_grad_bytes(int64_t M, int64_t N, int64_t K, int block);
int input_grad(const char* who, const void* dy, int64_t M, int64_t N, int64_t lddy, const void* w, const void* sw, int64_t K,
               int fmt, int block, void* out, int64_t ldo, void* workspace, int64_t workspace_bytes, const RowAdapters* more,
               void* stream);

}  // namespace mxl
