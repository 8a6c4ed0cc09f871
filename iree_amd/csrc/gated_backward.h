// What the translation units of the gated products' backward pass share: the products of its gradients, as the block kernels
// (product16_block.h) take them.
#ifndef IREE_AMD_CSRC_GATED_BACKWARD_H_
#define IREE_AMD_CSRC_GATED_BACKWARD_H_

#include "product16.h"

namespace uk {

// Gradients on their way to memory: copies of one layout (but for their strides), of which the first two have addresses of their own and
// all of a lhs gradient's parts lie `apart` bytes behind each other.
struct GradResults {
  uint8_t* out[2];
  int64_t stride0[2];
  int64_t apart;
  Layout at;
  Float type;
  const float* unit;           // of f16 operands: what dg and du are multiples of, a power of two
  int32_t accumulate;
  int32_t runs;                // eight (f32: four) columns from a multiple of that on lie next to each other, aligned
  uint32_t rows;               // of each
  uint32_t copies, tile_rows_of_copy, tile_rows_reciprocal;

  template <Float T, int AM, int BN>
  __device__ __forceinline__ void store_all(const p16_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0, uint32_t cols, int lane,
                                            uint8_t* to, int64_t of_stride0) const {
    const int r = lane & 31, half = lane >> 5;
    Layout l = at;
    l.stride0 = of_stride0;
    const float of_one = T == Float::kF16 ? *unit : 1;
#pragma unroll
    for (int i = 0; i < AM; ++i) {
      const uint32_t row = row0 + 32 * i + r;
      if (row >= rows) continue;
      const int64_t row_at = layout_row(l, row);
#pragma unroll
      for (int j = 0; j < BN; ++j) {
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          __builtin_amdgcn_sched_barrier(0);  // (or many fragments leave the accumulators at once, and registers are spilt)
          const uint32_t col = col0 + 32 * j + 8 * q;
          if (col >= cols) continue;
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = T == Float::kF16 ? acc[i][j][4 * q + e] * of_one : acc[i][j][4 * q + e];
          if (runs && col + 16 <= cols) store_runs<T>(v, to, l, row_at, col, half);
          else store_one_by_one<T>(v, to, l, row_at, col, cols, half);
        }
      }
    }
  }
  // A lane has columns 4 `half` to + 3 and 8 + 4 `half` to + 3 of sixteen.
  template <Float T>
  __device__ __forceinline__ void store_runs(float (&v)[8], uint8_t* to, const Layout& l, int64_t row_at, uint32_t col, int half) const {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t at = row_at + layout_col(l, col + 8 * q + 4 * half);
      float old[4] = {};
      if (accumulate) {
        if (type == Float::kF32) load_run<Float::kF32, 4>(to, at, old);
        else load_run<T, 4>(to, at, old);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] += old[e];
      if (type == Float::kF32) {
        const float x[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        store_run<Float::kF32, 4>(to, at, x);
      }
    }
    if (type == Float::kF32) return;
    *(uint4*)((uint16_t*)to + row_at + layout_col(l, col + 8 * half)) = eight_of_two_lanes<T>(v);
  }
  template <Float T>
  __device__ __forceinline__ void store_one_by_one(const float (&v)[8], uint8_t* to, const Layout& l, int64_t row_at, uint32_t col,
                                                   uint32_t cols, int half) const {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const uint32_t c = col + 8 * (e >> 2) + 4 * half + (e & 3);
      if (c >= cols) continue;
      const int64_t at = row_at + layout_col(l, c);
      put_element(type, to, at, accumulate ? element(type, to, at) + v[e] : v[e]);
    }
  }
};
struct LhsGrad : GradResults {
  static constexpr bool kPaired = false, kInTurn = true, kCopies = true;
  template <Float T, int AM, int BN>
  __device__ __forceinline__ void store(const p16_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0, uint32_t, uint32_t cols, int lane,
                                        uint32_t copy) const {
    store_all<T>(acc, row0, col0, cols, lane, out[0] + copy * apart, stride0[0]);
  }
};
struct WeightGrads : GradResults {
  static constexpr bool kPaired = false, kInTurn = false, kCopies = true;
  template <Float T, int AM, int BN>
  __device__ __forceinline__ void store(const p16_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0, uint32_t, uint32_t cols, int lane,
                                        uint32_t copy) const {
    store_all<T>(acc, row0, col0, cols, lane, copy ? out[1] : out[0], copy ? stride0[1] : stride0[0]);
  }
};

struct LhsGradProduct {
  Operand16 grads;         // [rows][dg, du], lhs_second bytes apart
  Strided16 gate;
  const uint8_t* up;
  int64_t up_stride0, lhs_second;
  uint32_t depth;          // columns of dg
  GradResults results;
};
struct WeightGradProduct {
  Strided16 grads;
  Strided16 lhs;
  int64_t lhs_second;
  uint32_t depth;          // rows
  GradResults results;
};

// Rows and columns of a workgroup's results.
struct GradTile {
  int rows, cols;
};
constexpr GradTile kGradTiles[] = {{256, 256}, {256, 128}, {128, 256}, {128, 128}, {128, 64}, {64, 128}, {64, 64}};
constexpr int kSmallestGradTile = 6;
hipError_t launch_lhs_grad_f16(const LhsGradProduct& p, int tile, hipStream_t stream);
hipError_t launch_lhs_grad_bf16(const LhsGradProduct& p, int tile, hipStream_t stream);
hipError_t launch_weight_grad_f16(const WeightGradProduct& p, int tile, hipStream_t stream);
hipError_t launch_weight_grad_bf16(const WeightGradProduct& p, int tile, hipStream_t stream);
// Both in one launch, in tiles of 64x64.
hipError_t launch_both_grads_f16(const LhsGradProduct& lhs, const WeightGradProduct& weights, hipStream_t stream);
hipError_t launch_both_grads_bf16(const LhsGradProduct& lhs, const WeightGradProduct& weights, hipStream_t stream);

}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_BACKWARD_H_
