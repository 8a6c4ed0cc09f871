// What the kernels of gated products share: a problem as the fast ones take it, and its results on their way to memory.
#ifndef IREE_AMD_CSRC_GATED_MMT4D_H_
#define IREE_AMD_CSRC_GATED_MMT4D_H_

#include "product16.h"

namespace uk {

struct GatedResults {
  static constexpr bool kPaired = true, kInTurn = false, kCopies = false;
  uint8_t *out, *gate_pre, *up_pre;  // the latter two null: none
  Layout out_at, gate_at, up_at;
  Curve curve;
  Float out_type, pre_type;
  int32_t pre_load, pre_store;
  int32_t runs;  // eight (f32: four) columns from a multiple of that on lie next to each other, aligned, in all of them

  // A block kernel's fragments. A lane has row lane % 32 and, of 16 columns, 4 g to 4 g + 3 and 8 + 4 g to 8 + 4 g + 3, g = lane /
  // 32, gates in the first half of its registers and ups in the second.
  template <Float T, int AM, int BN>
  __device__ __forceinline__ void store(const p16_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0, uint32_t rows, uint32_t cols,
                                        int lane, uint32_t) const {
    const int r = lane & 31, half = lane >> 5;
#pragma unroll
    for (int i = 0; i < AM; ++i) {
      const uint32_t row = row0 + 32 * i + r;
      if (row >= rows) continue;
      const int64_t out_row = layout_row(out_at, row), gate_row = gate_pre ? layout_row(gate_at, row) : 0,
                    up_row = gate_pre ? layout_row(up_at, row) : 0;
#pragma unroll
      for (int j = 0; j < BN; ++j) {
        __builtin_amdgcn_sched_barrier(0);  // (or many fragments leave the accumulators at once, and registers are spilt)
        const uint32_t col = col0 + 16 * j;
        if (col >= cols) continue;
        float gate[8], up[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          gate[e] = acc[i][j][e];
          up[e] = acc[i][j][8 + e];
        }
        if (runs && col + 16 <= cols) store_runs<T>(gate, up, gate_row, up_row, out_row, col, half);
        else store_one_by_one<T>(gate, up, gate_row, up_row, out_row, col, cols, half);
      }
    }
  }

  template <Float T>
  __device__ __forceinline__ void store_runs(float (&gate)[8], float (&up)[8], int64_t gate_row, int64_t up_row, int64_t out_row,
                                             uint32_t col, int half) const {
    float h[8];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t from = col + 8 * q + 4 * half;
      const int64_t gate_to = gate_pre ? gate_row + layout_col(gate_at, from) : 0, up_to = gate_pre ? up_row + layout_col(up_at, from) : 0;
      if (pre_load) {
        add_four<T>(gate_pre, gate_to, gate + 4 * q);
        add_four<T>(up_pre, up_to, up + 4 * q);
      }
      if (pre_store) {
        put_four<T>(pre_type, gate_pre, gate_to, gate + 4 * q);
        put_four<T>(pre_type, up_pre, up_to, up + 4 * q);
      }
#pragma unroll
      for (int e = 4 * q; e < 4 * q + 4; ++e) h[e] = activated(curve, gate[e]) * up[e];
      if (out_type == Float::kF32) put_four<T>(Float::kF32, out, out_row + layout_col(out_at, from), h + 4 * q);
    }
    if (out_type == Float::kF32) return;
    *(uint4*)((uint16_t*)out + out_row + layout_col(out_at, col + 8 * half)) = eight_of_two_lanes<T>(h);
  }
  template <Float T>
  __device__ __forceinline__ void add_four(const uint8_t* p, int64_t at, float* v) const {
    float old[4];
    if (pre_type == Float::kF32) load_run<Float::kF32, 4>(p, at, old);
    else load_run<T, 4>(p, at, old);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += old[i];
  }
  template <Float T>
  __device__ __forceinline__ void put_four(Float type, uint8_t* p, int64_t at, const float* from) const {
    const float v[4] = {from[0], from[1], from[2], from[3]};
    if (type == Float::kF32) store_run<Float::kF32, 4>(p, at, v);
    else store_run<T, 4>(p, at, v);
  }

  // Four columns from a multiple of four on.
  template <Float T>
  __device__ __forceinline__ void store_four(p16_v4f32 gate, p16_v4f32 up, uint32_t row, uint32_t col, uint32_t cols) const {
    const int64_t out_row = layout_row(out_at, row), gate_row = gate_pre ? layout_row(gate_at, row) : 0,
                  up_row = gate_pre ? layout_row(up_at, row) : 0;
    if (!runs || col + 4 > cols) {
#pragma unroll 1
      for (int e = 0; e < 4; ++e)
        if (col + e < cols) store_one<T>(gate[e], up[e], gate_row, up_row, out_row, col + e);
      return;
    }
    float g[4] = {gate[0], gate[1], gate[2], gate[3]}, u[4] = {up[0], up[1], up[2], up[3]}, h[4];
    const int64_t gate_to = gate_pre ? gate_row + layout_col(gate_at, col) : 0, up_to = gate_pre ? up_row + layout_col(up_at, col) : 0;
    if (pre_load) {
      add_four<T>(gate_pre, gate_to, g);
      add_four<T>(up_pre, up_to, u);
    }
    if (pre_store) {
      put_four<T>(pre_type, gate_pre, gate_to, g);
      put_four<T>(pre_type, up_pre, up_to, u);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = activated(curve, g[e]) * u[e];
    put_four<T>(out_type, out, out_row + layout_col(out_at, col), h);
  }

  // Columns that are not all there, or lie apart.
  template <Float T>
  __device__ __forceinline__ void store_one_by_one(const float (&gate)[8], const float (&up)[8], int64_t gate_row, int64_t up_row,
                                                   int64_t out_row, uint32_t col, uint32_t cols, int half) const {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const uint32_t at = col + 8 * (e >> 2) + 4 * half + (e & 3);
      if (at < cols) store_one<T>(gate[e], up[e], gate_row, up_row, out_row, at);
    }
  }
  template <Float T>
  __device__ __forceinline__ void store_one(float g, float u, int64_t gate_row, int64_t up_row, int64_t out_row, uint32_t col) const {
    if (gate_pre) {
      const int64_t gate_to = gate_row + layout_col(gate_at, col), up_to = up_row + layout_col(up_at, col);
      if (pre_load) {
        g += pre_type == Float::kF32 ? element<Float::kF32>(gate_pre, gate_to) : element<T>(gate_pre, gate_to);
        u += pre_type == Float::kF32 ? element<Float::kF32>(up_pre, up_to) : element<T>(up_pre, up_to);
      }
      if (pre_store) {
        put_element(pre_type, gate_pre, gate_to, g);
        put_element(pre_type, up_pre, up_to, u);
      }
    }
    put_element(out_type, out, out_row + layout_col(out_at, col), activated(curve, g) * u);
  }
};

struct GatedProduct {
  Operand16 lhs, gate;
  const uint8_t* up;
  int64_t up_stride0;  // bytes; everything else as gate's
  uint32_t depth;
  GatedResults results;
};

// The block kernels (product16_block.h): the rows and columns of a workgroup's results.
struct GatedTile {
  int rows, cols;
  const char* name;
};
constexpr GatedTile kGatedTiles[] = {{256, 128, "gated_mmt4d_256x128"}, {256, 96, "gated_mmt4d_256x96"},   {192, 96, "gated_mmt4d_192x96"},
                                     {192, 128, "gated_mmt4d_192x128"}, {128, 128, "gated_mmt4d_128x128"}, {128, 96, "gated_mmt4d_128x96"},
                                     {128, 64, "gated_mmt4d_128x64"},   {64, 128, "gated_mmt4d_64x128"},   {64, 96, "gated_mmt4d_64x96"},
                                     {64, 64, "gated_mmt4d_64x64"},     {64, 32, "gated_mmt4d_64x32"}};
// The kernels for few rows (gated_mmt4d_few.hip): fragments of 16 rows and of 16 results a row that a workgroup multiplies, and
// whether the lhs goes through LDS.
struct GatedFewShape {
  int mt, nt;
  bool staged;
  const char* name;
};
constexpr GatedFewShape kGatedFewShapes[] = {
    {1, 1, false, "gated_mmt4d_few_16x16"},       {1, 2, false, "gated_mmt4d_few_16x32"},       {1, 1, true, "gated_mmt4d_few_16x16_staged"},
    {2, 1, true, "gated_mmt4d_few_32x16_staged"}, {2, 2, true, "gated_mmt4d_few_32x32_staged"}, {4, 1, true, "gated_mmt4d_few_64x16_staged"}};
hipError_t launch_gated_few(const GatedProduct& p, Float type, int shape, hipStream_t stream);
hipError_t launch_gated_block_f16(const GatedProduct& p, int tile, hipStream_t stream);
hipError_t launch_gated_block_bf16(const GatedProduct& p, int tile, hipStream_t stream);

}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_MMT4D_H_
