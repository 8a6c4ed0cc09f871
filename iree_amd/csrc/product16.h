// Products of 16-bit floats whose operands have K in 64-byte chunks: what the block kernels (product16_block.h) and the few-row
// kernel of gated products (gated_mmt4d_few.hip) are given.
#ifndef IREE_AMD_CSRC_PRODUCT16_H_
#define IREE_AMD_CSRC_PRODUCT16_H_

#include "gated_device.h"

namespace uk {

// Row i of an operand lies in panel i / tile_rows, row_bytes apart within it; its K comes in 16-byte pieces, four to a chunk of 32
// values: piece c of a chunk is (c & 1) * piece1 + (c >> 1) * piece2 from the chunk's first, and chunks are 64 * tile_rows apart.
// Tiles one row tall of any K0 are that, and tiles with a K0 of 8, 16 or 32.
struct Operand16 {
  const uint8_t* data;
  int64_t stride0;  // bytes from a panel to the next
  uint32_t rows, tile_rows, tile_reciprocal;
  uint32_t row_bytes, piece1, piece2;
  uint32_t log2_pieces;  // of a chunk's pieces of a row lie next to each other: 4, 2 or 1
};

// An operand whose rows' values of one k lie next to each other: element (k, row) in panel k / tile_rows, row_bytes apart within it, and
// then as a matrix of tiles has its columns (tiles n0 wide, tile_bytes apart). tile_rows is 1, 2, 4, .. 32, n0 a multiple of 8.
struct Strided16 {
  const uint8_t* data;
  int64_t stride0;  // bytes from a panel to the next
  uint32_t rows, log2_tile_rows, row_bytes, n0, n0_reciprocal, tile_bytes;
};

// A result or another matrix laid out like it: element (row, col) at row / tile_rows * stride0 + (col / n0) * tile + (row %
// tile_rows) * n0 + col % n0.
struct Layout {
  int64_t stride0;  // elements
  uint32_t tile_rows, tile_reciprocal, n0, n0_reciprocal, tile;
};

__device__ __forceinline__ int64_t layout_row(const Layout& l, uint32_t row) {
  const uint32_t panel = divide(row, l.tile_rows, l.tile_reciprocal);
  return (int64_t)panel * l.stride0 + (int64_t)(row - panel * l.tile_rows) * l.n0;
}
__device__ __forceinline__ int64_t layout_col(const Layout& l, uint32_t col) {
  const uint32_t tile = divide(col, l.n0, l.n0_reciprocal);
  return (int64_t)tile * l.tile + (col - tile * l.n0);
}

// Whether an operand is one, and it then. (false: the kernels with one thread for each result.)
inline bool as_operand16(const uint8_t* data, int64_t stride0, int64_t panels, int64_t M0, int64_t K, int64_t K0, Operand16* o) {
  const int64_t rows = panels * M0;
  if (rows == 0 || rows > 0x7FFFFFFF - 512 || M0 > 512) return false;
  if (M0 != 1 && K0 != 8 && K0 != 16 && K0 != 32) return false;
  if ((uintptr_t)data % 16 != 0 || (panels > 1 && stride0 % 8 != 0)) return false;
  const uint32_t m0 = (uint32_t)M0, k0 = M0 == 1 ? 32 : (uint32_t)K0;
  o->data = data;
  o->stride0 = panels > 1 ? 2 * stride0 : 0;
  o->rows = (uint32_t)rows;
  o->tile_rows = m0;
  o->tile_reciprocal = reciprocal_of(m0);
  o->row_bytes = m0 == 1 ? 0 : 2 * k0;
  o->piece1 = k0 == 8 ? 16 * m0 : 16;
  o->piece2 = k0 == 32 ? 32 : 32 * m0;
  o->log2_pieces = k0 == 32 ? 2 : k0 == 16 ? 1 : 0;
  return true;
}
// The same matrix [panels][K][M0][K0] with its first dimension contracted. (32 of its rows within 31 bits of each other.)
inline bool as_strided16(const uint8_t* data, int64_t stride0, int64_t panels, int64_t M0, int64_t K, int64_t K0, Strided16* o) {
  const int64_t cols = K * K0, n0 = M0 == 1 ? cols : K0;
  if (cols == 0 || cols > 0x7FFFFFFF - 512 || n0 % 8 != 0 || M0 > 32 || (M0 & (M0 - 1)) != 0) return false;
  if ((uintptr_t)data % 16 != 0 || (panels > 1 && stride0 % 8 != 0)) return false;
  const int64_t apart = panels > 1 ? 2 * stride0 : 0;
  if (apart * (32 / M0) + 2 * M0 * cols >= 1ll << 31) return false;
  o->data = data;
  o->stride0 = apart;
  o->rows = (uint32_t)cols;
  o->log2_tile_rows = (uint32_t)__builtin_ctz((unsigned)M0);
  o->row_bytes = M0 == 1 ? 0 : (uint32_t)(2 * K0);
  o->n0 = (uint32_t)n0;
  o->n0_reciprocal = reciprocal_of(o->n0);
  o->tile_bytes = M0 == 1 ? 0 : (uint32_t)(2 * M0 * K0);
  return true;
}
// Whether rows up to `apart` apart lie within 31 bits of each other.
inline bool near16(const Operand16& o, int64_t apart) { return o.stride0 < (1ll << 31) / (apart / o.tile_rows + 2); }

inline Layout layout_of(int64_t stride0, int64_t M0, int64_t N, int64_t N0) {
  Layout l;
  l.stride0 = stride0;
  l.tile_rows = (uint32_t)M0;
  l.tile_reciprocal = reciprocal_of(l.tile_rows);
  // (Tiles one row tall are a row-major matrix, whatever their width.)
  l.n0 = M0 == 1 ? (uint32_t)(N * N0) : (uint32_t)N0;
  l.n0_reciprocal = reciprocal_of(l.n0);
  l.tile = M0 == 1 ? 0 : (uint32_t)(M0 * N0);
  return l;
}
// Whether `count` columns from a multiple of it on lie next to each other at an address that is a multiple of `to` bytes. (Of a
// row-major matrix the last ones may be fewer.)
inline bool runs_of(const Layout& l, const uint8_t* p, int64_t panels, int size, int count, int to) {
  return (l.tile_rows == 1 || l.n0 % count == 0) && (uintptr_t)p % to == 0 && (panels <= 1 || l.stride0 * size % to == 0);
}

typedef float p16_v4f32 __attribute__((ext_vector_type(4)));
typedef float p16_v16f32 __attribute__((ext_vector_type(16)));
typedef _Float16 p16_v8f16 __attribute__((ext_vector_type(8)));
typedef __bf16 p16_v8bf16 __attribute__((ext_vector_type(8)));

// Rows of the result along `a`'s rows (a lane has four consecutive ones), columns along b's.
template <Float T>
__device__ __forceinline__ p16_v16f32 mfma16_32(uint4 a, uint4 b, p16_v16f32 acc) {
  if constexpr (T == Float::kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(p16_v8f16, a), __builtin_bit_cast(p16_v8f16, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(p16_v8bf16, a), __builtin_bit_cast(p16_v8bf16, b), acc, 0, 0, 0);
}
template <Float T>
__device__ __forceinline__ p16_v4f32 mfma16_16(uint4 a, uint4 b, p16_v4f32 acc) {
  if constexpr (T == Float::kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(p16_v8f16, a), __builtin_bit_cast(p16_v8f16, b), acc, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(p16_v8bf16, a), __builtin_bit_cast(p16_v8bf16, b), acc, 0, 0, 0);
}

// A 16-byte piece of which the first `exist` values are there; the others are zero.
__device__ __forceinline__ uint4 last_piece(const uint8_t* at, int exist) {
  if (exist >= 8) return *(const uint4*)at;
  uint64_t low = 0, high = 0;
  for (int e = exist - 1; e >= 0; --e) {
    high = high << 16 | low >> 48;
    low = low << 16 | ((const uint16_t*)at)[e];
  }
  return make_uint4((uint32_t)low, (uint32_t)(low >> 32), (uint32_t)high, (uint32_t)(high >> 32));
}

// The same at an address that is a multiple of 2 only. (Loads of 16 bytes need no alignment here.)
__device__ __forceinline__ uint4 last_piece_anywhere(const uint8_t* at, int exist) {
  if (exist < 8) return last_piece(at, exist);
  uint4 v;
  __builtin_memcpy(&v, at, 16);
  return v;
}

// COUNT (4 or 8) consecutive elements at an address that is a multiple of their size, of 16 bytes at most.
template <Float T, int COUNT>
__device__ __forceinline__ void load_run(const uint8_t* p, int64_t at, float (&v)[COUNT]) {
  if constexpr (T == Float::kF32) {
    __builtin_memcpy(v, __builtin_assume_aligned((const float*)p + at, 16), 4 * COUNT);
  } else {
    uint32_t w[COUNT / 2];
    __builtin_memcpy(w, __builtin_assume_aligned((const uint16_t*)p + at, 2 * COUNT), 2 * COUNT);
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = mx_widen<T>((uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }
}
template <Float T, int COUNT>
__device__ __forceinline__ void store_run(uint8_t* p, int64_t at, const float (&v)[COUNT]) {
  if constexpr (T == Float::kF32) {
    __builtin_memcpy(__builtin_assume_aligned((float*)p + at, 16), v, 4 * COUNT);
  } else {
    uint32_t w[COUNT / 2];
#pragma unroll
    for (int i = 0; i < COUNT; i += 2) w[i / 2] = mx_narrow_pair<T>(v[i], v[i + 1]);
    __builtin_memcpy(__builtin_assume_aligned((uint16_t*)p + at, 2 * COUNT), w, 2 * COUNT);
  }
}

// Of sixteen columns of a row two lanes, 32 apart, have 4 half to + 3 and 8 + 4 half to + 3. They exchange halves, and each returns
// eight consecutive ones, from 8 half on, rounded.
template <Float T>
__device__ __forceinline__ uint4 eight_of_two_lanes(const float (&v)[8]) {
  typedef uint32_t v2u32 __attribute__((ext_vector_type(2)));
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const v2u32 both = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane32_swap(mx_narrow_pair<T>(v[2 * e], v[2 * e + 1]),
                                                                                  mx_narrow_pair<T>(v[4 + 2 * e], v[5 + 2 * e]), false, false));
    w[e] = both[0];
    w[2 + e] = both[1];
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace uk

#endif  // IREE_AMD_CSRC_PRODUCT16_H_
