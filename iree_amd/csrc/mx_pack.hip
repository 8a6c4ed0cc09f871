// Quantisation into microscaled tiles and back: iree_uk_mi355x_mx_pack_p and iree_uk_mi355x_mx_unpack_p.
//
// Both are bound by memory: 2 or 4 bytes a value on the plain side, 0.53 or 1.03 on the other. A lane takes eight consecutive
// values of a row and four neighbouring lanes a block, so a block's maximum is two exchanges within a quad of lanes and
// nothing passes through LDS. Lanes follow each other in the order of the codes.
#include <type_traits>

#include "mx_device.h"
#include "uk_device.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

// Where the eight values of segment n (the n-th of the tiled order) lie.
struct MxPlace {
  int64_t row, col;      // in the matrix
  int64_t code, scale;   // bytes from the operand's start; of the block that the segment belongs to
};

template <typename INDEX>
struct MxShape {
  INDEX segments;             // of 8 values, in all
  INDEX row_segments, tile0, outer1;
  uint32_t row_reciprocal, tile0_reciprocal, outer1_reciprocal;
  int64_t codes_stride0, scales_stride0;
};

template <int BITS, typename INDEX>
__device__ __forceinline__ MxPlace mx_place(const MxShape<INDEX>& s, INDEX n) {
  INDEX q, seg, t0, o1, o0;
  if constexpr (sizeof(INDEX) == 4) {
    q = divide(n, s.row_segments, s.row_reciprocal);
    seg = n - q * s.row_segments;
    const INDEX tile = divide(q, s.tile0, s.tile0_reciprocal);
    t0 = q - tile * s.tile0;
    o0 = divide(tile, s.outer1, s.outer1_reciprocal);
    o1 = tile - o0 * s.outer1;
  } else {
    q = n / s.row_segments;
    seg = n - q * s.row_segments;
    const INDEX tile = q / s.tile0;
    t0 = q - tile * s.tile0;
    o0 = tile / s.outer1;
    o1 = tile - o0 * s.outer1;
  }
  MxPlace p;
  p.row = (int64_t)o0 * s.tile0 + t0;
  p.col = ((int64_t)o1 * s.row_segments + seg) * 8;
  const int64_t in_panel = ((int64_t)o1 * s.tile0 + t0) * s.row_segments + seg;
  p.code = (int64_t)o0 * s.codes_stride0 + in_panel * BITS;
  p.scale = (int64_t)o0 * s.scales_stride0 + in_panel / 4;
  return p;
}

template <typename INDEX>
struct MxPackKernelArgs {
  MxShape<INDEX> shape;
  const uint8_t* in;
  uint8_t* codes;
  uint8_t* scales;
  int64_t in_stride0, in_stride1, in_size0, in_size1;
};

template <typename INDEX>
struct MxUnpackKernelArgs {
  MxShape<INDEX> shape;
  const uint8_t* codes;
  const uint8_t* scales;
  uint8_t* out;
  int64_t out_stride0, out_stride1, out_size0, out_size1;
};

// Rows whose values are next to each other (in_stride1 == 1).
template <Float T, int BITS, int AT_ONCE, typename INDEX>
__global__ __launch_bounds__(kThreads) void mx_pack_rows(const MxPackKernelArgs<INDEX> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  const INDEX first = (INDEX)blockIdx.x * (kThreads * AT_ONCE) + threadIdx.x;
  MxEight<T> v[AT_ONCE];
  MxPlace p[AT_ONCE];
#pragma unroll
  for (int u = 0; u < AT_ONCE; ++u) {
    const INDEX n = first + (INDEX)(u * kThreads);
    if (n >= a.shape.segments) break;
    p[u] = mx_place<BITS>(a.shape, n);
    const int64_t left = p[u].row < a.in_size0 ? a.in_size1 - p[u].col : 0;
    mx_load<T>(v[u], a.in + (p[u].row * a.in_stride0 + p[u].col) * SIZE, left);
  }
#pragma unroll
  for (int u = 0; u < AT_ONCE; ++u) {
    if (first + (INDEX)(u * kThreads) >= a.shape.segments) break;  // (segments come in fours: a block's lanes leave together)
    const uint32_t b = mx_scale_byte<BITS>(mx_largest_of_block(mx_largest<T>(v[u])));
    uint32_t codes[BITS / 4];
    mx_codes<BITS, T>(v[u], b, codes);
    __builtin_memcpy(a.codes + p[u].code, codes, BITS);
    if (threadIdx.x % 4 == 0) a.scales[p[u].scale] = (uint8_t)b;
  }
}

// Any strides: a lane takes a whole block and neighbouring lanes neighbouring rows, whose values are next to each other in
// a transposed matrix. Block number n: rows fastest.
template <Float T, int BITS>
__global__ __launch_bounds__(kThreads) void mx_pack_strided(const MxPackKernelArgs<uint64_t> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  const MxShape<uint64_t>& s = a.shape;
  const uint64_t rows = s.segments / (s.outer1 * s.row_segments), blocks = s.segments / 4;
  for (uint64_t n = (uint64_t)blockIdx.x * kThreads + threadIdx.x; n < blocks; n += (uint64_t)gridDim.x * kThreads) {
    const uint64_t row = n % rows, block = n / rows;
    const uint64_t o0 = row / s.tile0, t0 = row % s.tile0, o1 = block / (s.row_segments / 4), in_row = block % (s.row_segments / 4);
    MxEight<T> v[4];
    uint32_t largest = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int64_t col = (int64_t)block * 32 + h * 8 + i;
        const bool there = (int64_t)row < a.in_size0 && col < a.in_size1;
        const uint8_t* at = a.in + ((int64_t)row * a.in_stride0 + col * a.in_stride1) * SIZE;
        if constexpr (T == Float::kF32) {
          v[h].w[i] = there ? *(const uint32_t*)at : 0;
        } else {
          const uint32_t x = there ? *(const uint16_t*)at : 0;
          v[h].w[i / 2] = i & 1 ? v[h].w[i / 2] | x << 16 : x;
        }
      }
      const uint32_t m = mx_largest<T>(v[h]);
      largest = m > largest ? m : largest;
    }
    const uint32_t b = mx_scale_byte<BITS>(largest);
    uint32_t codes[BITS];
#pragma unroll
    for (int h = 0; h < 4; ++h) mx_codes<BITS, T>(v[h], b, codes + h * (BITS / 4));
    const int64_t in_panel = (int64_t)((o1 * s.tile0 + t0) * s.row_segments + in_row * 4);
    __builtin_memcpy(a.codes + (int64_t)o0 * s.codes_stride0 + in_panel * BITS, codes, 4 * BITS);
    a.scales[(int64_t)o0 * s.scales_stride0 + in_panel / 4] = (uint8_t)b;
  }
}

template <Float T, int BITS, int AT_ONCE, typename INDEX>
__global__ __launch_bounds__(kThreads) void mx_unpack_rows(const MxUnpackKernelArgs<INDEX> a) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  // (One turn, but for operands of 2^34 values and more.)
  for (INDEX first = (INDEX)blockIdx.x * (kThreads * AT_ONCE) + threadIdx.x; first < a.shape.segments;
       first += (INDEX)gridDim.x * (kThreads * AT_ONCE)) {
    uint32_t codes[AT_ONCE][BITS / 4], b[AT_ONCE];
    MxPlace p[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const INDEX n = first + (INDEX)(u * kThreads);
      if (n >= a.shape.segments) break;
      p[u] = mx_place<BITS>(a.shape, n);
      __builtin_memcpy(codes[u], a.codes + p[u].code, BITS);
      b[u] = a.scales[p[u].scale];
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (first + (INDEX)(u * kThreads) >= a.shape.segments) break;
      const int64_t left = p[u].row < a.out_size0 ? a.out_size1 - p[u].col : 0;
      if (left <= 0) continue;
      float f[8];
      mx_values<BITS>(codes[u], b[u], f);
      if (a.out_stride1 == 1) {
        mx_store_eight<T>(a.out + (p[u].row * a.out_stride0 + p[u].col) * SIZE, f, left);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) mx_store_eight<T>(a.out + (p[u].row * a.out_stride0 + (p[u].col + i) * a.out_stride1) * SIZE, f + i, 1);
      }
    }
  }
}

template <typename INDEX>
MxShape<INDEX> mx_shape(int64_t outer0, int64_t outer1, int64_t tile0, int64_t tile1, int64_t codes_stride0,
                        int64_t scales_stride0) {
  MxShape<INDEX> s;
  s.row_segments = (INDEX)(tile1 / 8);
  s.tile0 = (INDEX)tile0;
  s.outer1 = (INDEX)outer1;
  s.segments = (INDEX)(outer0 * outer1 * tile0 * (tile1 / 8));
  s.row_reciprocal = s.tile0_reciprocal = s.outer1_reciprocal = 0;
  if constexpr (sizeof(INDEX) == 4) {
    s.row_reciprocal = reciprocal_of(s.row_segments);
    s.tile0_reciprocal = reciprocal_of(s.tile0);
    s.outer1_reciprocal = reciprocal_of(s.outer1);
  }
  s.codes_stride0 = codes_stride0;
  s.scales_stride0 = scales_stride0;
  return s;
}

// (Fits: the tiles of a result lie apart in memory.)
int64_t segments_of(int64_t outer0, int64_t outer1, int64_t tile0, int64_t tile1) { return outer0 * outer1 * tile0 * (tile1 / 8); }

template <Float T, int BITS>
hipError_t pack(const MxPackArgs& a, hipStream_t stream, const char** name) {
  const int64_t segments = segments_of(a.outer0, a.outer1, a.tile0, a.tile1);
  auto fill = [&](auto& k) {
    k.in = a.in; k.codes = a.codes; k.scales = a.scales;
    k.in_stride0 = a.in_stride0; k.in_stride1 = a.in_stride1;
    k.in_size0 = a.in_size0; k.in_size1 = a.in_size1;
  };
  if (a.in_stride1 == 1 && segments < (1ll << 31)) {
    MxPackKernelArgs<uint32_t> k;
    k.shape = mx_shape<uint32_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
    fill(k);
    *name = "mx_pack_rows";
    constexpr int MANY = 4;
    if (segments >= (int64_t)MANY * kThreads * 1024)
      return launch_kernel(mx_pack_rows<T, BITS, MANY, uint32_t>,
                           (unsigned)((segments + MANY * kThreads - 1) / (MANY * kThreads)), kThreads, 0, stream, k);
    return launch_kernel(mx_pack_rows<T, BITS, 1, uint32_t>, (unsigned)((segments + kThreads - 1) / kThreads), kThreads, 0,
                         stream, k);
  }
  MxPackKernelArgs<uint64_t> k;
  k.shape = mx_shape<uint64_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
  fill(k);
  *name = "mx_pack_strided";
  const int64_t groups = (segments / 4 + kThreads - 1) / kThreads;
  return launch_kernel(mx_pack_strided<T, BITS>, (unsigned)(groups < (1 << 22) ? groups : 1 << 22), kThreads, 0, stream, k);
}

template <Float T, int BITS>
hipError_t unpack(const MxUnpackArgs& given, hipStream_t stream, const char** name) {
  // Tiles that hold nothing of the result are not visited (panels may coincide, so that their number says nothing).
  MxUnpackArgs a = given;
  a.outer0 = (a.out_size0 - 1) / a.tile0 + 1;
  a.outer1 = (a.out_size1 - 1) / a.tile1 + 1;
  const int64_t segments = segments_of(a.outer0, a.outer1, a.tile0, a.tile1);
  auto fill = [&](auto& k) {
    k.codes = a.codes; k.scales = a.scales; k.out = a.out;
    k.out_stride0 = a.out_stride0; k.out_stride1 = a.out_stride1;
    k.out_size0 = a.out_size0; k.out_size1 = a.out_size1;
  };
  *name = "mx_unpack_rows";
  constexpr int MANY = 4;
  const unsigned groups = (unsigned)((segments + kThreads - 1) / kThreads);
  if (segments < (1ll << 31)) {
    MxUnpackKernelArgs<uint32_t> k;
    k.shape = mx_shape<uint32_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
    fill(k);
    if (segments >= (int64_t)MANY * kThreads * 1024)
      return launch_kernel(mx_unpack_rows<T, BITS, MANY, uint32_t>,
                           (unsigned)((segments + MANY * kThreads - 1) / (MANY * kThreads)), kThreads, 0, stream, k);
    return launch_kernel(mx_unpack_rows<T, BITS, 1, uint32_t>, groups, kThreads, 0, stream, k);
  }
  MxUnpackKernelArgs<uint64_t> k;
  k.shape = mx_shape<uint64_t>(a.outer0, a.outer1, a.tile0, a.tile1, a.codes_stride0, a.scales_stride0);
  fill(k);
  return launch_kernel(mx_unpack_rows<T, BITS, MANY, uint64_t>, 1u << 21, kThreads, 0, stream, k);
}

}  // namespace

hipError_t launch_mx_pack(const MxPackArgs& a, hipStream_t stream, const char** name) {
  const bool four = a.bits == 4;
  switch (a.type) {
    case Float::kF32: return four ? pack<Float::kF32, 4>(a, stream, name) : pack<Float::kF32, 8>(a, stream, name);
    case Float::kF16: return four ? pack<Float::kF16, 4>(a, stream, name) : pack<Float::kF16, 8>(a, stream, name);
    default: return four ? pack<Float::kBf16, 4>(a, stream, name) : pack<Float::kBf16, 8>(a, stream, name);
  }
}

hipError_t launch_mx_unpack(const MxUnpackArgs& a, hipStream_t stream, const char** name) {
  const bool four = a.bits == 4;
  switch (a.type) {
    case Float::kF32: return four ? unpack<Float::kF32, 4>(a, stream, name) : unpack<Float::kF32, 8>(a, stream, name);
    case Float::kF16: return four ? unpack<Float::kF16, 4>(a, stream, name) : unpack<Float::kF16, 8>(a, stream, name);
    default: return four ? unpack<Float::kBf16, 4>(a, stream, name) : unpack<Float::kBf16, 8>(a, stream, name);
  }
}

}  // namespace uk
