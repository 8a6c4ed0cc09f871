// Microscaled products of few rows: the rhs (the weights) is streamed from memory straight into registers, once, and K is
// split over the wavefronts of a workgroup.
#include <type_traits>

#include "mx_mmt4d.h"

namespace uk {
namespace {

// Four chunks' scales of sixteen rows: lane (g, r) has loaded those of row r in chunk g, and gets block g's in chunk u as byte u,
// where the matrix instruction picks it from. One load for what takes four if every lane loads its own bytes.
__device__ __forceinline__ uint32_t scales_of_blocks(uint32_t loaded, int g) {
  typedef uint32_t v2u32 __attribute__((ext_vector_type(2)));
  const v2u32 halves = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane32_swap(loaded, loaded, false, false));
  const v2u32 low = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false));
  const v2u32 high = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false));
  const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t)g;  // byte g of the second operand, then of the first
  return __builtin_amdgcn_perm(low[1], low[0], pick) | __builtin_amdgcn_perm(high[1], high[0], pick) << 16;
}

// A workgroup multiplies 16 * MT rows of the lhs with 16 * NT of the rhs; its wavefronts take four chunks of 128 of K in turn, and
// add their sums through LDS in the order of their numbers. A chunk's registers are loaded again as soon as it is multiplied.
// Rows beyond the last are read as the last one and not stored.
template <int LBITS, int MT, int NT, int WAVES, bool STREAM, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void mx_mmt4d_few_kernel(const MxProduct p) {
  __shared__ mx_v4f32 partial[WAVES][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t first_col = blockIdx.x * (16 * NT), first_row = blockIdx.y * (16 * MT);

  const uint8_t *rhs[NT], *rhs_scales[NT], *lhs[MT], *lhs_scales[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint32_t col = first_col + 16 * j + r, row = col < p.rhs.rows ? col : p.rhs.rows - 1;
    rhs[j] = p.rhs.codes + mx_row_codes<4>(p.rhs, row) + 16 * g;
    rhs_scales[j] = p.rhs.scales + mx_row_scales(p.rhs, row);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const uint32_t at = first_row + 16 * i + r, row = at < p.lhs.rows ? at : p.lhs.rows - 1;
    lhs[i] = p.lhs.codes + mx_row_codes<LBITS>(p.lhs, row) + 16 * g;
    lhs_scales[i] = p.lhs.scales + mx_row_scales(p.lhs, row);
  }
  const int64_t rhs_step = 64 * (int64_t)p.rhs.tile_rows, lhs_step = 16 * LBITS * (int64_t)p.lhs.tile_rows;
  const int64_t rhs_scales_step = 4 * (int64_t)p.rhs.tile_rows, lhs_scales_step = 4 * (int64_t)p.lhs.tile_rows;

  mx_v4f32 acc[MT][NT] = {};
  MxFragment<4> b[4][NT];
  MxFragment<LBITS> a[4][MT];
  uint32_t bs[NT], as[MT], b_loaded[NT], a_loaded[MT];
  auto load_scales = [&](uint32_t first) {
    const uint32_t chunk = first + g < p.chunks ? first + g : p.chunks - 1;
#pragma unroll
    for (int j = 0; j < NT; ++j) b_loaded[j] = *(const uint32_t*)(rhs_scales[j] + chunk * rhs_scales_step);
#pragma unroll
    for (int i = 0; i < MT; ++i) a_loaded[i] = *(const uint32_t*)(lhs_scales[i] + chunk * lhs_scales_step);
  };
  auto take_scales = [&] {
#pragma unroll
    for (int j = 0; j < NT; ++j) bs[j] = scales_of_blocks(b_loaded[j], g);
#pragma unroll
    for (int i = 0; i < MT; ++i) as[i] = scales_of_blocks(a_loaded[i], g);
  };
  auto load = [&](auto number, uint32_t first) {
    constexpr int U = decltype(number)::value;
    const uint32_t chunk = first + U < p.chunks ? first + U : p.chunks - 1;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint8_t* from = rhs[j] + chunk * rhs_step;
      if constexpr (STREAM) {
        const mx_v4f32 v = __builtin_nontemporal_load((const mx_v4f32*)from);
        __builtin_memcpy(b[U][j].w, &v, 16);
      } else {
        __builtin_memcpy(b[U][j].w, __builtin_assume_aligned(from, 16), 16);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint8_t* from = lhs[i] + chunk * lhs_step;
      __builtin_memcpy(a[U][i].w, __builtin_assume_aligned(from, 16), 16);
      if constexpr (LBITS == 8) __builtin_memcpy(a[U][i].w + 4, __builtin_assume_aligned(from + 64, 16), 16);
    }
  };
  auto multiply = [&](auto number) {
    constexpr int U = decltype(number)::value;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (SPLIT) {
        MxFragment<8> high, low;
        mx_split(a[U][i], high, low);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[i][j] = mx_mfma_16<4, 8, U>(b[U][j], bs[j], high, as[i], acc[i][j]);
          acc[i][j] = mx_mfma_16<4, 8, U>(b[U][j], bs[j], low, as[i], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx_mfma_16<4, LBITS, U>(b[U][j], bs[j], a[U][i], as[i], acc[i][j]);
      }
    }
  };
  auto of_four = [](auto f) {
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
  };

  // Four chunks from `first` on; where they are not all there, the last four of K, of which those before `first` are skipped.
  const uint32_t fours = (p.chunks + 3) / 4;
  auto begin = [&](uint32_t four) {
    const uint32_t last = p.chunks > 4 ? p.chunks - 4 : 0;
    return 4 * four < last ? 4 * four : last;
  };
  if ((uint32_t)wave < fours) {
    uint32_t four = wave, first = begin(four);
    load_scales(first);
    of_four([&](auto u) { load(u, first); });
    for (; four + WAVES < fours; four += WAVES) {  // (all of four chunks)
      take_scales();
      first = begin(four + WAVES);
      load_scales(first);
      of_four([&](auto u) {
        multiply(u);
        load(u, first);
      });
    }
    take_scales();
    const uint32_t skip = 4 * four - first, end = p.chunks - first;
    of_four([&](auto u) {
      constexpr uint32_t U = decltype(u)::value;
      if (U >= skip && U < end) multiply(u);
    });
  }

#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) partial[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += WAVES) {
    mx_v4f32 v = partial[0][f][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += partial[w][f][lane];
    const uint32_t row = first_row + 16 * (f / NT) + r, col = first_col + 16 * (f % NT) + 4 * g;
    if (row < p.lhs.rows) mx_store_four(p, mx_out_row(p, row), col, v);
  }
}

template <int LBITS, int MT, int NT, int WAVES>
hipError_t launch(const MxProduct& p, hipStream_t stream) {
  const dim3 grid((p.rhs.rows + 16 * NT - 1) / (16 * NT), (p.lhs.rows + 16 * MT - 1) / (16 * MT));
  void* args[] = {const_cast<MxProduct*>(&p)};
  const bool stream_rhs = comes_from_hbm((int64_t)p.rhs.rows * p.chunks * 64);
  const bool split = LBITS == 8 && p.out_type == Float::kF32;
  const void* kernel = split ? (stream_rhs ? (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, true, LBITS == 8>
                                           : (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, false, LBITS == 8>)
                             : (stream_rhs ? (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, true, false>
                                           : (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, false, false>);
  return hipLaunchKernel(kernel, grid, dim3(64 * WAVES), args, 0, stream);
}

template <int LBITS>
hipError_t launch_of(const MxProduct& p, int shape, hipStream_t stream) {
  switch (shape) {  // kMxFewShapes
    case 0: return launch<LBITS, 1, 1, 8>(p, stream);
    case 1: return launch<LBITS, 1, 2, 8>(p, stream);
    case 2: return launch<LBITS, 1, 4, 8>(p, stream);
    case 3: return launch<LBITS, 2, 1, 8>(p, stream);
    case 4: return launch<LBITS, 2, 2, 8>(p, stream);
    case 5: return launch<LBITS, 2, 4, 8>(p, stream);
    case 6: if constexpr (LBITS == 4) return launch<4, 4, 4, 8>(p, stream);  // (8-bit codes do not fit the registers)
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_mx_few(const MxProduct& p, int lhs_bits, int shape, hipStream_t stream) {
  return lhs_bits == 4 ? launch_of<4>(p, shape, stream) : launch_of<8>(p, shape, stream);
}

}  // namespace uk
