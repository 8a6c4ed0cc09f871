// Microscaled products of few rows: the rhs (the weights) is streamed from memory straight into registers, once, and K is
// split over the wavefronts of a workgroup.
#include <type_traits>

#include "mx_mmt4d.h"

namespace uk {
namespace {

// A workgroup multiplies 16 * MT rows of the lhs with 16 * NT of the rhs; its wavefronts take chunks of 128 of K in turn, AHEAD of
// them in flight each, and add their sums through LDS in the order of their numbers. Rows beyond the last are read as the
// last one and not stored.
template <int LBITS, int MT, int NT, int WAVES, int AHEAD, bool STREAM, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES) void mx_mmt4d_few_kernel(const MxProduct p) {
  __shared__ mx_v4f32 partial[WAVES][MT * NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const uint32_t first_col = blockIdx.x * (16 * NT), first_row = blockIdx.y * (16 * MT);

  const uint8_t *rhs[NT], *rhs_scales[NT], *lhs[MT], *lhs_scales[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint32_t col = first_col + 16 * j + r, row = col < p.rhs.rows ? col : p.rhs.rows - 1;
    rhs[j] = p.rhs.codes + mx_row_codes<4>(p.rhs, row) + 16 * g;
    rhs_scales[j] = p.rhs.scales + mx_row_scales(p.rhs, row) + g;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const uint32_t at = first_row + 16 * i + r, row = at < p.lhs.rows ? at : p.lhs.rows - 1;
    lhs[i] = p.lhs.codes + mx_row_codes<LBITS>(p.lhs, row) + 16 * g;
    lhs_scales[i] = p.lhs.scales + mx_row_scales(p.lhs, row) + g;
  }
  const int64_t rhs_step = 64 * (int64_t)p.rhs.tile_rows, rhs_scales_step = 4 * (int64_t)p.rhs.tile_rows;
  const int64_t lhs_step = 16 * LBITS * (int64_t)p.lhs.tile_rows, lhs_scales_step = 4 * (int64_t)p.lhs.tile_rows;

  mx_v4f32 acc[MT][NT] = {};
  MxFragment<4> b[AHEAD][NT];
  MxFragment<LBITS> a[AHEAD][MT];
  uint32_t bs[AHEAD][NT], as[AHEAD][MT];
  auto load = [&](int u, uint32_t chunk) {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint8_t* from = rhs[j] + chunk * rhs_step;
      if constexpr (STREAM) {
        const mx_v4f32 v = __builtin_nontemporal_load((const mx_v4f32*)from);
        __builtin_memcpy(b[u][j].w, &v, 16);
      } else {
        __builtin_memcpy(b[u][j].w, __builtin_assume_aligned(from, 16), 16);
      }
      bs[u][j] = rhs_scales[j][chunk * rhs_scales_step];
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const uint8_t* from = lhs[i] + chunk * lhs_step;
      __builtin_memcpy(a[u][i].w, __builtin_assume_aligned(from, 16), 16);
      if constexpr (LBITS == 8) __builtin_memcpy(a[u][i].w + 4, __builtin_assume_aligned(from + 64, 16), 16);
      as[u][i] = lhs_scales[i][chunk * lhs_scales_step];
    }
  };
  auto multiply = [&](int u) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (SPLIT) {
        MxFragment<8> high, low;
        mx_split(a[u][i], high, low);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[i][j] = mx_mfma_16<4, 8>(b[u][j], bs[u][j], high, as[u][i], acc[i][j]);
          acc[i][j] = mx_mfma_16<4, 8>(b[u][j], bs[u][j], low, as[u][i], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx_mfma_16<4, LBITS>(b[u][j], bs[u][j], a[u][i], as[u][i], acc[i][j]);
      }
    }
  };

  const uint32_t mine = p.chunks > (uint32_t)wave ? (p.chunks - wave + WAVES - 1) / WAVES : 0;  // wave, wave + WAVES, ..
  const uint32_t batches = mine / AHEAD;
  uint32_t c = wave;
  for (uint32_t n = 0; n < batches; ++n, c += AHEAD * WAVES) {
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) load(u, c + u * WAVES);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) multiply(u);
  }
  const uint32_t rest = mine - batches * AHEAD;
#pragma unroll
  for (int u = 0; u < AHEAD - 1; ++u)
    if (u < (int)rest) load(u, c + u * WAVES);
#pragma unroll
  for (int u = 0; u < AHEAD - 1; ++u)
    if (u < (int)rest) multiply(u);

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

template <int LBITS, int MT, int NT, int WAVES, int AHEAD>
hipError_t launch(const MxProduct& p, hipStream_t stream) {
  const dim3 grid((p.rhs.rows + 16 * NT - 1) / (16 * NT), (p.lhs.rows + 16 * MT - 1) / (16 * MT));
  void* args[] = {const_cast<MxProduct*>(&p)};
  const bool stream_rhs = comes_from_hbm((int64_t)p.rhs.rows * p.chunks * 64);
  const bool split = LBITS == 8 && p.out_type == Float::kF32;
  const void* kernel = split ? (stream_rhs ? (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, AHEAD, true, LBITS == 8>
                                           : (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, AHEAD, false, LBITS == 8>)
                             : (stream_rhs ? (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, AHEAD, true, false>
                                           : (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, WAVES, AHEAD, false, false>);
  return hipLaunchKernel(kernel, grid, dim3(64 * WAVES), args, 0, stream);
}

template <int LBITS>
hipError_t launch_of(const MxProduct& p, hipStream_t stream) {
  if (p.lhs.rows <= 16) return launch<LBITS, 1, 1, 4, 4>(p, stream);
  if (p.lhs.rows <= 32) return launch<LBITS, 2, 1, 4, 4>(p, stream);
  return launch<LBITS, 4, 1, 4, 2>(p, stream);
}

}  // namespace

hipError_t launch_mx_few(const MxProduct& p, int lhs_bits, hipStream_t stream, const char** name) {
  *name = "mx_mmt4d_few";
  return lhs_bits == 4 ? launch_of<4>(p, stream) : launch_of<8>(p, stream);
}

}  // namespace uk
