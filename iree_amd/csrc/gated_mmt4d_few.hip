// Gated products of few rows: both weights are streamed from memory straight into registers, once, and K is split over the
// wavefronts of a workgroup.
#include <type_traits>

#include "gated_mmt4d.h"

namespace uk {
namespace {

constexpr int kWaves = 8;

extern __shared__ uint4 few_lds[];

// 64 x 16 bytes to LDS byte offset `lds` (of the wavefront) from `base` + the lane's `offset`, unseen by the compiler.
__device__ __forceinline__ void load_pieces(uint32_t lds, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// At most the last N loads of the wavefront are still under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A workgroup multiplies 16 * MT rows of the lhs with 16 * NT columns of gate and of up; its wavefronts take four chunks of 32 of K
// in turn, and add their sums through LDS in the order of their numbers. A chunk is loaded again as soon as it is multiplied. Rows
// beyond the last are read as the last one and not stored.
//
// STAGED: the lhs goes through LDS, a wavefront's own part of it, where a row's pieces are exchanged among themselves for the
// banks' sake. Straight into registers a load's neighbouring lanes have 16 rows, 16 cache lines; to LDS four neighbouring lanes
// have one row. (24 rows x 4096 x 4096 15.9 us staged, 17.5 not; 130 x 1000 x 512 4.3 and 5.3.)
//
// Memory bounds it where the weights are large (16 x 28672 x 8192 143 us, 940 MB at 6.6 TB/s), else the loads' way through a compute unit,
// 18 ns for each fragment of 16 rows and 32 values of K, and a start of two microseconds: 1 row x 1000 x 500 3 us. Four chunks under way
// are enough; eight to twelve took as long.
template <Float T, int MT, int NT, bool STREAM, bool STAGED>
__global__ __launch_bounds__(64 * kWaves) void gated_mmt4d_few_kernel(const GatedProduct p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t first_col = blockIdx.x * (16 * NT), first_row = blockIdx.y * (16 * MT);
  const uint32_t full = p.depth >> 5, rest = p.depth & 31;

  auto row_of = [&](const Operand16& o, int64_t stride0, uint32_t row) {
    row = row < o.rows ? row : o.rows - 1;
    const uint32_t panel = divide(row, o.tile_rows, o.tile_reciprocal);
    return (int64_t)panel * stride0 + (row - panel * o.tile_rows) * o.row_bytes + (g & 1) * o.piece1 + (g >> 1) * o.piece2;
  };
  const uint8_t *rhs[2 * NT], *lhs[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    rhs[j] = p.gate.data + row_of(p.gate, p.gate.stride0, first_col + 16 * j + r);
    rhs[NT + j] = p.up + row_of(p.gate, p.up_stride0, first_col + 16 * j + r);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) lhs[i] = p.lhs.data + row_of(p.lhs, p.lhs.stride0, first_row + 16 * i + r);
  const int64_t rhs_step = 64 * (int64_t)p.gate.tile_rows, lhs_step = 64 * (int64_t)p.lhs.tile_rows;

  // Staged: load n of a chunk has rows 16 n + lane / 4; a row's piece c lies at c ^ exchanged(row).
  auto exchanged = [](uint32_t row) { return ((row >> 2) & 3) ^ (row & 2); };
  constexpr int CHUNK = MT * 1024;
  const uint32_t first_panel = divide(first_row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
  const uint8_t* const lhs_base = p.lhs.data + (int64_t)first_panel * p.lhs.stride0;
  uint32_t lhs_from[STAGED ? MT : 1];
  if constexpr (STAGED) {
#pragma unroll
    for (int n = 0; n < MT; ++n) {
      const uint32_t at = n * 16 + lane / 4, piece = (lane % 4) ^ exchanged(at);
      const uint32_t row = first_row + at < p.lhs.rows ? first_row + at : p.lhs.rows - 1;
      const uint32_t panel = divide(row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
      lhs_from[n] = (uint32_t)((panel - first_panel) * p.lhs.stride0) + (row - panel * p.lhs.tile_rows) * p.lhs.row_bytes +
                    (piece & 1) * p.lhs.piece1 + (piece >> 1) * p.lhs.piece2;
    }
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)few_lds + wave * (4 * CHUNK);
  const uint8_t* const staged = (const uint8_t*)few_lds + wave * (4 * CHUNK) + r * 64 + 16 * (g ^ exchanged(r));

  p16_v4f32 acc[MT][2 * NT] = {};
  uint4 a[STAGED ? 1 : 4][MT], b[4][2 * NT];
  auto load = [&](int u, uint32_t first) {
    const uint32_t chunk = first + u < full ? first + u : full - 1;
    if constexpr (STAGED) {
#pragma unroll
      for (int n = 0; n < MT; ++n) load_pieces(lds0 + u * CHUNK + n * 1024, lhs_from[n], lhs_base + chunk * lhs_step);
    }
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) {
      const uint8_t* from = rhs[j] + chunk * rhs_step;
      if constexpr (STREAM) {
        const p16_v4f32 v = __builtin_nontemporal_load((const p16_v4f32*)from);
        b[u][j] = __builtin_bit_cast(uint4, v);
      } else {
        b[u][j] = *(const uint4*)from;
      }
    }
    if constexpr (!STAGED) {
#pragma unroll
      for (int i = 0; i < MT; ++i) a[u][i] = *(const uint4*)(lhs[i] + chunk * lhs_step);
    }
  };
  auto multiply = [&](int u) {
    if constexpr (STAGED) {
#pragma unroll
      for (int i = 0; i < MT; ++i) a[0][i] = *(const uint4*)(staged + u * CHUNK + i * 1024);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) acc[i][j] = mfma16_16<T>(b[u][j], a[STAGED ? 0 : u][i], acc[i][j]);
    // (What has been read from LDS has been read before its place is loaded again.)
    if constexpr (STAGED) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  // Four chunks from `first` on; where they are not all there, the last four of K, of which those before `first` are skipped.
  const uint32_t fours = (full + 3) / 4;
  auto begin = [&](uint32_t four) {
    const uint32_t last = full > 4 ? full - 4 : 0;
    return 4 * four < last ? 4 * four : last;
  };
  if ((uint32_t)wave < fours) {
    uint32_t four = wave, first = begin(four);
#pragma unroll
    for (int u = 0; u < 4; ++u) load(u, first);
    for (; four + kWaves < fours; four += kWaves) {  // (all of four chunks)
      first = begin(four + kWaves);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        // (Behind a chunk's loads come three chunks', and of each only those to LDS are counted on: the compiler may leave out or
        // join its own.)
        if constexpr (STAGED) wait_loads<3 * MT>();
        multiply(u);
        load(u, first);
      }
    }
    const uint32_t skip = 4 * four - first, end = full - first;
    if constexpr (STAGED) wait_loads<0>();
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if ((uint32_t)u >= skip && (uint32_t)u < end) multiply(u);
  }
  // What K has behind its last whole chunk, zeros behind it.
  if (rest != 0 && wave == (int)(fours % kWaves)) {
    const int exist = (int)rest - 8 * g;
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) b[0][j] = last_piece(rhs[j] + full * rhs_step, exist);
#pragma unroll
    for (int i = 0; i < MT; ++i) a[0][i] = last_piece(lhs[i] + full * lhs_step, exist);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 2 * NT; ++j) acc[i][j] = mfma16_16<T>(b[0][j], a[0][i], acc[i][j]);
  }

  p16_v4f32* const partial = (p16_v4f32*)few_lds;  // [kWaves][MT * 2 NT][64]
  if constexpr (STAGED) __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 2 * NT; ++j) partial[(wave * (MT * 2 * NT) + i * 2 * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += kWaves) {
    const int i = f / NT, j = f % NT;
    const p16_v4f32* const of = partial + (i * 2 * NT + j) * 64 + lane;
    p16_v4f32 gate = of[0], up = of[NT * 64];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      gate += of[w * (MT * 2 * NT) * 64];
      up += of[(w * (MT * 2 * NT) + NT) * 64];
    }
    const uint32_t row = first_row + 16 * i + r, col = first_col + 16 * j + 4 * g;
    if (row < p.lhs.rows && col < p.gate.rows) p.results.store_four<T>(gate, up, row, col, p.gate.rows);
  }
}

template <Float T, int MT, int NT, bool STAGED>
hipError_t launch(const GatedProduct& p, hipStream_t stream) {
  const dim3 grid((p.gate.rows + 16 * NT - 1) / (16 * NT), (p.lhs.rows + 16 * MT - 1) / (16 * MT));
  void* args[] = {const_cast<GatedProduct*>(&p)};
  const void* kernel = comes_from_hbm(4 * (int64_t)p.gate.rows * p.depth) ? (const void*)gated_mmt4d_few_kernel<T, MT, NT, true, STAGED>
                                                                          : (const void*)gated_mmt4d_few_kernel<T, MT, NT, false, STAGED>;
  constexpr int SUMS = kWaves * MT * 2 * NT * 1024, LHS = STAGED ? kWaves * 4 * MT * 1024 : 0, LDS = SUMS > LHS ? SUMS : LHS;
  static_assert(LDS <= 160 * 1024, "LDS");
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return e;
  }
  return hipLaunchKernel(kernel, grid, dim3(64 * kWaves), args, LDS, stream);
}

template <Float T>
hipError_t launch_of(const GatedProduct& p, int shape, hipStream_t stream) {
  switch (shape) {  // kGatedFewShapes
    case 0: return launch<T, 1, 1, false>(p, stream);
    case 1: return launch<T, 1, 2, false>(p, stream);
    case 2: return launch<T, 1, 1, true>(p, stream);
    case 3: return launch<T, 2, 1, true>(p, stream);
    case 4: return launch<T, 2, 2, true>(p, stream);
    case 5: return launch<T, 4, 1, true>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_gated_few(const GatedProduct& p, Float type, int shape, hipStream_t stream) {
  return type == Float::kF16 ? launch_of<Float::kF16>(p, shape, stream) : launch_of<Float::kBf16>(p, shape, stream);
}

}  // namespace uk
