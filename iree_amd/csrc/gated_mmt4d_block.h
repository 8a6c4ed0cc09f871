// The block kernels of gated products, one translation unit for each type.
#ifndef IREE_AMD_CSRC_GATED_MMT4D_BLOCK_H_
#define IREE_AMD_CSRC_GATED_MMT4D_BLOCK_H_

#include "gated_mmt4d.h"
#include "product16_lines.h"

namespace uk {
namespace {

template <Float T>
hipError_t launch_gated_block(const GatedProduct& g, int tile, hipStream_t stream) {
  BlockProduct<GatedResults, Operand16, Operand16> p;
  p.lhs = g.lhs;
  p.rhs = g.gate;
  p.second = g.up;
  p.second_stride0 = g.up_stride0;
  p.lhs_second = 0;
  p.depth = g.depth;
  p.epilogue = g.results;
  // Weights that a tile or two of rows read once go past the caches where the layer's three matrices (the third is as large as one of
  // these) do not fit them, 256 MiB, and so are gone when the next token comes. 64 rows x 28672 x 8192, 940 MB, 165 -> 148 us in 64x128
  // tiles; where other calls have filled the caches in between, 40 x 11008 x 4096 (180 MB) 38.1 -> 35.1, 64 x 14336 x 4096 47.1 -> 43.4 and
  // 128 x 11008 x 4096 53.2 -> 50.2. The same call made again at once finds its weights there: 29 -> 35, 36 -> 43 and 33 -> 49.
  const bool stream_rhs = g.lhs.rows <= 128 && 6 * (int64_t)g.gate.rows * g.depth > (256ll << 20);
  // Row-major rows that are whole cache lines are loaded by whole lines in the four largest tiles, one workgroup of which fits a compute
  // unit, and in two others that still fit it twice with the longer ring: 512 x 11008 x 4096 in 256x96 tiles 102 -> 90 us,
  // 4096 x 11008 x 4096 in 256x128 ones 678 -> 654, 300 x 11008 x 4096 in 192x96 75.7 -> 72.4, 128 x 11008 x 4096 in 64x96 50.4 -> 46.6,
  // 400 x 4096 x 4096 in 128x64 38.6 -> 37.3 (weights from memory, clocks settled, both in turn). 64x64 tiles won 43.8 -> 40.2 for 64 rows but lost 35.2 -> 36.2 for 40 and 23.5 -> 24.3
  // for 77, 64x32 ones gained nothing where they are taken. The other three would fit once and not twice, and so take it where there is
  // a tile at most for a compute unit: 256 x 11008 x 4096 in 230 of 128x96 70.3 -> 61.5, 200 x 14336 x 4096 in 224 of 128x128
  // 77.6 -> 70.2, 1024 x 4096 x 4096 in 256 67.0 -> 65.2, 400 x 4096 x 4096 in 224 of 64x128 38.6 -> 35.9; more tiles lost, 700 x 5632 x
  // 2048 in 264 of 128x128 50.0 -> 56.7.
  const GatedTile& shape = kGatedTiles[tile];
  const bool one_each = ((int64_t)g.lhs.rows + shape.rows - 1) / shape.rows * (((int64_t)g.gate.rows + shape.cols - 1) / shape.cols) <= 256;
  if (whole_lines(g.lhs, g.depth)) {
    switch (tile) {
      case 0: return launch_lines_tile<T, 4, 4>(p, stream);
      case 1: return launch_lines_tile<T, 4, 3>(p, stream);
      case 2: return launch_lines_tile<T, 3, 3>(p, stream);
      case 3: return launch_lines_tile<T, 3, 4>(p, stream);
      case 4:
        if (!one_each) break;
        return launch_lines_tile<T, 2, 4>(p, stream);
      case 5:
        if (!one_each) break;
        return launch_lines_tile<T, 2, 3>(p, stream);
      case 6: return stream_rhs ? launch_lines_tile<T, 2, 2, true>(p, stream) : launch_lines_tile<T, 2, 2>(p, stream);
      case 7:
        if (!one_each || stream_rhs) break;  // (no call takes this tile for a compute unit's one and such weights)
        return launch_lines_tile<T, 1, 4>(p, stream);
      case 8: return stream_rhs ? launch_lines_tile<T, 1, 3, true>(p, stream) : launch_lines_tile<T, 1, 3>(p, stream);
    }
  }
  switch (tile) {  // kGatedTiles
    case 0: return launch_block_tile<T, 4, 4, 4>(p, stream);
    case 1: return launch_block_tile<T, 4, 3, 4>(p, stream);
    case 2: return launch_block_tile<T, 3, 3, 4>(p, stream);
    case 3: return launch_block_tile<T, 3, 4, 4>(p, stream);
    case 4: return launch_block_tile<T, 2, 4, 3>(p, stream);
    case 5: return launch_block_tile<T, 2, 3, 4>(p, stream);
    case 6: return stream_rhs ? launch_block_tile<T, 2, 2, 5, true>(p, stream) : launch_block_tile<T, 2, 2, 5>(p, stream);
    case 7: return stream_rhs ? launch_block_tile<T, 1, 4, 4, true>(p, stream) : launch_block_tile<T, 1, 4, 4>(p, stream);
    case 8: return stream_rhs ? launch_block_tile<T, 1, 3, 5, true>(p, stream) : launch_block_tile<T, 1, 3, 5>(p, stream);
    case 9: return stream_rhs ? launch_block_tile<T, 1, 2, 6, true>(p, stream) : launch_block_tile<T, 1, 2, 6>(p, stream);
    case 10: return stream_rhs ? launch_block_tile<T, 1, 1, 8, true>(p, stream) : launch_block_tile<T, 1, 1, 8>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_MMT4D_BLOCK_H_
