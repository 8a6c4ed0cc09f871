// The block kernels of the gated products' gradients, one translation unit for each type.
#ifndef IREE_AMD_CSRC_GATED_BACKWARD_BLOCK_H_
#define IREE_AMD_CSRC_GATED_BACKWARD_BLOCK_H_

#include "gated_backward.h"
#include "product16_block.h"

namespace uk {
namespace {

// What bounds them: as the gated products. 4096 x 11008 x 4096, lhs_grad 600 us, 1.23 PFLOP/s, in 256x256 tiles (256x128 820, 128x256 770,
// 128x128 900), the weights' gradients 630, 1.17, in 128x256, two to a compute unit (256x256 637, 256x128 690, 128x128 750).
template <Float T, typename P>
hipError_t launch_grad_tile(const P& p, int tile, hipStream_t stream) {
  switch (tile) {  // kGradTiles
    case 0: return launch_block_tile<T, 4, 4, 4>(p, stream);
    case 1: return launch_block_tile<T, 4, 2, 4>(p, stream);
    case 2: return launch_block_tile<T, 2, 4, 3>(p, stream);
    case 3: return launch_block_tile<T, 2, 2, 5>(p, stream);
    case 4: return launch_block_tile<T, 2, 1, 6>(p, stream);
    case 5: return launch_block_tile<T, 1, 2, 6>(p, stream);
    case 6: return launch_block_tile<T, 1, 1, 8>(p, stream);
  }
  return hipErrorInvalidValue;
}

template <Float T>
hipError_t launch_lhs_grad(const LhsGradProduct& g, int tile, hipStream_t stream) {
  BlockProduct<LhsGrad, Operand16, Strided16> p;
  p.lhs = g.grads;
  p.rhs = g.gate;
  p.second = g.up;
  p.second_stride0 = g.up_stride0;
  p.lhs_second = g.lhs_second;
  p.depth = g.depth;
  (GradResults&)p.epilogue = g.results;
  return launch_grad_tile<T>(p, tile, stream);
}
template <Float T>
hipError_t launch_weight_grad(const WeightGradProduct& g, int tile, hipStream_t stream) {
  BlockProduct<WeightGrads, Strided16, Strided16> p;
  p.lhs = g.grads;
  p.rhs = g.lhs;
  p.second = nullptr;
  p.second_stride0 = g.lhs.stride0;
  p.lhs_second = g.lhs_second;
  p.depth = g.depth;
  (GradResults&)p.epilogue = g.results;
  return launch_grad_tile<T>(p, tile, stream);
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_BACKWARD_BLOCK_H_
