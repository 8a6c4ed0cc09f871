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

inline BlockProduct<LhsGrad, Operand16, Strided16> as_block_product(const LhsGradProduct& g) {
  BlockProduct<LhsGrad, Operand16, Strided16> p;
  p.lhs = g.grads;
  p.rhs = g.gate;
  p.second = g.up;
  p.second_stride0 = g.up_stride0;
  p.lhs_second = g.lhs_second;
  p.depth = g.depth;
  (GradResults&)p.epilogue = g.results;
  return p;
}
inline BlockProduct<WeightGrads, Strided16, Strided16> as_block_product(const WeightGradProduct& g) {
  BlockProduct<WeightGrads, Strided16, Strided16> p;
  p.lhs = g.grads;
  p.rhs = g.lhs;
  p.second = nullptr;
  p.second_stride0 = g.lhs.stride0;
  p.lhs_second = g.lhs_second;
  p.depth = g.depth;
  (GradResults&)p.epilogue = g.results;
  return p;
}

// Both products' workgroups in one launch, 64x64 tiles of each: small gradients, which launches and starts bound.
struct BothGrads {
  BlockProduct<LhsGrad, Operand16, Strided16> lhs;
  BlockProduct<WeightGrads, Strided16, Strided16> weights;
  uint32_t of_lhs;  // workgroups, a multiple of 8
};
template <Float T>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void both_grads_kernel(const BothGrads p) {
  if (blockIdx.x < p.of_lhs) product16_block<T, 1, 1, 8, false>(p.lhs, blockIdx.x);
  else product16_block<T, 1, 1, 8, false>(p.weights, blockIdx.x - p.of_lhs);
}
template <Float T>
hipError_t launch_both_grads(const LhsGradProduct& lhs, const WeightGradProduct& weights, hipStream_t stream) {
  constexpr int LDS = block_lds_bytes(1, 1, 8);
  static_assert(LDS <= 64 * 1024, "LDS");
  BothGrads p{as_block_product(lhs), as_block_product(weights), 0};
  p.of_lhs = lay_out_tiles<1, 1>(p.lhs);
  const unsigned of_weights = lay_out_tiles<1, 1>(p.weights);
  return launch_kernel(both_grads_kernel<T>, p.of_lhs + of_weights, 256, LDS, stream, p);
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_BACKWARD_BLOCK_H_
