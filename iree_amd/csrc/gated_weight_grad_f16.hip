#include "gated_backward_block.h"

namespace uk {
hipError_t launch_weight_grad_f16(const WeightGradProduct& p, int tile, hipStream_t stream) {
  return launch_grad_tile<Float::kF16>(as_block_product(p), tile, stream);
}
hipError_t launch_both_grads_f16(const LhsGradProduct& lhs, const WeightGradProduct& weights, hipStream_t stream) {
  return launch_both_grads<Float::kF16>(lhs, weights, stream);
}
}  // namespace uk
