#include "gated_backward_block.h"

namespace uk {
hipError_t launch_weight_grad_bf16(const WeightGradProduct& p, int tile, hipStream_t stream) {
  return launch_grad_tile<Float::kBf16>(as_block_product(p), tile, stream);
}
hipError_t launch_both_grads_bf16(const LhsGradProduct& lhs, const WeightGradProduct& weights, hipStream_t stream) {
  return launch_both_grads<Float::kBf16>(lhs, weights, stream);
}
}  // namespace uk
