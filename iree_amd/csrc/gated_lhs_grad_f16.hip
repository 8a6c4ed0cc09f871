#include "gated_backward_block.h"

namespace uk {
hipError_t launch_lhs_grad_f16(const LhsGradProduct& p, int tile, hipStream_t stream) {
  return launch_grad_tile<Float::kF16>(as_block_product(p), tile, stream);
}
}  // namespace uk
