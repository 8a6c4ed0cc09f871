#include "gated_backward_block.h"

namespace uk {
hipError_t launch_lhs_grad_f16(const LhsGradProduct& p, int tile, hipStream_t stream) { return launch_lhs_grad<Float::kF16>(p, tile, stream); }
}  // namespace uk
