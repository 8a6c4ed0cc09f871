#include "gated_backward_block.h"

namespace uk {
hipError_t launch_weight_grad_f16(const WeightGradProduct& p, int tile, hipStream_t stream) { return launch_weight_grad<Float::kF16>(p, tile, stream); }
}  // namespace uk
