#include "gated_backward_block.h"

namespace uk {
hipError_t launch_weight_grad_bf16(const WeightGradProduct& p, int tile, hipStream_t stream) { return launch_weight_grad<Float::kBf16>(p, tile, stream); }
}  // namespace uk
