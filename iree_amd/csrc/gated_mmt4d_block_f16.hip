#include "gated_mmt4d_block.h"

namespace uk {
hipError_t launch_gated_block_f16(const GatedProduct& p, int tile, hipStream_t stream) { return launch_gated_block<Float::kF16>(p, tile, stream); }
}  // namespace uk
