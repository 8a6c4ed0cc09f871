// Block kernels of microscaled products: E2M1 times E2M1.
#include "mx_mmt4d_block.h"

namespace uk {
hipError_t launch_mx_block_e2m1(const MxProduct& p, int tile, hipStream_t stream) { return launch_block<4>(p, tile, stream); }
}  // namespace uk
