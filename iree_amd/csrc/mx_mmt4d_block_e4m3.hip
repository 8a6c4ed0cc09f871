// Block kernels of microscaled products: E4M3 times E2M1.
#include "mx_mmt4d_block.h"

namespace uk {
hipError_t launch_mx_block_e4m3(const MxProduct& p, int tile, hipStream_t stream) { return launch_block<8>(p, tile, stream); }
}  // namespace uk
