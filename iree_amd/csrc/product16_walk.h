// Which chunk of K a workgroup of the block kernels (product16_block.h) loads next. Plain C++, so that it can be walked on the CPU.
#ifndef IREE_AMD_CSRC_PRODUCT16_WALK_H_
#define IREE_AMD_CSRC_PRODUCT16_WALK_H_

#include <stdint.h>

#ifdef __HIPCC__
#define UK_WALK __host__ __device__ __forceinline__
#else
#define UK_WALK inline
#endif

namespace uk {

// Whole chunks at .. end - 1, numbered through both halves of a K in two halves of `full` each (of one half: full = end). Behind the
// last one it is the last that is loaded again.
struct ChunkWalk {
  uint32_t at, end, full;
  enum Step { kStay, kNext, kSecondHalf };
  // From the chunk that has been loaded to the next.
  UK_WALK Step next() {
    if (at + 1 >= end) return kStay;
    ++at;
    return at == full ? kSecondHalf : kNext;
  }
};

// The whole chunks of split `split` of `splits`, of `chunks` >= splits in all: at least one.
UK_WALK uint32_t first_of_split(uint32_t chunks, uint32_t split, uint32_t splits) {
  return (uint32_t)((uint64_t)chunks * split / splits);
}

}  // namespace uk

#endif  // IREE_AMD_CSRC_PRODUCT16_WALK_H_
