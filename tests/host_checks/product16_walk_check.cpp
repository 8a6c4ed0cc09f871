// Which chunks the block kernels of 16-bit products load, walked for every split of K: each whole chunk once, none that isn't there.
#include <cstdio>
#include <vector>

#include "product16_walk.h"

using uk::ChunkWalk;
using uk::first_of_split;

static long walks, wrong;

static void expect(bool ok, uint32_t full, uint32_t halves, uint32_t splits, uint32_t split) {
  if (!ok && wrong++ < 10) printf("%u chunks of %u halves, split %u of %u\n", full, halves, split, splits);
}

// The pointers as the kernel moves them: a half and a chunk of it. Loads go on behind a split's last chunk.
static void walk(uint32_t full, uint32_t halves, uint32_t split, uint32_t splits, std::vector<int>* loaded) {
  ChunkWalk w = {0, full, full};
  if (halves == 2) {
    w.at = first_of_split(2 * full, split, splits);
    w.end = first_of_split(2 * full, split + 1, splits);
  }
  const uint32_t begin = w.at, end = w.end;
  expect(full == 0 || begin < end, full, halves, splits, split);
  bool second = w.at != 0 && w.at >= full;
  int64_t at = second ? (int64_t)w.at - full : w.at;
  for (uint32_t load = 0; load < end - begin + 12; ++load) {
    ++walks;
    if (full == 0) {
      expect(at == 0 && !second, full, halves, splits, split);  // (what is there of a chunk)
    } else {
      const uint32_t number = begin + load < end ? begin + load : end - 1;
      expect(at >= 0 && at < full && (second ? full : 0) + at == number, full, halves, splits, split);
      if (begin + load < end) ++(*loaded)[number];
    }
    switch (w.next()) {
      case ChunkWalk::kSecondHalf:
        second = true;
        at = 0;
        break;
      case ChunkWalk::kNext: ++at; break;
      case ChunkWalk::kStay: break;
    }
  }
}

int main() {
  for (uint32_t full = 0; full < 130; ++full)
    for (uint32_t halves = 1; halves <= 2; ++halves)
      for (uint32_t splits = 1; splits <= (halves == 1 ? 1u : 32u); ++splits) {
        if (splits > 1 && splits > 2 * full) break;
        std::vector<int> loaded(halves * full, 0);
        for (uint32_t split = 0; split < splits; ++split) walk(full, halves, split, splits, &loaded);
        for (int n : loaded) expect(n == 1, full, halves, splits, splits);
      }
  printf("%ld loads, %ld wrong\n", walks, wrong);
  return wrong != 0;
}
