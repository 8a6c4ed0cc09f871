// The block kernel of 16-bit products (product16_block.h) for a row-major lhs whose rows are whole cache lines.
//
// A chunk of 32 values is half a line of a row, and each half is a request of its own. Here a load takes 128 bytes of eight rows, two
// chunks: the lhs lies in LDS as a ring of three pairs of chunks beside a ring of four chunks of the rhs. In every chunk's time a
// wavefront loads a chunk of the rhs, three ahead, and half of its rows of a pair, whose first half is on its way four chunks ahead of
// use. So the loop is that of four stages: as many loads a chunk, the same waits. K is a multiple of 64.
//
// What it saves is the L2's requests: 512 x 11008 x 4096, gate and up from memory, makes 11.0 million by half lines, 7.0 with the rows in
// tiles, where a chunk's pieces lie together, and takes 102, 87 and, by whole lines, 90 us (1.03 PFLOP/s, 2.2 TB/s) once the clocks have
// settled; in the first millisecond under load 85. 4096 x 11008 x 4096 takes 611 to 654 us from card to card, 1.13 to 1.21 PFLOP/s, which the
// board's power bounds.
#ifndef IREE_AMD_CSRC_PRODUCT16_LINES_H_
#define IREE_AMD_CSRC_PRODUCT16_LINES_H_

#include "product16_block.h"

namespace uk {
namespace {

constexpr int lines_lds_bytes(int am, int bn) { return 3 * 64 * am * 128 + 4 * 64 * bn * 64; }

template <Float T, int AM, int BN, bool STREAM, typename E>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(lines_lds_bytes(AM, BN) <= 80 * 1024 ? 2 : 1, 2)))
void product16_lines_kernel(const BlockProduct<E, Operand16, Operand16> p) {
  static_assert(E::kPaired && !E::kInTurn && !E::kCopies, "an epilogue of a pair");
  constexpr int ROWS = 64 * AM, COLS = 64 * BN, RESULTS = COLS / 2;
  constexpr int PAIR = ROWS * 128, B_STAGE = COLS * 64, B_AT = 3 * PAIR;
  constexpr int A_LOADS = AM, B_LOADS = BN, LOADS = A_LOADS + B_LOADS;  // of a wavefront, for a chunk

  const uint32_t tiles = p.tile_rows * p.tile_cols, per_xcd = (tiles + 7) >> 3;
  const uint32_t linear = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per_xcd || linear >= tiles) return;
  int tile_row, tile_col;
  tile_of_number(linear, p.tile_rows, p.tile_cols, p.band_reciprocal, &tile_row, &tile_col);
  const uint32_t first_row = (uint32_t)tile_row * ROWS, first_col = (uint32_t)tile_col * RESULTS;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;

  // Loads. Of the lhs: row lane / 8 of eight, of its eight pieces lane % 8 ^ that row. Rows behind the last are read as the last.
  const uint8_t* lhs = uniform_pointer(p.lhs.data + (int64_t)first_row * p.lhs.stride0);
  uint32_t a_from[2][A_LOADS], b_from[B_LOADS];
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < A_LOADS; ++i) {
      const uint32_t in_tile = 8 * ((2 * wave + half) * A_LOADS + i) + lane / 8;
      const uint32_t row = first_row + in_tile < p.lhs.rows ? in_tile : p.lhs.rows - 1 - first_row;
      a_from[half][i] = row * (uint32_t)p.lhs.stride0 + 16 * ((lane ^ (lane >> 3)) & 7);
    }
  auto is_second = [&](int i) { return ((wave * B_LOADS + i) & 1) != 0; };
  const uint8_t* const rhs_first = first_of<BN>(p.rhs, p.rhs.data, p.rhs.stride0, first_col);
  const uint8_t* const rhs_second = first_of<BN>(p.rhs, p.second, p.second_stride0, first_col);
#pragma unroll
  for (int i = 0; i < B_LOADS; ++i) {
    const uint32_t number = wave * B_LOADS + i;
    b_from[i] = offset_of<BN>(p.rhs, is_second(i) ? p.second_stride0 : p.rhs.stride0, first_col, number, number / 2, lane, p.depth);
  }
  const uint8_t *rhs_even = is_second(0) ? rhs_second : rhs_first, *rhs_odd = is_second(1) ? rhs_second : rhs_first;
  const int64_t rhs_step = chunk_step(p.rhs);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)ring;
  uint32_t a_to = lds0;                                               // of the pair that is loaded
  uint32_t freed = lds0 + B_AT;                                       // of the chunk of the rhs that is
  // Load number I: half `half` of the rows of a pair of the lhs, then a chunk of the rhs.
  auto load = [&](auto half, auto number) {
    constexpr int H = decltype(half)::value, I = decltype(number)::value;
    if constexpr (I < A_LOADS) load_pieces(a_to + ((2 * wave + H) * A_LOADS + I) * 1024, a_from[H][I], lhs);
    else load_pieces<STREAM>(freed + (wave * B_LOADS + I - A_LOADS) * 1024, b_from[I - A_LOADS], (I - A_LOADS) % 2 ? rhs_odd : rhs_even);
  };
  const uint32_t chunks = p.depth >> 5;  // even
  uint32_t pairs_left = chunks / 2 - 1, chunks_left = chunks - 1;  // behind those that are loaded; the last ones again where there are none
  auto next_pair = [&] {
    lhs += pairs_left != 0 ? 128 : 0;
    pairs_left -= pairs_left != 0 ? 1 : 0;
    a_to = a_to + PAIR == lds0 + B_AT ? lds0 : a_to + PAIR;
  };
  auto next_chunk = [&] {
    const bool more = chunks_left != 0;
    rhs_even += more ? rhs_step : 0;
    if constexpr (BN > 1) rhs_odd += more ? rhs_step : 0;
    else rhs_odd = rhs_even;
    chunks_left -= more ? 1 : 0;
  };

  // Reads: of the lhs row r's piece 4 half + 2 step + g lies at that ^ r % 8.
  const uint8_t* const lds = (const uint8_t*)ring;
  const uint32_t r = lane & 31, g = lane >> 5;
  const uint32_t a_read = (wave_m * 32 * AM + r) * 128 + 16 * (g ^ (r & 7)), b_read = read_at<BN>(p.rhs, wave_n, lane);
  uint4 a[2][AM], b[2][BN];
  constexpr int READS = AM + BN;
  auto read = [&](const uint8_t* of_a, const uint8_t* of_b, auto half, auto step, auto number) {
    constexpr int H = decltype(half)::value, S = decltype(step)::value, I = decltype(number)::value;
    if constexpr (I < AM) a[S][I] = *(const uint4*)(of_a + I * 4096 + (a_read ^ (64 * H | 32 * S)));
    else read_piece<BN, I - AM, S, 0>(p.rhs, of_b, b_read, b[S][I - AM]);
  };
  p16_v16f32 acc[AM][BN] = {};
  constexpr int MFMAS = AM * BN;
  auto multiply = [&](auto step, auto read_one, auto load_count, auto load_one) {
    constexpr int S = decltype(step)::value, L = decltype(load_count)::value;
    each_of<MFMAS>([&](auto m) {
      constexpr int N = decltype(m)::value, I = N / BN, J = N % BN;
      acc[I][J] = mfma16_32<T>(b[S][J], a[S][I], acc[I][J]);
      __builtin_amdgcn_sched_barrier(0);
      each_between<N * L / MFMAS, (N + 1) * L / MFMAS>(load_one);
      each_between<N * READS / MFMAS, (N + 1) * READS / MFMAS>(read_one);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  typedef std::integral_constant<int, 0> First;
  typedef std::integral_constant<int, 1> Second;
  constexpr int EARLY = LOADS - LOADS / 2;
  typedef std::integral_constant<int, EARLY> EarlyLoads;
  typedef std::integral_constant<int, LOADS - EARLY> LateLoads;

  // Chunk w of the rhs goes with half w + 1 & 1 of pair (w + 1) / 2.
  each_of<A_LOADS>([&](auto i) { load(First{}, i); });
  each_of<LOADS>([&](auto i) { load(Second{}, i); });
  next_chunk();
  next_pair();
  freed += B_STAGE;
  each_of<LOADS>([&](auto i) { load(First{}, i); });
  next_chunk();
  freed += B_STAGE;
  each_of<LOADS>([&](auto i) { load(Second{}, i); });
  next_chunk();
  next_pair();
  freed += B_STAGE;
  each_of<EARLY>([&](auto i) { load(First{}, i); });
  wait_and_meet<2 * LOADS + EARLY>();
  uint32_t pair = 0, stage = B_AT;  // (LDS offsets of what is multiplied)
  each_of<READS>([&](auto i) { read(lds, lds + B_AT, First{}, First{}, i); });
  // A chunk, the first or second of a pair.
  auto chunk = [&](auto which) {
    constexpr int W = decltype(which)::value;
    typedef std::integral_constant<int, W> Late;        // half of the pair whose loads are under way
    typedef std::integral_constant<int, 1 - W> Early;
    multiply(First{}, [&](auto i) { read(lds + pair, lds + stage, which, Second{}, i); }, LateLoads{},
             [&](auto i) { load(Late{}, std::integral_constant<int, EARLY + decltype(i)::value>{}); });
    next_chunk();
    if constexpr (W == 1) next_pair();
    wait_and_meet<2 * LOADS>();
    freed = lds0 + stage;
    stage = stage + B_STAGE == B_AT + 4 * B_STAGE ? B_AT : stage + B_STAGE;
    if constexpr (W == 1) pair = pair + PAIR == B_AT ? 0 : pair + PAIR;
    multiply(Second{}, [&](auto i) { read(lds + pair, lds + stage, Early{}, First{}, i); }, EarlyLoads{}, [&](auto i) { load(Early{}, i); });
  };
  for (uint32_t c = 0; c < chunks; c += 2) {
    chunk(First{});
    chunk(Second{});
  }

  // (Pinned, or the compiler moves accumulators between register files in the loop for the code behind it.)
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j) asm volatile("" : "+a"(acc[i][j]));
  p.epilogue.template store<T, AM, BN>(acc, first_row + wave_m * 32 * AM, first_col + wave_n * (RESULTS / 2), p.lhs.rows, p.rhs.rows, lane, 0);
  // (The last loads have reached LDS before it is given to another workgroup.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// Whether the lhs is one for that.
inline bool whole_lines(const Operand16& lhs, uint32_t depth) {
  return lhs.tile_rows == 1 && depth % 64 == 0 && lhs.stride0 % 128 == 0 && (uintptr_t)lhs.data % 128 == 0;
}

template <Float T, int AM, int BN, bool STREAM = false, typename E>
hipError_t launch_lines_tile(BlockProduct<E, Operand16, Operand16> p, hipStream_t stream) {
  constexpr int LDS = lines_lds_bytes(AM, BN);
  static_assert(LDS <= 160 * 1024 && 2 * (AM + BN) + AM + BN <= 63, "LDS, and loads under way");
  const unsigned groups = lay_out_tiles<AM, BN>(p);
  void (*kernel)(const BlockProduct<E, Operand16, Operand16>) = product16_lines_kernel<T, AM, BN, STREAM, E>;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return e;
  return launch_kernel(kernel, groups, 256, LDS, stream, p);
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_PRODUCT16_LINES_H_
