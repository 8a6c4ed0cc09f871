// Products of 16-bit floats of many rows: block tiles through LDS.
//
// A workgroup of four wavefronts (2 x 2) multiplies 64 AM rows of the lhs with 64 BN rows of the rhs, each wavefront AM x BN
// fragments of v_mfma_f32_32x32x16. K goes by in chunks of 32 values, 64 bytes of a row, which travel global memory -> LDS without
// passing through registers into a ring of STAGES stages.
//
// LDS holds a chunk's rows one after the other, a row's 16-byte pieces exchanged among themselves so that the lanes that a read
// serves together find theirs in different banks. Loads write LDS in lane order, so it is the global address of a lane that is
// chosen; four neighbouring lanes still read one row's 64 bytes.
//
// The rhs fragment is the instruction's row operand, so that a lane ends up with four consecutive columns of one row of the result.
//
// An epilogue E takes the accumulators. With E::kPaired the rhs are two matrices of the same layout: of each 32 rows in LDS the
// first 16 are the first's, the others the second's of the same numbers, so that a lane has both products of a column.
#ifndef IREE_AMD_CSRC_PRODUCT16_BLOCK_H_
#define IREE_AMD_CSRC_PRODUCT16_BLOCK_H_

#include <type_traits>

#include "product16.h"

namespace uk {

template <typename E>
struct BlockProduct {
  Operand16 lhs, rhs;
  const uint8_t* second;  // of a pair: the other rhs
  int64_t second_stride0;
  uint32_t depth;         // 32 at least
  uint32_t tile_rows, tile_cols, band_reciprocal;
  E epilogue;
};

namespace {

extern __shared__ uint4 ring[];

// 64 x 16 bytes to LDS byte offset `lds` (of the wavefront) from `base` + the lane's `offset`, past the caches or through them. The compiler does not see that they
// write LDS and keeps no order between them and reads: wait_and_meet does.
template <bool STREAM = false>
__device__ __forceinline__ void load_pieces(uint32_t lds, uint32_t offset, const uint8_t* base) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(offset), "s"(base) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// This wavefront's loads have ended but for the last N, its LDS reads all, and then so have everyone's.
template <int N>
__device__ __forceinline__ void wait_and_meet() {
  static_assert(N >= 0 && N <= 63, "vmcnt is a 6-bit counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ const uint8_t* uniform_pointer(const uint8_t* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const uint8_t*)(((uint64_t)hi << 32) | lo);
}

// f of each number from FROM to TO as a type of its own.
template <int FROM, int TO, typename F>
__device__ __forceinline__ void each_between(F& f) {
  if constexpr (FROM < TO) {
    f(std::integral_constant<int, FROM>{});
    each_between<FROM + 1, TO>(f);
  }
}
template <int N, typename F>
__device__ __forceinline__ void each_of(F f) {
  each_between<0, N>(f);
}

// A row's piece `c` lies at piece c ^ exchanged(row).
__device__ __forceinline__ uint32_t exchanged(uint32_t row) { return ((row >> 2) & 3) ^ (row & 2); }

constexpr int block_lds_bytes(int am, int bn, int stages) { return stages * 64 * (am + bn) * 64; }

template <Float T, int AM, int BN, int STAGES, bool STREAM, typename E>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(AM * BN <= 8 && block_lds_bytes(AM, BN, STAGES) <= 80 * 1024 ? 2 : 1, 2)))
void product16_block_kernel(const BlockProduct<E> p) {
  constexpr bool PAIRED = E::kPaired;
  constexpr int ROWS = 64 * AM, COLS = 64 * BN, RESULTS = PAIRED ? COLS / 2 : COLS;
  constexpr int A_BYTES = ROWS * 64, STAGE = A_BYTES + COLS * 64;
  constexpr int A_LOADS = AM, B_LOADS = BN, LOADS = A_LOADS + B_LOADS;  // of a wavefront, for a chunk
  static_assert(STAGES >= 3 && (STAGES - 1) * LOADS <= 63, "ring depth");

  const uint32_t tiles = p.tile_rows * p.tile_cols, per_xcd = (tiles + 7) >> 3;
  const uint32_t linear = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per_xcd || linear >= tiles) return;
  int tile_row, tile_col;
  tile_of_number(linear, p.tile_rows, p.tile_cols, p.band_reciprocal, &tile_row, &tile_col);
  const uint32_t first_row = (uint32_t)tile_row * ROWS, first_col = (uint32_t)tile_col * RESULTS;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;
  const int r = lane & 31, g = lane >> 5;

  // Loads: offsets of a lane from the panel that the tile begins in. Rows behind the last are read as the last.
  const uint32_t lhs_panel = divide(first_row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
  const uint32_t rhs_panel = divide(first_col, p.rhs.tile_rows, p.rhs.tile_reciprocal);
  const uint8_t* lhs = uniform_pointer(p.lhs.data + (int64_t)lhs_panel * p.lhs.stride0);
  const uint8_t* const rhs_first = uniform_pointer(p.rhs.data + (int64_t)rhs_panel * p.rhs.stride0);
  const uint8_t* const rhs_second = PAIRED ? uniform_pointer(p.second + (int64_t)rhs_panel * p.second_stride0) : rhs_first;
  auto row_offset = [](const Operand16& o, int64_t stride0, uint32_t row, uint32_t first_panel, uint32_t piece) {
    row = row < o.rows ? row : o.rows - 1;
    const uint32_t panel = divide(row, o.tile_rows, o.tile_reciprocal);
    return (uint32_t)((int64_t)(panel - first_panel) * stride0) + (row - panel * o.tile_rows) * o.row_bytes + (piece & 1) * o.piece1 +
           (piece >> 1) * o.piece2;
  };
  // A load has sixteen rows in LDS; of a pair they are the first's or the second's.
  auto is_second = [&](int i) { return PAIRED && ((wave * B_LOADS + i) & 1) != 0; };
  uint32_t a_from[A_LOADS], b_from[B_LOADS];
  auto a_piece_of = [&](int i) { return (lane % 4) ^ exchanged((wave * A_LOADS + i) * 16 + lane / 4); };
  auto b_piece_of = [&](int i) { return (lane % 4) ^ exchanged((wave * B_LOADS + i) * 16 + lane / 4); };
  auto a_offset = [&](int i) {
    return row_offset(p.lhs, p.lhs.stride0, first_row + (wave * A_LOADS + i) * 16 + lane / 4, lhs_panel, a_piece_of(i));
  };
  auto b_offset = [&](int i) {
    const uint32_t number = wave * B_LOADS + i, row = first_col + (PAIRED ? number / 2 : number) * 16 + lane / 4;
    return row_offset(p.rhs, is_second(i) ? p.second_stride0 : p.rhs.stride0, row, rhs_panel, b_piece_of(i));
  };
#pragma unroll
  for (int i = 0; i < A_LOADS; ++i) a_from[i] = a_offset(i);
#pragma unroll
  for (int i = 0; i < B_LOADS; ++i) b_from[i] = b_offset(i);
  const uint32_t lhs_step = 64 * p.lhs.tile_rows, rhs_step = 64 * p.rhs.tile_rows;
  // Of loads 0, 2, .. and of loads 1, 3, .. (of a pair the one's and the other's, in turn)
  const uint8_t *rhs_even = is_second(0) ? rhs_second : rhs_first, *rhs_odd = is_second(1) ? rhs_second : rhs_first;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)ring;
  // Load number I of a chunk, into the stage at LDS offset `at`.
  auto load = [&](uint32_t at, auto number) {
    constexpr int I = decltype(number)::value;
    if constexpr (I < A_LOADS) load_pieces(at + (wave * A_LOADS + I) * 1024, a_from[I], lhs);
    else load_pieces<STREAM>(at + A_BYTES + (wave * B_LOADS + I - A_LOADS) * 1024, b_from[I - A_LOADS], (I - A_LOADS) % 2 ? rhs_odd : rhs_even);
  };
  // Behind the last chunk it is the last that is loaded again: no step is unlike the others.
  const uint32_t full = p.depth >> 5, rest = p.depth & 31, chunks = full + (rest != 0);
  uint32_t loading = 1;
  auto to_next_chunk = [&] {
    const bool more = loading++ < full;
    lhs += more ? lhs_step : 0;
    rhs_even += more ? rhs_step : 0;
    if constexpr (PAIRED && BN > 1) rhs_odd += more ? rhs_step : 0;
    else rhs_odd = rhs_even;
  };

  // Reads: a lane has row r of a fragment and, of the step's 16 values, piece g.
  const uint8_t* lds = (const uint8_t*)ring;
  const uint32_t a_row = (wave_m * 32 * AM + r) * 64, b_row = A_BYTES + (wave_n * 32 * BN + r) * 64;
  const uint32_t piece = 16 * (g ^ exchanged(r));
  uint4 a[2][AM], b[2][BN];
  constexpr int READS = AM + BN;
  // Read number I of step S of the chunk at `at`.
  auto read = [&](const uint8_t* at, auto step, auto number) {
    constexpr int S = decltype(step)::value, I = decltype(number)::value;
    if constexpr (I < AM) a[S][I] = *(const uint4*)(at + a_row + I * 2048 + (piece ^ (32 * S)));
    else b[S][I - AM] = *(const uint4*)(at + b_row + (I - AM) * 2048 + (piece ^ (32 * S)));
  };
  p16_v16f32 acc[AM][BN] = {};
  // A step's MFMAs, and R reads and L loads (numbered) dealt out among them: a wavefront issues in order, what stands in front of
  // an MFMA keeps the matrix pipe waiting.
  constexpr int MFMAS = AM * BN;
  auto multiply = [&](auto step, auto read_count, auto read_one, auto load_count, auto load_one) {
    constexpr int S = decltype(step)::value, R = decltype(read_count)::value, L = decltype(load_count)::value;
    each_of<MFMAS>([&](auto m) {
      constexpr int N = decltype(m)::value, I = N / BN, J = N % BN;
      acc[I][J] = mfma16_32<T>(b[S][J], a[S][I], acc[I][J]);
      __builtin_amdgcn_sched_barrier(0);
      each_between<N * L / MFMAS, (N + 1) * L / MFMAS>(load_one);
      each_between<N * R / MFMAS, (N + 1) * R / MFMAS>(read_one);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  typedef std::integral_constant<int, 0> First;
  typedef std::integral_constant<int, 1> Second;
  typedef std::integral_constant<int, READS> Reads;
  constexpr int EARLY = LOADS - LOADS / 2;  // loads of a chunk that are made in the second step after its stage is free
  typedef std::integral_constant<int, EARLY> EarlyLoads;
  typedef std::integral_constant<int, LOADS - EARLY> LateLoads;

  // What K has behind its last whole chunk comes first, by way of registers, zeros behind it: the loop knows whole chunks only.
  if (rest != 0) {
    auto by_registers = [&](const uint8_t* at, uint32_t to, uint32_t c) {
      *(uint4*)((uint8_t*)ring + to + 16 * lane) = last_piece(at, (int)rest - 8 * (int)c);
    };
#pragma unroll 1
    for (int i = 0; i < A_LOADS; ++i)
      by_registers(lhs + (uint64_t)full * lhs_step + a_offset(i), (wave * A_LOADS + i) * 1024, a_piece_of(i));
#pragma unroll 1
    for (int i = 0; i < B_LOADS; ++i)
      by_registers((is_second(i) ? rhs_second : rhs_first) + (uint64_t)full * rhs_step + b_offset(i), A_BYTES + (wave * B_LOADS + i) * 1024,
                   b_piece_of(i));
  }
  // A chunk: its first step's MFMAs, among them its second step's reads; then the next chunk has come for everyone and this one's
  // stage is free; the second step's MFMAs, among them the next chunk's first reads. The loads of the chunk that goes into the
  // freed stage are dealt out over the two steps behind it.
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (s == 0 && rest != 0) continue;
    each_of<LOADS>([&](auto i) { load(lds0 + s * STAGE, i); });
    to_next_chunk();
  }
  uint32_t stage = 0, freed = lds0 + (STAGES - 1) * STAGE;  // (LDS offsets)
  each_of<EARLY>([&](auto i) { load(freed, i); });
  wait_and_meet<(STAGES - 2) * LOADS + EARLY>();
  each_of<READS>([&](auto i) { read(lds, First{}, i); });
  for (uint32_t c = 0; c < chunks; ++c) {
    multiply(First{}, Reads{}, [&](auto i) { read(lds + stage, Second{}, i); }, LateLoads{},
             [&](auto i) { load(freed, std::integral_constant<int, EARLY + decltype(i)::value>{}); });
    to_next_chunk();
    wait_and_meet<(STAGES - 2) * LOADS>();
    freed = lds0 + stage;
    stage = stage + STAGE == STAGES * STAGE ? 0 : stage + STAGE;
    multiply(Second{}, Reads{}, [&](auto i) { read(lds + stage, First{}, i); }, EarlyLoads{},
             [&](auto i) { load(freed, i); });
  }

  // (Pinned, or the compiler moves accumulators between register files in the loop for the code behind it.)
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j) asm volatile("" : "+a"(acc[i][j]));
  p.epilogue.template store<T, AM, BN>(acc, first_row + wave_m * 32 * AM, first_col + wave_n * (RESULTS / 2), p.lhs.rows, p.rhs.rows, lane);
  // (The last loads have reached LDS before it is given to another workgroup.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <Float T, int AM, int BN, int STAGES, bool STREAM = false, typename E>
hipError_t launch_block_tile(BlockProduct<E> p, hipStream_t stream) {
  constexpr int RESULTS = E::kPaired ? 32 * BN : 64 * BN, LDS = block_lds_bytes(AM, BN, STAGES);
  static_assert(LDS <= 160 * 1024, "LDS");
  p.tile_rows = (p.lhs.rows + 64 * AM - 1) / (64 * AM);
  p.tile_cols = (p.rhs.rows + RESULTS - 1) / RESULTS;
  p.band_reciprocal = band_reciprocal(p.tile_cols);
  const unsigned tiles = p.tile_rows * p.tile_cols;
  void (*kernel)(const BlockProduct<E>) = product16_block_kernel<T, AM, BN, STAGES, STREAM, E>;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return e;
  return launch_kernel(kernel, (tiles + 7) / 8 * 8, 256, LDS, stream, p);
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_PRODUCT16_BLOCK_H_
