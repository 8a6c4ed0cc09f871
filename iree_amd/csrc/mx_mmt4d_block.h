// Microscaled products of many rows: block tiles through LDS.
//
// A workgroup of four wavefronts (2 x 2) multiplies a tile of 64 AM x 64 BN results, each wavefront AM x BN fragments of
// v_mfma_scale_f32_32x32x64. K goes by in chunks of 128 values: 64 bytes of a row of E2M1, 128 of E4M3, and its four scales,
// which travel global memory -> LDS without passing through registers into a ring of STAGES stages.
//
// LDS holds a chunk's rows one after the other, a row's 16-byte pieces exchanged among themselves so that the lanes that a
// read serves together (8 or 16 rows, same piece) find theirs in different banks. Loads write LDS in lane order, so it is the
// global address of a lane that is chosen; four (eight) neighbouring lanes still read one row's 64 (128) bytes.
#ifndef IREE_AMD_CSRC_MX_MMT4D_BLOCK_H_
#define IREE_AMD_CSRC_MX_MMT4D_BLOCK_H_

#include <type_traits>

#include "mx_mmt4d.h"

namespace uk {
namespace {

extern __shared__ uint4 ring[];

// 64 x 16 (or 4) bytes to LDS byte offset `lds` (of the wavefront) from `base` + the lane's `offset`. The compiler does not
// see that they write LDS and keeps no order between them and reads: wait_and_meet does.
__device__ __forceinline__ void load_pieces(uint32_t lds, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_words(uint32_t lds, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
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

// f of each number in [0, N), or from FROM to TO, as a type of its own.
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
template <int BITS>
__device__ __forceinline__ uint32_t exchanged(uint32_t row) {
  if constexpr (BITS == 4) return ((row >> 2) & 3) ^ (row & 2);
  else return ((row >> 1) & 7) ^ ((row & 1) << 2);
}

template <int A_BITS, int B_BITS, int STEP>
__device__ __forceinline__ mx_v16f32 mfma_32(const MxFragment<A_BITS>& a, uint32_t a_scales, const MxFragment<B_BITS>& b,
                                             uint32_t b_scales, mx_v16f32 acc) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(a), mx_operand(b), acc, MxFormat<A_BITS>::value,
                                                         MxFormat<B_BITS>::value, 2 * STEP, (int)a_scales, 2 * STEP,
                                                         (int)b_scales);
}

// A wavefront's fragments to memory, of which a lane has column r = lane % 32 and rows 8 q + 4 g + {0..3}, q = 0..3, g = lane /
// 32. An instruction writes 32 neighbouring columns of two rows. Of 16-bit results two neighbouring lanes exchange one of two
// rows, and each writes two columns of one row (PAIRS).
//
// Eight rows from a multiple of eight on are equally far apart (tiles one row tall, or a multiple of eight): an address is a
// part that is the wavefront's (scalar) and 32 bits that are the lane's. WHOLE: every row and column exists, and the code is
// straight: 4096^2 f32 results of K = 128 took 14.6 us with a test in front of each store.
template <Float OUT, bool ACCUMULATE, bool PAIRS, bool WHOLE, int AM, int BN>
__device__ __forceinline__ void store_results(const MxProduct& p, const mx_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0,
                                              int lane) {
  constexpr int SIZE = OUT == Float::kF32 ? 4 : 2;
  const int r = lane & 31, g = lane >> 5;
  const int64_t row_step = (p.lhs.tile_rows == 1 ? p.out_stride0 : (int64_t)p.n0) * SIZE;
  const int odd = PAIRS ? lane & 1 : 0;
  const uint32_t lane_row = 4 * g + odd;
  const int64_t first_col_at = mx_out_col(p, col0);
  uint8_t* const first = p.out + first_col_at * SIZE;
#pragma unroll
  for (int j = 0; j < BN; ++j) {
    const uint32_t col = col0 + 32 * j + r;
    if (!WHOLE && col >= p.rhs.rows) continue;  // (pairs: the number of columns is even)
    const uint32_t lane_at = (uint32_t)(mx_out_col(p, col - odd) - first_col_at) * SIZE + lane_row * (uint32_t)row_step;
#pragma unroll
    for (int i = 0; i < AM; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t row = row0 + 32 * i + 8 * q;
        if (!WHOLE && row >= p.lhs.rows) continue;
        uint8_t* const at = first + mx_out_row(p, row) * SIZE;
#pragma unroll
        for (int e = 0; e < 4; e += PAIRS ? 2 : 1) {
          uint8_t* const to = at + e * row_step + lane_at;
          if constexpr (PAIRS) {
            const float mine = acc[i][j][4 * q + e], next = acc[i][j][4 * q + e + 1];
            const float given = odd ? mine : next;
            const float taken = __builtin_bit_cast(
                float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, given), 0xB1, 0xF, 0xF, true));
            float left = odd ? taken : mine, right = odd ? next : taken;
            if (!WHOLE && row + lane_row + e >= p.lhs.rows) continue;
            if constexpr (ACCUMULATE) {
              const uint32_t old = *(uint32_t*)to;
              left += mx_widen<OUT>((uint16_t)old);
              right += mx_widen<OUT>((uint16_t)(old >> 16));
            }
            *(uint32_t*)to = mx_narrow_pair<OUT>(left, right);
          } else {
            if (!WHOLE && row + lane_row + e >= p.lhs.rows) continue;
            float v = acc[i][j][4 * q + e];
            if constexpr (OUT == Float::kF32) {
              *(float*)to = ACCUMULATE ? *(float*)to + v : v;
            } else {
              if constexpr (ACCUMULATE) v += mx_widen<OUT>(*(uint16_t*)to);
              *(uint16_t*)to = mx_narrow<OUT>(v);
            }
          }
        }
      }
    }
  }
}

template <Float OUT, int AM, int BN>
__device__ __forceinline__ void store_tile(const MxProduct& p, const mx_v16f32 (&acc)[AM][BN], uint32_t row0, uint32_t col0,
                                           int lane) {
  constexpr bool PAIRS = OUT != Float::kF32;
  const bool whole = row0 + 32 * AM <= p.lhs.rows && col0 + 32 * BN <= p.rhs.rows && (!PAIRS || p.fours);
  if (p.accumulate) {
    if (whole) store_results<OUT, true, PAIRS, true, AM, BN>(p, acc, row0, col0, lane);
    else store_results<OUT, true, false, false, AM, BN>(p, acc, row0, col0, lane);
  } else {
    if (whole) store_results<OUT, false, PAIRS, true, AM, BN>(p, acc, row0, col0, lane);
    else store_results<OUT, false, false, false, AM, BN>(p, acc, row0, col0, lane);
  }
}

// Groups of four chunks' scales in LDS: one is loaded with the four chunks before its own, `stages` chunks ahead of the
// multiplication, which may then still read the one that held its place: 4 * groups > stages + 6.
constexpr int groups_held(int stages) { return (stages + 6) / 4 + 1; }
constexpr int lds_bytes(int lbits, int am, int bn, int stages, bool grouped) {
  return stages * (64 * am * 16 * lbits + 64 * bn * 68 + (grouped ? 0 : 256 * am)) + (grouped ? groups_held(stages) * 64 * am * 16 : 0);
}

// GROUPED: the lhs is row-major. A chunk's scales are then four bytes of each row, a cache line each, and a load takes a cycle for
// every line that it touches: 64 rows, 64 cycles, where 16 bytes a lane take 16. So they come four chunks at a time, 16 bytes
// of a row, sixteen rows with each chunk's loads and a whole group of four chunks ahead of its use.
template <int LBITS, int AM, int BN, int STAGES, bool GROUPED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(AM * BN <= 8 && lds_bytes(LBITS, AM, BN, STAGES, GROUPED) <= 80 * 1024 ? 2 : 1, 2)))
void mx_mmt4d_block_kernel(const MxProduct p) {
  constexpr int ROWS = 64 * AM, COLS = 64 * BN;
  constexpr int A_ROW = 16 * LBITS, B_ROW = 64;                       // bytes of a row's chunk
  constexpr int A_BYTES = ROWS * A_ROW, B_BYTES = COLS * B_ROW;
  constexpr int S_ROWS = (GROUPED ? 0 : AM) + BN;                      // of 64: scales that come chunk by chunk
  constexpr int STAGE = A_BYTES + B_BYTES + 256 * S_ROWS;
  constexpr int GROUP = 16 * ROWS, GROUPS_AT = STAGES * STAGE;        // scales of four chunks; where they lie
  constexpr int A_LOADS = A_BYTES / 4096, B_LOADS = B_BYTES / 4096;   // of a wavefront, for a chunk
  constexpr int S_LOADS = (S_ROWS + 3) / 4;                           // (64 rows each; those left over are made twice)
  constexpr int LOADS = A_LOADS + B_LOADS + S_LOADS + (GROUPED ? 1 : 0);
  static_assert(STAGES >= 3 && (STAGES - 1) * LOADS <= 63, "ring depth");

  const uint32_t tiles = p.tile_rows * p.tile_cols, per_xcd = (tiles + 7) >> 3;
  const uint32_t linear = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per_xcd || linear >= tiles) return;
  int tile_row, tile_col;
  tile_of_number(linear, p.tile_rows, p.tile_cols, p.band_reciprocal, &tile_row, &tile_col);
  const uint32_t first_row = (uint32_t)tile_row * ROWS, first_col = (uint32_t)tile_col * COLS;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;
  const int r = lane & 31, g = lane >> 5;

  // Loads: offsets of a lane from the panel that the tile begins in. Rows behind the last are read as the last.
  const uint32_t lhs_panel = divide(first_row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
  const uint32_t rhs_panel = divide(first_col, p.rhs.tile_rows, p.rhs.tile_reciprocal);
  const uint8_t* lhs = uniform_pointer(p.lhs.codes + (int64_t)lhs_panel * p.lhs.stride0);
  const uint8_t* rhs = uniform_pointer(p.rhs.codes + (int64_t)rhs_panel * p.rhs.stride0);
  const uint8_t* lhs_scales = uniform_pointer(p.lhs.scales + (int64_t)lhs_panel * p.lhs.scales_stride0);
  const uint8_t* rhs_scales = uniform_pointer(p.rhs.scales + (int64_t)rhs_panel * p.rhs.scales_stride0);
  auto row_offset = [](const MxOperand& o, uint32_t row, uint32_t first_panel, int64_t stride, uint32_t row_bytes) {
    row = row < o.rows ? row : o.rows - 1;
    const uint32_t panel = divide(row, o.tile_rows, o.tile_reciprocal);
    return (uint32_t)((int64_t)(panel - first_panel) * stride) + (row - panel * o.tile_rows) * row_bytes;
  };
  uint32_t a_from[A_LOADS], b_from[B_LOADS], s_from[S_LOADS], s_to[S_LOADS];
  bool s_of_lhs[S_LOADS];
#pragma unroll
  for (int i = 0; i < A_LOADS; ++i) {
    constexpr int PIECES = A_ROW / 16, AT_ONCE = 64 / PIECES;  // of a row; rows of a load
    const uint32_t row = (wave * A_LOADS + i) * AT_ONCE + lane / PIECES;
    a_from[i] = row_offset(p.lhs, first_row + row, lhs_panel, p.lhs.stride0, A_ROW) + 16 * ((lane % PIECES) ^ exchanged<LBITS>(row));
  }
#pragma unroll
  for (int i = 0; i < B_LOADS; ++i) {
    const uint32_t row = (wave * B_LOADS + i) * 16 + lane / 4;
    b_from[i] = row_offset(p.rhs, first_col + row, rhs_panel, p.rhs.stride0, B_ROW) + 16 * ((lane % 4) ^ exchanged<4>(row));
  }
#pragma unroll
  for (int i = 0; i < S_LOADS; ++i) {
    const int number = (wave + 4 * i) % S_ROWS, of_rhs = number - (S_ROWS - BN);
    s_of_lhs[i] = of_rhs < 0;
    s_to[i] = A_BYTES + B_BYTES + 256 * number;
    s_from[i] = s_of_lhs[i] ? row_offset(p.lhs, first_row + 64 * number + lane, lhs_panel, p.lhs.scales_stride0, 4)
                            : row_offset(p.rhs, first_col + 64 * of_rhs + lane, rhs_panel, p.rhs.scales_stride0, 4);
  }
  // Groups: a wavefront loads sixteen rows of a quarter of the tile's (64-row tiles: of all of it), a lane four bytes.
  constexpr int QUARTER = 16 * AM, SHARES = AM >= 4 ? 4 : AM;          // rows; wavefronts that they are dealt to, over and over
  const uint32_t group_row = (wave % SHARES) * 16 + lane / 4;
  const uint32_t last_row = p.lhs.rows - 1 - first_row;
  const uint32_t lhs_step = A_ROW * p.lhs.tile_rows, rhs_step = B_ROW * p.rhs.tile_rows;
  const uint32_t lhs_scales_step = 4 * p.lhs.tile_rows, rhs_scales_step = 4 * p.rhs.tile_rows;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)ring;
  // A quarter of the group of scales at `group_from` (the last group ends with the last chunk), to LDS offset `group_to`.
  const uint8_t* group_from = lhs_scales;
  uint32_t group_to = GROUPS_AT, group_quarter = 0, group_first = 0;
  auto load_group = [&](uint32_t quarter) {
    const uint32_t row = quarter * QUARTER + group_row;
    load_words(lds0 + group_to + quarter * (QUARTER * 16) + (wave % SHARES) * 256,
               (row < last_row ? row : last_row) * (uint32_t)p.lhs.scales_stride0 + 4 * (lane % 4), group_from);
  };
  auto to_next_group = [&] {
    group_first = group_first + 8 <= p.chunks ? group_first + 4 : p.chunks - 4;
    group_from = lhs_scales + 4 * group_first;
    group_to = group_to + GROUP == GROUPS_AT + groups_held(STAGES) * GROUP ? GROUPS_AT : group_to + GROUP;
  };
  // Load number I of a chunk, into the stage at LDS offset `at`.
  auto load = [&](uint32_t at, auto number) {
    constexpr int I = decltype(number)::value;
    if constexpr (I < A_LOADS) load_pieces(at + (wave * A_LOADS + I) * 1024, a_from[I], lhs);
    else if constexpr (I < A_LOADS + B_LOADS)
      load_pieces(at + A_BYTES + (wave * B_LOADS + I - A_LOADS) * 1024, b_from[I - A_LOADS], rhs);
    else if constexpr (I < A_LOADS + B_LOADS + S_LOADS)
      load_words(at + s_to[I - A_LOADS - B_LOADS], s_from[I - A_LOADS - B_LOADS],
                 s_of_lhs[I - A_LOADS - B_LOADS] ? lhs_scales : rhs_scales);
    else
      load_group(group_quarter);
  };
  // Behind the last chunk it is the last that is loaded again: no step is unlike the others (with steps of their own for the
  // last chunks the compiler keeps the accumulators twice, or in scratch memory).
  const uint32_t chunks = p.chunks;
  uint32_t loading = 1;
  auto to_next_chunk = [&] {
    const bool more = loading++ < chunks;
    lhs += more ? lhs_step : 0;
    rhs += more ? rhs_step : 0;
    if constexpr (GROUPED) {
      group_quarter = (group_quarter + 1) & 3;
      if (group_quarter == 0) to_next_group();
    } else {
      lhs_scales += more ? lhs_scales_step : 0;
    }
    rhs_scales += more ? rhs_scales_step : 0;
  };

  // Reads: a lane has row r of a fragment and, of the step's 64 values, block g (see MxFragment for the halves of 8-bit codes).
  const uint8_t* lds = (const uint8_t*)ring;
  const uint32_t a_row = (wave_m * 32 * AM + r) * A_ROW, b_row = A_BYTES + (wave_n * 32 * BN + r) * B_ROW;
  const uint32_t a_piece = 16 * (g ^ exchanged<LBITS>(r)), b_piece = 16 * (g ^ exchanged<4>(r));
  const uint32_t a_scale = (GROUPED ? 16 : 4) * (wave_m * 32 * AM + r) + (GROUPED ? 0 : A_BYTES + B_BYTES);
  const uint32_t b_scale = A_BYTES + B_BYTES + 4 * (64 * (S_ROWS - BN) + wave_n * 32 * BN + r);
  MxFragment<LBITS> a[2][AM];
  MxFragment<4> b[2][BN];
  uint32_t a_read[AM], b_read[BN], as[AM], bs[BN];
  constexpr int A_READS = AM * LBITS / 4, READS = A_READS + BN;  // and AM + BN of scales, with a chunk's first step
  // Groups: where the scales of the chunk to be read lie, by its number.
  uint32_t scales_at = GROUPS_AT, scales_group = 0, scales_first = 0;
  auto scales_of_chunk = [&](uint32_t c) {
    c = c < p.chunks ? c : p.chunks - 1;
    if (c % 4 == 0 && c != 0) {
      scales_group = scales_group == groups_held(STAGES) - 1 ? 0 : scales_group + 1;
      scales_first = c + 4 <= p.chunks ? c : p.chunks - 4;
    }
    scales_at = GROUPS_AT + scales_group * GROUP + 4 * (c - scales_first);
  };
  // Read number I of step S of the chunk at `at`.
  auto read = [&](const uint8_t* at, auto step, auto number) {
    constexpr int S = decltype(step)::value, I = decltype(number)::value;
    if constexpr (I < A_READS) {
      constexpr int HALF = LBITS == 8 ? I % 2 : 0, F = LBITS == 8 ? I / 2 : I;
      *(uint4*)(a[S][F].w + 4 * HALF) = *(const uint4*)(at + a_row + F * 32 * A_ROW + (a_piece ^ (8 * LBITS * S) ^ (32 * HALF)));
    } else if constexpr (I < READS) {
      constexpr int F = I - A_READS;
      *(uint4*)b[S][F].w = *(const uint4*)(at + b_row + F * 32 * B_ROW + (b_piece ^ (32 * S)));
    } else if constexpr (I < READS + AM) {
      if constexpr (GROUPED) a_read[I - READS] = *(const uint32_t*)(lds + scales_at + a_scale + (I - READS) * 512);
      else a_read[I - READS] = *(const uint32_t*)(at + a_scale + (I - READS) * 128);
    } else {
      b_read[I - READS - AM] = *(const uint32_t*)(at + b_scale + (I - READS - AM) * 128);
    }
  };
  // A lane's scales of the chunk: blocks g and 2 + g of four, now in bytes 0 and 2.
  auto take_scales = [&] {
#pragma unroll
    for (int i = 0; i < AM; ++i) as[i] = a_read[i] >> (8 * g);
#pragma unroll
    for (int j = 0; j < BN; ++j) bs[j] = b_read[j] >> (8 * g);
  };
  mx_v16f32 acc[AM][BN] = {};
  // A step's MFMAs, and R reads and L loads (numbered) dealt out among them: a wavefront issues in order, what stands in front
  // of an MFMA keeps the matrix pipe waiting, and a load stands there for 16 cycles of every wavefront's.
  constexpr bool SPLIT = LBITS == 8;  // (mx_split)
  constexpr int MFMAS = AM * BN * (SPLIT ? 2 : 1);
  auto multiply = [&](auto step, auto read_count, auto read_one, auto load_count, auto load_one) {
    constexpr int S = decltype(step)::value, R = decltype(read_count)::value, L = decltype(load_count)::value;
    MxFragment<8> high, low;
    each_of<MFMAS>([&](auto m) {
      constexpr int N = decltype(m)::value, PART = SPLIT ? N / BN % 2 : 0, I = SPLIT ? N / BN / 2 : N / BN, J = N % BN;
      if constexpr (SPLIT) {
        if constexpr (PART == 0 && J == 0) mx_split(a[S][I], high, low);
        acc[I][J] = mfma_32<8, 4, S>(PART == 0 ? high : low, as[I], b[S][J], bs[J], acc[I][J]);
      } else {
        acc[I][J] = mfma_32<LBITS, 4, S>(a[S][I], as[I], b[S][J], bs[J], acc[I][J]);
      }
      __builtin_amdgcn_sched_barrier(0);
      each_between<N * L / MFMAS, (N + 1) * L / MFMAS>(load_one);
      each_between<N * R / MFMAS, (N + 1) * R / MFMAS>(read_one);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  typedef std::integral_constant<int, 0> First;
  typedef std::integral_constant<int, 1> Second;
  typedef std::integral_constant<int, READS> Reads;
  typedef std::integral_constant<int, READS + AM + BN> FirstReads;
  constexpr int EARLY = LOADS - LOADS / 2;  // loads of a chunk that are made in the second step after its stage is free
  typedef std::integral_constant<int, EARLY> EarlyLoads;
  typedef std::integral_constant<int, LOADS - EARLY> LateLoads;

  // A chunk: its first step's MFMAs, among them its second step's reads; then the next chunk has come for everyone and this
  // one's stage is free; the second step's MFMAs, among them the next chunk's first reads. The loads of the chunk that goes
  // into the freed stage are dealt out over the two steps behind it.
  if constexpr (GROUPED) {
#pragma unroll
    for (int q = 0; q < 4; ++q) load_group(q);
    to_next_group();
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    each_of<LOADS>([&](auto i) { load(lds0 + s * STAGE, i); });
    to_next_chunk();
  }
  uint32_t stage = 0, freed = lds0 + (STAGES - 1) * STAGE;  // (LDS offsets)
  each_of<EARLY>([&](auto i) { load(freed, i); });
  wait_and_meet<(STAGES - 2) * LOADS + EARLY>();
  each_of<READS + AM + BN>([&](auto i) { read(lds, First{}, i); });
  for (uint32_t c = 0; c < chunks; ++c) {
    take_scales();
    multiply(First{}, Reads{}, [&](auto i) { read(lds + stage, Second{}, i); }, LateLoads{},
             [&](auto i) { load(freed, std::integral_constant<int, EARLY + decltype(i)::value>{}); });
    to_next_chunk();
    wait_and_meet<(STAGES - 2) * LOADS>();
    freed = lds0 + stage;
    stage = stage + STAGE == STAGES * STAGE ? 0 : stage + STAGE;
    if constexpr (GROUPED) scales_of_chunk(c + 1);
    multiply(Second{}, FirstReads{}, [&](auto i) { read(lds + stage, First{}, i); }, EarlyLoads{},
             [&](auto i) { load(freed, i); });
  }

  // (Pinned, or the compiler moves accumulators between register files in the loop for the code behind it.)
#pragma unroll
  for (int i = 0; i < AM; ++i)
#pragma unroll
    for (int j = 0; j < BN; ++j) asm volatile("" : "+a"(acc[i][j]));
  const uint32_t row0 = first_row + wave_m * 32 * AM, col0 = first_col + wave_n * 32 * BN;
  if (p.out_type == Float::kF32) store_tile<Float::kF32, AM, BN>(p, acc, row0, col0, lane);
  else if (p.out_type == Float::kF16) store_tile<Float::kF16, AM, BN>(p, acc, row0, col0, lane);
  else store_tile<Float::kBf16, AM, BN>(p, acc, row0, col0, lane);
  // (The last loads have reached LDS before it is given to another workgroup.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int LBITS, int AM, int BN, int STAGES>
hipError_t launch(MxProduct p, hipStream_t stream) {
  p.tile_rows = (p.lhs.rows + 64 * AM - 1) / (64 * AM);
  p.tile_cols = (p.rhs.rows + 64 * BN - 1) / (64 * BN);
  p.band_reciprocal = band_reciprocal(p.tile_cols);
  const unsigned tiles = p.tile_rows * p.tile_cols;
  const bool grouped = p.lhs.tile_rows == 1 && p.chunks >= 4;
  const int lds = lds_bytes(LBITS, AM, BN, STAGES, grouped);
  static_assert(lds_bytes(LBITS, AM, BN, STAGES, true) <= 160 * 1024 && lds_bytes(LBITS, AM, BN, STAGES, false) <= 160 * 1024, "LDS");
  auto* kernel = grouped ? mx_mmt4d_block_kernel<LBITS, AM, BN, STAGES, true>
                         : mx_mmt4d_block_kernel<LBITS, AM, BN, STAGES, false>;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  return launch_kernel(kernel, (tiles + 7) / 8 * 8, 256, lds, stream, p);
}

template <int LBITS>
hipError_t launch_block(const MxProduct& p, int tile, hipStream_t stream) {
  constexpr bool FOUR = LBITS == 4;
  switch (tile) {  // kMxBlockTiles
    case 0: return launch<LBITS, 4, 4, FOUR ? 4 : 3>(p, stream);
    case 1: return launch<LBITS, 2, 2, FOUR ? 4 : 3>(p, stream);
    case 2: return launch<LBITS, 2, 3, 3>(p, stream);
    case 3: return launch<LBITS, 2, 4, FOUR ? 3 : 4>(p, stream);
    case 4: return launch<LBITS, 1, 1, FOUR ? 6 : 5>(p, stream);
    case 5: return launch<LBITS, 2, 1, FOUR ? 5 : 3>(p, stream);
    case 6: return launch<LBITS, 1, 2, FOUR ? 5 : 4>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_MX_MMT4D_BLOCK_H_
