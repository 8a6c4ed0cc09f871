// Products of 16-bit floats of many rows: block tiles through LDS.
//
// A workgroup of four wavefronts (2 x 2) multiplies 64 AM rows of the lhs with 64 BN rows of the rhs, each wavefront AM x BN
// fragments of v_mfma_f32_32x32x16. K goes by in chunks of 32 values, which travel global memory -> LDS without passing through
// registers into a ring of STAGES stages.
//
// An operand is of one of two kinds. Operand16: a row's K comes in pieces of 16 bytes, four a chunk. LDS holds a chunk's rows sixteen
// by sixteen: one after the other where a row's pieces lie next to each other, these exchanged among themselves so that the lanes that a
// read serves together find theirs in different banks; else as the tiles have them, two pieces of sixteen rows and the two others, or
// a piece of each and then the next, which is no read's conflict. Strided16: the rows' values of one k are contiguous. LDS holds a chunk's 32 ks one after the other, 128 bytes for each 64
// rows, and the transposing read hands a lane four ks of its row: sixteen lanes read 32 bytes of each of four ks, which lie in
// different banks because a k's 32-byte units are exchanged among themselves. Loads write LDS in lane order, so it is the global
// address of a lane that is chosen; neighbouring lanes still read neighbouring pieces.
//
// The rhs fragment is the instruction's row operand, so that a lane ends up with four consecutive columns of one row of the result.
//
// An epilogue E takes the accumulators, and says what the rhs is. E::kPaired: two matrices of the same layout side by side: of each 32
// rows in LDS the first 16 are the first's, the others the second's of the same numbers, so that a lane has both products of a
// column. E::kInTurn: two matrices one behind the other along K, the lhs's K being twice as long (its second half `lhs_second` bytes
// behind its first). E::kCopies: the grid's rows of tiles come several times over, for another lhs and result (`lhs_second` behind the
// first) or, in turn, for another part of K.
//
// What bounds it. (Figures of row-major rows are those of product16_lines.h where their K allows.) Large products the board's power: 4096 x
// 11008 x 4096, gate and up in 256x128 tiles, 611 us with row-major rows, 1.21 PFLOP/s (6 rounds of 256 tiles where 5.4 would do), 2048 x
// 8192 x 4096, two whole rounds, 220 us, 1.25, where a library's plain product of 8192^3 reaches 1.35; with fewer compute units at work a
// chunk takes 0.5 us and not 0.8. Some hundred rows the tiles' number: 512 x 11008 x 4096 in 230 tiles of 256x96 81 us from the caches and
// 90 from memory (87 with the rows in tiles, 102 by half lines). Few rows the weights: 40 x 11008 x 4096 35 us, 180 MB at 5.2 TB/s, and
// short of that LDS, which 64 rows of chunks go into and come out of twice: 64x32 tiles take 0.12 us a chunk however few there are. Neither
// deeper rings, nor touching all of the lhs first, nor columns in two launches (whole rounds, then the rest) gained.
#ifndef IREE_AMD_CSRC_PRODUCT16_BLOCK_H_
#define IREE_AMD_CSRC_PRODUCT16_BLOCK_H_

#include <type_traits>

#include "product16.h"
#include "product16_walk.h"

namespace uk {

template <typename E, typename A, typename B>
struct BlockProduct {
  A lhs;
  B rhs;
  const uint8_t* second;  // the other rhs
  int64_t second_stride0;
  int64_t lhs_second;
  uint32_t depth;         // of one rhs
  uint32_t tile_rows, tile_cols, band_reciprocal;
  E epilogue;
};

namespace {

extern __shared__ uint4 ring[];

// 64 x 16 bytes to LDS byte offset `lds` (of the wavefront) from `base` + the lane's `offset`, past the caches or through them. The
// compiler does not see that they write LDS and keeps no order between them and reads: wait_and_meet does.
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

// Where four pieces of a row lie next to each other, piece `c` lies at c ^ exchanged(row) in LDS.
__device__ __forceinline__ uint32_t exchanged(uint32_t row) { return ((row >> 2) & 3) ^ (row & 2); }

// One side of a tile: 64 W rows from `first` on, loaded 16 bytes a lane, W loads a wavefront for a chunk. `number` of a load: 0 to 4 W -
// 1; `row_number`: the sixteen rows that it has (of a pair half of them are another matrix's).
template <int W>
__device__ __forceinline__ const uint8_t* first_of(const Operand16& o, const uint8_t* data, int64_t stride0, uint32_t first) {
  return uniform_pointer(data + (int64_t)divide(first, o.tile_rows, o.tile_reciprocal) * stride0);
}
// Which of the sixteen rows and which piece of it a lane loads: neighbouring lanes have neighbouring pieces.
__device__ __forceinline__ uint32_t row_of_lane(const Operand16& o, int lane) { return (lane >> o.log2_pieces) & 15; }
__device__ __forceinline__ uint32_t piece_of_lane(const Operand16& o, int lane) {
  const uint32_t next = lane & ((1u << o.log2_pieces) - 1);
  return o.log2_pieces == 2 ? next ^ exchanged(lane >> 2) : next + ((uint32_t)lane >> (4 + o.log2_pieces) << o.log2_pieces);
}
// Where in LDS that is, of sixteen rows: row r's piece g, g < 2; two pieces further on it is at at ^ of_next_step().
__device__ __forceinline__ uint32_t place_of(const Operand16& o, uint32_t r, uint32_t g) {
  return o.log2_pieces == 2 ? r * 64 + 16 * (g ^ exchanged(r)) : o.log2_pieces == 1 ? r * 32 + 16 * g : g * 256 + 16 * r;
}
__device__ __forceinline__ uint32_t of_next_step(const Operand16& o) { return o.log2_pieces == 2 ? 32 : 512; }
// A lane's offset from there. Rows behind the last are read as the last.
template <int W>
__device__ __forceinline__ uint32_t offset_of(const Operand16& o, int64_t stride0, uint32_t first, uint32_t, uint32_t row_number,
                                              int lane, uint32_t depth) {
  uint32_t row = first + row_number * 16 + row_of_lane(o, lane), piece = piece_of_lane(o, lane);
  row = row < o.rows ? row : o.rows - 1;
  if (8 * piece >= depth) piece = 0;  // (less than a chunk of K: it is loaded for nothing, and only what is there)
  const uint32_t panel = divide(row, o.tile_rows, o.tile_reciprocal), first_panel = divide(first, o.tile_rows, o.tile_reciprocal);
  return (uint32_t)((int64_t)(panel - first_panel) * stride0) + (row - panel * o.tile_rows) * o.row_bytes + (piece & 1) * o.piece1 +
         (piece >> 1) * o.piece2;
}
// The lane's piece of what K has behind `full` whole chunks, `rest` values.
template <int W>
__device__ __forceinline__ uint4 rest_of(const Operand16& o, const uint8_t* at, uint32_t, int lane, uint32_t rest) {
  return last_piece(at, (int)rest - 8 * (int)piece_of_lane(o, lane));
}
__device__ __forceinline__ int64_t chunk_step(const Operand16& o) { return 64 * (int64_t)o.tile_rows; }

__device__ __forceinline__ uint32_t column_bytes(const Strided16& o, uint32_t row) {
  const uint32_t tile = divide(row, o.n0, o.n0_reciprocal);
  return tile * o.tile_bytes + 2 * (row - tile * o.n0);
}
template <int W>
__device__ __forceinline__ const uint8_t* first_of(const Strided16& o, const uint8_t* data, int64_t, uint32_t first) {
  return uniform_pointer(data + column_bytes(o, first));
}
template <int W>
__device__ __forceinline__ uint32_t k_of(uint32_t number, int lane) { return (number * 64 + lane) / (8 * W); }
template <int W>
__device__ __forceinline__ uint32_t offset_of(const Strided16& o, int64_t stride0, uint32_t first, uint32_t number, uint32_t, int lane,
                                              uint32_t depth) {
  uint32_t k = k_of<W>(number, lane);
  const uint32_t at = (number * 64 + lane) % (8 * W), piece = 2 * ((at >> 1) ^ (k & 3)) + (at & 1);
  const uint32_t row = first + 8 * piece < o.rows ? first + 8 * piece : o.rows - 8;
  if (k >= depth) k = 0;
  return (k >> o.log2_tile_rows) * (uint32_t)stride0 + (k & ((1u << o.log2_tile_rows) - 1)) * o.row_bytes + column_bytes(o, row) -
         column_bytes(o, first);
}
template <int W>
__device__ __forceinline__ uint4 rest_of(const Strided16&, const uint8_t* at, uint32_t number, int lane, uint32_t rest) {
  return k_of<W>(number, lane) < rest ? *(const uint4*)at : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ int64_t chunk_step(const Strided16& o) { return o.stride0 * (32 >> o.log2_tile_rows); }

// Reads of a fragment of 32 rows: lane (r, g) has row r of it and, of a step's 16 ks, 8 g to 8 g + 7. kReads of them; where a lane's
// first one is in a chunk, `half`: the wavefront's of two.
template <typename O> constexpr int kReads = std::is_same<O, Strided16>::value ? 2 : 1;
template <int W>
__device__ __forceinline__ uint32_t read_at(const Operand16& o, int half, int lane) {
  const int r = lane & 31, g = lane >> 5;
  return half * 2048 * W + (r >> 4) * 1024 + place_of(o, r & 15, g);
}
template <int W>
__device__ __forceinline__ uint32_t read_at(const Strided16&, int half, int lane) {
  const int q = lane >> 4, i = lane & 15;
  return (8 * (q >> 1) + (i >> 2)) * (128 * W) + ((2 * W * half + (q & 1)) ^ (i >> 2)) * 32 + (i & 3) * 8;
}
// Read H of fragment F in step S.
template <int W, int F, int S, int H>
__device__ __forceinline__ void read_piece(const Operand16& o, const uint8_t* side, uint32_t at, uint4& to) {
  to = *(const uint4*)(side + F * 2048 + (S == 0 ? at : at ^ of_next_step(o)));
}
template <int W, int F, int S, int H>
__device__ __forceinline__ void read_piece(const Strided16&, const uint8_t* side, uint32_t at, uint4& to) {
  typedef short v4i16 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) v4i16* Pointer;
  const uint8_t* const from = side + (at ^ (64 * (F & 1))) + 128 * (F >> 1) + (16 * S + 4 * H) * (128 * W);
  const uint2 v = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Pointer)(v4i16*)const_cast<uint8_t*>(from)));
  if constexpr (H == 0) {
    to.x = v.x;
    to.y = v.y;
  } else {
    to.z = v.x;
    to.w = v.y;
  }
}

constexpr int block_lds_bytes(int am, int bn, int stages) { return stages * 64 * (am + bn) * 64; }

constexpr bool two_fit(int am, int bn, int stages) { return am * bn <= 8 && block_lds_bytes(am, bn, stages) <= 80 * 1024; }

// Workgroup `number` of a product's.
template <Float T, int AM, int BN, int STAGES, bool STREAM, typename E, typename A, typename B>
__device__ __forceinline__ void product16_block(const BlockProduct<E, A, B>& p, uint32_t number) {
  constexpr bool PAIRED = E::kPaired, IN_TURN = E::kInTurn;
  constexpr int ROWS = 64 * AM, COLS = 64 * BN, RESULTS = PAIRED ? COLS / 2 : COLS;
  constexpr int A_BYTES = ROWS * 64, STAGE = A_BYTES + COLS * 64;
  constexpr int A_LOADS = AM, B_LOADS = BN, LOADS = A_LOADS + B_LOADS;  // of a wavefront, for a chunk
  static_assert(STAGES >= 3 && (STAGES - 1) * LOADS <= 63, "ring depth");

  const uint32_t tiles = p.tile_rows * p.tile_cols, per_xcd = (tiles + 7) >> 3;
  const uint32_t linear = (number & 7) * per_xcd + (number >> 3);
  if ((number >> 3) >= per_xcd || linear >= tiles) return;
  int tile_row, tile_col;
  tile_of_number(linear, p.tile_rows, p.tile_cols, p.band_reciprocal, &tile_row, &tile_col);
  // (An epilogue's copies: a second result's tiles, or another part of K's, come behind those of the first.)
  uint32_t copy = 0;
  if constexpr (E::kCopies) {
    copy = divide((uint32_t)tile_row, p.epilogue.tile_rows_of_copy, p.epilogue.tile_rows_reciprocal);
    tile_row -= copy * p.epilogue.tile_rows_of_copy;
  }
  const uint32_t first_row = (uint32_t)tile_row * ROWS;
  const uint32_t first_col = (uint32_t)tile_col * RESULTS;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave_m = wave >> 1, wave_n = wave & 1;

  // Loads. Of a pair a load has sixteen rows of the first or of the second.
  const uint8_t* lhs = first_of<AM>(p.lhs, p.lhs.data + (E::kCopies && !IN_TURN ? copy * p.lhs_second : 0), p.lhs.stride0, first_row);
  const uint8_t* const lhs_first = lhs;
  const uint8_t* const rhs_first = first_of<BN>(p.rhs, p.rhs.data, p.rhs.stride0, first_col);
  const uint8_t* const rhs_second = PAIRED || IN_TURN ? first_of<BN>(p.rhs, p.second, p.second_stride0, first_col) : rhs_first;
  auto is_second = [&](int i) { return PAIRED && ((wave * B_LOADS + i) & 1) != 0; };
  auto a_offset = [&](int i) {
    const uint32_t number = wave * A_LOADS + i;
    return offset_of<AM>(p.lhs, p.lhs.stride0, first_row, number, number, lane, p.depth);
  };
  auto b_offset = [&](int i) {
    const uint32_t number = wave * B_LOADS + i;
    return offset_of<BN>(p.rhs, is_second(i) ? p.second_stride0 : p.rhs.stride0, first_col, number, PAIRED ? number / 2 : number, lane, p.depth);
  };
  uint32_t a_from[A_LOADS], b_from[B_LOADS];
#pragma unroll
  for (int i = 0; i < A_LOADS; ++i) a_from[i] = a_offset(i);
#pragma unroll
  for (int i = 0; i < B_LOADS; ++i) b_from[i] = b_offset(i);
  const int64_t lhs_step = chunk_step(p.lhs);
  int64_t rhs_step = chunk_step(p.rhs);
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
  const uint32_t full = p.depth >> 5, rest = p.depth & 31;
  uint32_t by_registers = rest == 0 ? 0 : 1;
  ChunkWalk walk = {0, full, full};
  if constexpr (IN_TURN) {
    by_registers = copy == 0 ? 2 * by_registers : 0;
    walk.at = first_of_split(2 * full, copy, p.epilogue.copies);
    walk.end = first_of_split(2 * full, copy + 1, p.epilogue.copies);
  }
  const uint32_t chunks = walk.end - walk.at + by_registers;
  // Of the second rhs offsets and steps are others where its stride is.
  auto to_second = [&] {
    B other = p.rhs;
    other.stride0 = p.second_stride0;
    rhs_step = chunk_step(other);
    rhs_even = rhs_second;
#pragma unroll
    for (int i = 0; i < B_LOADS; ++i)
      b_from[i] = offset_of<BN>(other, other.stride0, first_col, wave * B_LOADS + i, wave * B_LOADS + i, lane, p.depth);
    lhs = lhs_first + p.lhs_second;
  };
  if constexpr (IN_TURN) {
    uint32_t skipped = walk.at;
    if (walk.at != 0 && walk.at >= full) {
      to_second();
      skipped -= full;
    }
    lhs += skipped * lhs_step;
    rhs_even += skipped * rhs_step;
    rhs_odd = rhs_even;
  }
  auto to_next_chunk = [&] {
    const ChunkWalk::Step step = walk.next();
    if (IN_TURN && step == ChunkWalk::kSecondHalf) {
      to_second();
    } else {
      const bool more = step != ChunkWalk::kStay;
      lhs += more ? lhs_step : 0;
      rhs_even += more ? rhs_step : 0;
      if constexpr (PAIRED && BN > 1) rhs_odd += more ? rhs_step : 0;
    }
    if constexpr (!PAIRED || BN == 1) rhs_odd = rhs_even;
  };

  const uint8_t* lds = (const uint8_t*)ring;
  const uint32_t a_read = read_at<AM>(p.lhs, wave_m, lane), b_read = read_at<BN>(p.rhs, wave_n, lane);
  uint4 a[2][AM], b[2][BN];
  constexpr int A_READS = AM * kReads<A>, READS = A_READS + BN * kReads<B>;
  // Read number I of step S of the chunk at `at`.
  auto read = [&](const uint8_t* at, auto step, auto number) {
    constexpr int S = decltype(step)::value, I = decltype(number)::value;
    if constexpr (I < A_READS) read_piece<AM, I / kReads<A>, S, I % kReads<A>>(p.lhs, at, a_read, a[S][I / kReads<A>]);
    else read_piece<BN, (I - A_READS) / kReads<B>, S, (I - A_READS) % kReads<B>>(p.rhs, at + A_BYTES, b_read, b[S][(I - A_READS) / kReads<B>]);
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

  // What K (of one rhs, and of the other in turn) has behind its last whole chunk comes first, by way of registers, zeros behind it:
  // the loop knows whole chunks only.
  for (uint32_t s = 0; s < by_registers; ++s) {
    const uint8_t* const of_lhs = lhs_first + (s == 0 ? 0 : p.lhs_second) + (int64_t)full * lhs_step;
    B other = p.rhs;
    other.stride0 = p.second_stride0;
    const uint8_t* const of_second = rhs_second + (int64_t)full * chunk_step(other);
    const uint8_t* const of_rhs = s == 0 ? rhs_first + (int64_t)full * chunk_step(p.rhs) : of_second;
    uint8_t* const stage = (uint8_t*)ring + s * STAGE;
#pragma unroll 1
    for (int i = 0; i < A_LOADS; ++i) {
      const uint32_t number = wave * A_LOADS + i;
      *(uint4*)(stage + number * 1024 + 16 * lane) =
          rest_of<AM>(p.lhs, of_lhs + offset_of<AM>(p.lhs, p.lhs.stride0, first_row, number, number, lane, rest), number, lane, rest);
    }
#pragma unroll 1
    for (int i = 0; i < B_LOADS; ++i) {
      const uint32_t number = wave * B_LOADS + i;
      const bool second = is_second(i) || s != 0;
      const uint32_t offset = offset_of<BN>(p.rhs, second ? p.second_stride0 : p.rhs.stride0, first_col, number, PAIRED ? number / 2 : number, lane, rest);
      *(uint4*)(stage + A_BYTES + number * 1024 + 16 * lane) =
          rest_of<BN>(p.rhs, (is_second(i) ? of_second : of_rhs) + offset, number, lane, rest);
    }
  }
  // A chunk: its first step's MFMAs, among them its second step's reads; then the next chunk has come for everyone and this one's
  // stage is free; the second step's MFMAs, among them the next chunk's first reads. The loads of the chunk that goes into the
  // freed stage are dealt out over the two steps behind it.
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if ((uint32_t)s < by_registers) continue;
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
  p.epilogue.template store<T, AM, BN>(acc, first_row + wave_m * 32 * AM, first_col + wave_n * (RESULTS / 2), p.lhs.rows, p.rhs.rows, lane, copy);
  // (The last loads have reached LDS before it is given to another workgroup.)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <Float T, int AM, int BN, int STAGES, bool STREAM, typename E, typename A, typename B>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(two_fit(AM, BN, STAGES) ? 2 : 1, 2)))
void product16_block_kernel(const BlockProduct<E, A, B> p) {
  product16_block<T, AM, BN, STAGES, STREAM>(p, blockIdx.x);
}

// Fills in what a kernel of these tiles needs of the grid, and returns its workgroups, a multiple of 8.
template <int AM, int BN, typename E, typename A, typename B>
unsigned lay_out_tiles(BlockProduct<E, A, B>& p) {
  constexpr int RESULTS = E::kPaired ? 32 * BN : 64 * BN;
  p.tile_rows = (p.lhs.rows + 64 * AM - 1) / (64 * AM);
  if constexpr (E::kCopies) {
    p.epilogue.tile_rows_of_copy = p.tile_rows;
    p.epilogue.tile_rows_reciprocal = reciprocal_of(p.tile_rows);
    p.tile_rows *= p.epilogue.copies;
  }
  p.tile_cols = (p.rhs.rows + RESULTS - 1) / RESULTS;
  p.band_reciprocal = band_reciprocal(p.tile_cols);
  return (p.tile_rows * p.tile_cols + 7) / 8 * 8;
}

template <Float T, int AM, int BN, int STAGES, bool STREAM = false, typename E, typename A, typename B>
hipError_t launch_block_tile(BlockProduct<E, A, B> p, hipStream_t stream) {
  constexpr int LDS = block_lds_bytes(AM, BN, STAGES);
  static_assert(LDS <= 160 * 1024, "LDS");
  const unsigned groups = lay_out_tiles<AM, BN>(p);
  void (*kernel)(const BlockProduct<E, A, B>) = product16_block_kernel<T, AM, BN, STAGES, STREAM, E, A, B>;
  const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
  if (e != hipSuccess) return e;
  return launch_kernel(kernel, groups, 256, LDS, stream, p);
}

}  // namespace
}  // namespace uk

#endif  // IREE_AMD_CSRC_PRODUCT16_BLOCK_H_
