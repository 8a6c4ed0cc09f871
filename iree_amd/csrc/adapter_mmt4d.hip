// Low-rank adapters of many requests at once: each row of the lhs times the `down` of its adapter, rank sums of f32 in the
// workspace, then those times its `up`.
#include <type_traits>

#include "product16.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

struct AdapterKernelArgs {
  AdapterArgs p;
  int64_t results;
};

// The adapter of a row; -1: none.
__device__ __forceinline__ int32_t adapter_of(const AdapterArgs& a, int64_t row) {
  if (a.count == 0) return -1;
  const int32_t i = a.index[row];
  return i < 0 || i >= a.count ? -1 : i;
}

template <Float T>
__global__ __launch_bounds__(kThreads) void adapter_down_generic(const AdapterKernelArgs g) {
  const AdapterArgs& a = g.p;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t row = n / a.rank, r = n % a.rank;
    const int32_t of = adapter_of(a, row);
    if (of < 0) continue;
    const uint16_t* lhs = (const uint16_t*)a.lhs + row / a.M0 * a.lhs_stride0 + row % a.M0 * a.K0;
    const uint16_t* down = (const uint16_t*)a.down + of * a.down_stride0 + r * a.down_stride1;
    float sum = 0;
    for (int64_t k = 0; k < a.K; ++k)
      for (int k0 = 0; k0 < a.K0; ++k0) sum += mx_widen<T>(lhs[k * a.M0 * a.K0 + k0]) * mx_widen<T>(down[k * a.K0 + k0]);
    ((float*)a.workspace)[n] = sum;
  }
}

template <Float T>
__global__ __launch_bounds__(kThreads) void adapter_up_generic(const AdapterKernelArgs g) {
  const AdapterArgs& a = g.p;
  const int64_t cols = a.N * a.N0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t row = n / cols, col = n % cols;
    const int32_t of = adapter_of(a, row);
    if (of < 0 && a.accumulate) continue;
    float sum = 0;
    if (of >= 0) {
      const uint16_t* up = (const uint16_t*)a.up + of * a.up_stride0 + col * a.up_stride1;
      const float* t = (const float*)a.workspace + row * a.rank;
      for (int64_t r = 0; r < a.rank; ++r) sum += t[r] * mx_widen<T>(up[r]);
      if (a.scales) sum *= a.scales[of];
    }
    const int64_t at = row / a.M0 * a.out_stride0 + (col / a.N0 * a.M0 + row % a.M0) * a.N0 + col % a.N0;
    put_element(a.out_type, a.out, at, a.accumulate ? element(a.out_type, a.out, at) + sum : sum);
  }
}

hipError_t launch_over(void (*f16)(const AdapterKernelArgs), void (*bf16)(const AdapterKernelArgs), const AdapterArgs& a, int64_t results,
                       hipStream_t stream) {
  AdapterKernelArgs g{a, results};
  const int64_t groups = (results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  return launch_kernel(a.type == Float::kF16 ? f16 : bf16, grid, kThreads, 0, stream, g);
}

//===----------------------------------------------------------------------===//
// On the matrix pipe
//===----------------------------------------------------------------------===//
//
// Sixteen rows at a time, and of these all that one adapter has: the tile's adapters are numbered in the order of their first
// rows, and a workgroup takes every SLOTS-th of them. A row has one adapter, so nobody else writes its results; what the matrix
// instructions compute of the other rows is thrown away, and what is not finite there stays there.
//
// Many rows of few adapters are put in order first: a tile is then sixteen rows of one adapter, wherever they are, and each adapter is
// read once for every sixteen of its rows whatever the order of rows. (Which of an adapter's rows share a tile is up to atomics, and does
// not matter: a row's results do not depend on the others.)

constexpr int kFragments = 4;  // of 16 columns that a wavefront multiplies by `up`, and of 16 ranks by `down`, at most

struct AdapterProduct {
  Operand16 lhs;
  const uint8_t *down, *up;
  int64_t down_stride0, down_stride1, up_stride0, up_stride1;  // bytes
  const int32_t* index;
  const float* scales;
  float* sums;              // [splits][rows][pitch]
  uint8_t* out;
  Layout out_at;
  Float out_type;
  uint32_t depth, rank, count, cols, pitch, splits;
  uint32_t turns;           // blocks of columns that a wavefront multiplies by `up`, one after the other
  uint32_t tiles, slots, units;  // of a launch: workgroups' pieces of work
  const uint4* heads;       // rows in order: of each tile its adapter (count: none), its first row's place in the order, its rows
  const uint32_t* ids;      // and the sixteen rows; else null
  uint32_t parts, parts_reciprocal, slots_reciprocal;
  int32_t accumulate, runs;
};

// f(adapter, which of the tile's sixteen rows have it, the row of lane % 16, the first one's place among the sums) for every `slots`-th
// adapter of a tile. zeros(which of the rows have none, the row of lane % 16), by the first slot.
template <typename F, typename Z>
__device__ __forceinline__ void of_adapters(const AdapterProduct& p, uint32_t tile, uint32_t slot, int lane, F f, Z zeros) {
  const uint32_t at = tile * 16 + (lane & 15);
  uint32_t row, first = tile * 16, without, todo;  // todo: a bit for each adapter left, that of its first row
  int32_t named;
  if (p.heads) {
    const uint32_t id = p.ids[at];
    const uint4 head = p.heads[tile];
    const uint32_t rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)head.z), mask = (1u << rows) - 1;
    named = (uint32_t)(lane & 15) < rows && head.x < p.count ? (int32_t)head.x : -1;
    // (Read by all lanes: as an operand of the choice only those lanes would read it that have no row, and the first of them.)
    const uint32_t first_id = (uint32_t)__builtin_amdgcn_readfirstlane((int)id);
    row = (uint32_t)(lane & 15) < rows ? id : first_id;
    first = (uint32_t)__builtin_amdgcn_readfirstlane((int)head.y);
    const bool any = (uint32_t)__builtin_amdgcn_readfirstlane((int)head.x) < p.count;
    todo = any && rows != 0 ? 1 : 0;
    without = any ? 0 : mask;
  } else {
    row = at < p.lhs.rows ? at : p.lhs.rows - 1;
    named = at < p.lhs.rows ? p.index[at] : -1;
    const uint32_t with = (uint32_t)__builtin_amdgcn_ballot_w64(named >= 0 && (uint32_t)named < p.count) & 0xFFFF;
    // The first rows of adapters: nobody before has the same. (Lanes compare with the fifteen in front of them; -1 where there is none, and such a row has no adapter.)
    bool again = false;
    int32_t before = named;
#pragma unroll
    for (int back = 1; back < 16; ++back) {
      before = __builtin_amdgcn_update_dpp(-1, before, 0x111, 0xF, 0xF, false);  // (of the lane in front, within sixteen)
      again |= before == named;
    }
    todo = (uint32_t)__builtin_amdgcn_ballot_w64(!again) & with;
    for (uint32_t i = slot; i != 0 && todo != 0; --i) todo &= todo - 1;
    without = slot == 0 ? ~with & (p.lhs.rows - first < 16 ? (1u << (p.lhs.rows - first)) - 1 : 0xFFFF) : 0;
  }
  while (todo != 0) {
    const int32_t of = __builtin_amdgcn_readlane(named, __builtin_ctz(todo));
    f((uint32_t)of, (uint32_t)__builtin_amdgcn_ballot_w64(named == of) & 0xFFFF, row, first);
    for (uint32_t i = 0; i < p.slots && todo != 0; ++i) todo &= todo - 1;
  }
  zeros(without, row);
}

// Rows in the order of their adapters, those without one behind them, and the tiles that this makes, by one workgroup: each row takes a
// number among its adapter's, then where an adapter's first row and first tile come makes that a place. Adapters' counts are in LDS; a
// wavefront's rows of one adapter take their numbers at once while they are many. The first rows of a thread stay in registers, others'
// numbers wait in memory. (2000 rows, 12 adapters in runs: 4.9 us; one row at a time, and twice over the indices, 7.3.)
constexpr uint32_t kMostOrdered = 2047, kOrderThreads = 1024;
struct OrderArgs {
  const int32_t* index;
  uint4* heads;
  uint32_t* ids;
  uint32_t* numbers;            // of rows; what the rank sums take later
  uint32_t rows, count, tiles;  // tiles: as many as there may be
};
__global__ __launch_bounds__(kOrderThreads) void adapter_order_kernel(const OrderArgs p) {
  __shared__ uint32_t rows_of[kMostOrdered + 1], first_row[kMostOrdered + 1], first_tile[kMostOrdered + 1];
  __shared__ uint32_t wave_rows[kOrderThreads / 64], wave_tiles[kOrderThreads / 64];
  constexpr uint32_t KEPT = 4;
  const uint32_t thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, entries = p.count + 1;
  auto adapter_of = [&](uint32_t row) {
    const int32_t i = p.index[row < p.rows ? row : p.rows - 1];
    return i < 0 || (uint32_t)i >= p.count ? p.count : (uint32_t)i;
  };
  // (By all lanes of a wavefront.)
  auto number_of = [&](uint32_t adapter, bool is_row) {
    uint64_t todo = __builtin_amdgcn_ballot_w64(is_row);
    uint32_t number = 0;
    for (bool many = true; many && todo != 0;) {
      const uint32_t leader = (uint32_t)__builtin_ctzll(todo), of = (uint32_t)__builtin_amdgcn_readlane((int)adapter, (int)leader);
      const bool same = is_row && adapter == of;
      const uint64_t all = __builtin_amdgcn_ballot_w64(same);
      uint32_t base = 0;
      if (lane == leader) base = atomicAdd(&rows_of[of], (uint32_t)__builtin_popcountll(all));
      base = (uint32_t)__builtin_amdgcn_readlane((int)base, (int)leader);
      const uint32_t in_front = __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
      number = same ? base + in_front : number;
      todo &= ~all;
      many = __builtin_popcountll(all) >= 16;  // (else rows are mixed, and hinder each other little)
    }
    if ((todo >> lane & 1) != 0) number = atomicAdd(&rows_of[adapter], 1u);
    return number;
  };
  uint32_t adapters[KEPT], numbers[KEPT];
#pragma unroll
  for (uint32_t i = 0; i < KEPT; ++i) adapters[i] = adapter_of(i * kOrderThreads + thread);
  for (uint32_t a = thread; a < entries; a += kOrderThreads) rows_of[a] = 0;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < KEPT; ++i) numbers[i] = number_of(adapters[i], i * kOrderThreads + thread < p.rows);
  for (uint32_t at = KEPT * kOrderThreads; at < p.rows; at += kOrderThreads) {
    const uint32_t row = at + thread, number = number_of(adapter_of(row), row < p.rows);
    if (row < p.rows) p.numbers[row] = number;
  }
  __syncthreads();
  // Two adapters a thread; sums over the threads in front of it.
  constexpr uint32_t EACH = (kMostOrdered + 1) / kOrderThreads;
  uint32_t rows[EACH], own_rows = 0, own_tiles = 0;
#pragma unroll
  for (uint32_t e = 0; e < EACH; ++e) {
    rows[e] = EACH * thread + e < entries ? rows_of[EACH * thread + e] : 0;
    own_rows += rows[e];
    own_tiles += (rows[e] + 15) >> 4;
  }
  uint32_t rows_here = own_rows, tiles_here = own_tiles;
#pragma unroll
  for (int by = 1; by < 64; by *= 2) {
    const uint32_t r = __shfl_up(rows_here, by), t = __shfl_up(tiles_here, by);
    if (lane >= (uint32_t)by) {
      rows_here += r;
      tiles_here += t;
    }
  }
  if (lane == 63) {
    wave_rows[wave] = rows_here;
    wave_tiles[wave] = tiles_here;
  }
  __syncthreads();
  uint32_t row_at = rows_here - own_rows, tile_at = tiles_here - own_tiles, all_tiles = 0;
  for (uint32_t w = 0; w < kOrderThreads / 64; ++w) {
    if (w < wave) {
      row_at += wave_rows[w];
      tile_at += wave_tiles[w];
    }
    all_tiles += wave_tiles[w];
  }
#pragma unroll
  for (uint32_t e = 0; e < EACH; ++e) {
    if (EACH * thread + e < entries) {
      first_row[EACH * thread + e] = row_at;
      first_tile[EACH * thread + e] = tile_at;
    }
    row_at += rows[e];
    tile_at += (rows[e] + 15) >> 4;
  }
  __syncthreads();
  auto place = [&](uint32_t row, uint32_t a, uint32_t n) {
    if (row >= p.rows) return;
    const uint32_t tile = first_tile[a] + (n >> 4), left = rows_of[a] - n;
    p.ids[tile * 16 + (n & 15)] = row;
    if ((n & 15) == 0) p.heads[tile] = make_uint4(a, first_row[a] + n, left < 16 ? left : 16, 0);
  };
#pragma unroll
  for (uint32_t i = 0; i < KEPT; ++i) place(i * kOrderThreads + thread, adapters[i], numbers[i]);
  for (uint32_t row = KEPT * kOrderThreads + thread; row < p.rows; row += kOrderThreads) place(row, adapter_of(row), p.numbers[row]);
  for (uint32_t tile = all_tiles + thread; tile < p.tiles; tile += kOrderThreads) p.heads[tile] = make_uint4(0, 0, 0, 0);
}

extern __shared__ uint4 staged[];

// 64 x 16 bytes to LDS byte offset `lds` (of the wavefront), unseen by the compiler.
__device__ __forceinline__ void load_pieces(uint32_t lds, const uint8_t* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}

// Wavefronts of a workgroup that multiplies by `down`, and its LDS: 4 KB a wavefront for the lhs and for each 16 ranks.
template <int RT> constexpr int kWaves = RT > 2 ? 4 : 8;
template <int RT> constexpr int kDownLds = kWaves<RT> * (1 + RT) * 4096;

// Sums of 16 rows with 16 * RT ranks over a split's part of K, which the wavefronts share four chunks of 32 at a time; they meet in
// LDS, in the order of the wavefronts' numbers.
//
// A wavefront loads four chunks of sixteen rows, of the lhs and of `down`, into a part of LDS of its own, four rows a load: sixteen
// lanes have 256 bytes of a row. A row's piece c of 16 bytes lies at c ^ r, for the banks' sake. (Straight into registers neighbouring
// lanes have different rows, sixteen cache lines to a quarter of a load: 2000 rows of 12 adapters in runs, rank 64, K 4096, took 24.7 us and
// not 12.6; of one token or 64 it is 4 and 5.6 us either way, which a launch, the indices and then a load take.) What it reads: the rows
// once, `down` once for every sixteen rows.
template <Float T, int RT>
__global__ __launch_bounds__(64 * kWaves<RT>) void adapter_down_kernel(const AdapterProduct p) {
  constexpr int WAVES = kWaves<RT>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t full = p.depth >> 5, rest = p.depth & 31;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)staged + wave * ((1 + RT) * 4096);
  const uint8_t* const own = (const uint8_t*)staged + wave * ((1 + RT) * 4096) + r * 256;
  p16_v4f32* const partial = (p16_v4f32*)staged;  // [WAVES][RT][64]
  for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    // unit = (tile * slots + slot) * parts + (block of ranks * splits + split)
    const uint32_t upper = divide(unit, p.parts, p.parts_reciprocal), part = unit - upper * p.parts;
    const uint32_t tile = divide(upper, p.slots, p.slots_reciprocal), slot = upper - tile * p.slots;
    const uint32_t block = part / p.splits, split = part - block * p.splits;
    const uint32_t first_rank = block * (16 * RT);
    // (Splits begin with whole fours.)
    const uint32_t fours = (full + 3) / 4;
    const uint32_t from = (uint32_t)((uint64_t)fours * split / p.splits), to = (uint32_t)((uint64_t)fours * (split + 1) / p.splits);
    auto lhs_row = [&](uint32_t row) {
      const uint32_t panel = divide(row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
      return p.lhs.data + (int64_t)panel * p.lhs.stride0 + (row - panel * p.lhs.tile_rows) * p.lhs.row_bytes;
    };
    const int64_t lhs_step = 64 * (int64_t)p.lhs.tile_rows;
    auto no_zeros = [](uint32_t, uint32_t) {};
    of_adapters(p, tile, slot, lane, [&](uint32_t of, uint32_t same, uint32_t row, uint32_t first) {
      const uint8_t* rows[4];  // of the lane's loads
#pragma unroll
      for (int i = 0; i < 4; ++i) rows[i] = lhs_row((uint32_t)__shfl((int)row, 4 * i + g));
      auto down_row = [&](uint32_t rank) {
        return p.down + of * p.down_stride0 + (int64_t)(rank < p.rank ? rank : p.rank - 1) * p.down_stride1;
      };
      p16_v4f32 acc[RT] = {};
      for (uint32_t four = from + wave; four < to; four += WAVES) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t of_sixteen = 4 * i + g, piece = (uint32_t)r ^ of_sixteen;
          const uint32_t chunk = 4 * four + (piece >> 2) < full ? 4 * four + (piece >> 2) : full - 1;
          load_pieces(lds0 + i * 1024, rows[i] + chunk * lhs_step + (piece & 1) * p.lhs.piece1 + (piece >> 1 & 1) * p.lhs.piece2);
#pragma unroll
          for (int j = 0; j < RT; ++j)
            load_pieces(lds0 + (1 + j) * 4096 + i * 1024, down_row(first_rank + 16 * j + of_sixteen) + (int64_t)chunk * 64 + (piece & 3) * 16);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (4 * four + u >= full) continue;
          const uint32_t at = 16 * ((4 * u + g) ^ r);
          const uint4 a = *(const uint4*)(own + at);
#pragma unroll
          for (int j = 0; j < RT; ++j) acc[j] = mfma16_16<T>(*(const uint4*)(own + (1 + j) * 4096 + at), a, acc[j]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (before its place is loaded again)
      }
      // What K has behind its last whole chunk, zeros behind it.
      if (rest != 0 && split == p.splits - 1 && wave == (int)((to - from) % WAVES)) {
        const int exist = (int)rest - 8 * g;
        const uint4 a = last_piece(lhs_row(row) + full * lhs_step + (g & 1) * p.lhs.piece1 + (g >> 1) * p.lhs.piece2, exist);
#pragma unroll
        for (int j = 0; j < RT; ++j)
          acc[j] = mfma16_16<T>(last_piece(down_row(first_rank + 16 * j + r) + (int64_t)full * 64 + 16 * g, exist), a, acc[j]);
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < RT; ++j) partial[(wave * RT + j) * 64 + lane] = acc[j];
      __syncthreads();
      for (int j = wave; j < RT; j += WAVES) {
        p16_v4f32 v = partial[j * 64 + lane];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += partial[(w * RT + j) * 64 + lane];
        const uint32_t rank = first_rank + 16 * j + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = rank + e < p.rank ? v[e] : 0;  // (ranks behind the last meet zeros, and are finite)
        if ((same >> r & 1) != 0 && rank < p.pitch) *(p16_v4f32*)(p.sums + ((int64_t)split * p.lhs.rows + first + r) * p.pitch + rank) = v;
      }
      __syncthreads();
    }, no_zeros);
  }
}

// A sum in f32 as two or three 16-bit floats that add up to it: bf16 takes the 24 bits of its mantissa eight at a time, exactly; f16
// the nearest, then the nearest to what that leaves, which is 2^-24 of it off at most, a sum having been brought into f16's range with
// the others of its row first (`unit`, a power of two).
template <Float T> constexpr int kSumParts = T == Float::kF16 ? 2 : 3;
template <Float T>
__device__ __forceinline__ void split_sum(float v, uint16_t (&part)[3]) {
  if constexpr (T == Float::kBf16) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const uint32_t bits = __builtin_bit_cast(uint32_t, v);
      part[i] = (uint16_t)(bits >> 16);
      const float rest = v - __builtin_bit_cast(float, bits & 0xFFFF0000u);
      v = rest == rest ? rest : 0;  // (of an infinity nothing is left)
    }
  } else {
    part[0] = mx_narrow<T>(v);
    const float rest = v - mx_widen<T>(part[0]);
    part[1] = mx_narrow<T>(rest == rest ? rest : 0);
    part[2] = 0;
  }
}

// 16 rows times 16 * F columns a wavefront and turn. The rank sums are multiplied as 16-bit floats of which they are the sums, with
// v_mfma_f32_16x16x32: of up to 16 ranks (HALF) two parts are one instruction's 32, lane (r, g) with eight from 8 (g & 1) on, of row r
// of the sums and of column r. Otherwise a part of 32 CHUNKS ranks is CHUNKS instructions. (On v_mfma_f32_16x16x4, with `up` widened to
// f32, 64 rows of 64 adapters x 14336, rank 16, took 17.5 us and not 14.0, of which the matrix instructions 3 and the widening and what
// runs in front of a wavefront's first load most of the rest.)
//
// MANY: more ranks than that, whose sums are taken anew in every turn.
//
// The splits' sums are added on their way into LDS, where a workgroup's four wavefronts have them from; only those of rows that have the
// adapter are read. A turn's `up` is asked for when the one before it has been multiplied, and its results when that one's are stored.
//
// 64 rows of 64 adapters x 14336, rank 16, take 14.0 us, 36 MB at 2.6 TB/s: a wavefront waits for its index, then for its sums, then has
// three turns to make up for it. 2000 rows in runs x 4096, rank 64, take 20 to 23 us, of which the f32
// results, read and written, are 65 MB. Results turned in LDS, so that four lanes have 64 bytes of a row, gained 4 % there and lost 10 % here.
//
// FAST: columns come in whole sixteens that lie next to each other, aligned, and an adapter's row of `up` in whole eights, aligned. (As
// two branches of one kernel the slow one's registers halved the number of wavefronts on a compute unit.) Without it results go one by
// one, also where only `up` is in the way: both launches of 64 rows of 64 adapters x 14336 x 4096 into f32 take 54 us with rank 4, 62
// with 7 and 69 with 30, where 8 takes 19, 16 20 and 32 24; of 2000 rows in runs x 4096 x 4096 50, 52 and 57, and 26, 27 and 31.
template <Float T, Float OUT, bool HALF, int CHUNKS, int F, bool FAST, bool MANY>
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterProduct p) {
  constexpr int SIZE = OUT == Float::kF32 ? 4 : 2, GROUP = HALF ? 16 : 32 * CHUNKS, PITCH = GROUP + 4;  // (rows 4 banks apart)
  constexpr int PARTS = HALF ? (kSumParts<T> + 1) / 2 : kSumParts<T> * CHUNKS;  // operands of 32 values
  __shared__ float sums[16 * PITCH];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t own_rank = HALF ? 8 * (g & 1) : 8 * g;  // of a chunk's, the lane's first
  for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    // unit = (tile * slots + slot) * parts + block of columns
    const uint32_t upper = divide(unit, p.parts, p.parts_reciprocal), part = unit - upper * p.parts;
    const uint32_t tile = divide(upper, p.slots, p.slots_reciprocal), slot = upper - tile * p.slots;
    const uint32_t first_col = (part * 4 + wave) * (16 * F * p.turns);
    const uint32_t end_col = first_col + 16 * F * p.turns < p.cols ? first_col + 16 * F * p.turns : p.cols;
    // Four results of a row, of the fragment at `col`, as they lie in memory.
    typedef uint32_t Words __attribute__((ext_vector_type(SIZE)));
    auto results_of = [&](uint32_t row) { return p.out + (layout_row(p.out_at, row) + 4 * g) * SIZE; };
    auto four_at = [&](uint8_t* results, uint32_t col) {
      return (Words*)__builtin_assume_aligned(results + layout_col(p.out_at, col) * SIZE, 4 * SIZE);
    };
    auto store_one_by_one = [&](uint32_t row, uint32_t from, p16_v4f32 v) {
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        const uint32_t col = from + 4 * g + e;
        if (col >= p.cols) continue;
        const int64_t at = layout_row(p.out_at, row) + layout_col(p.out_at, col);
        const float x = v[e] + (p.accumulate ? element<OUT>(p.out, at) : 0);
        if constexpr (OUT == Float::kF32) ((float*)p.out)[at] = x;
        else ((uint16_t*)p.out)[at] = mx_narrow<OUT>(x);
      }
    };
    auto add = [&](uint32_t of, uint32_t same, uint32_t row, uint32_t first) {
      const bool mine = (same >> r & 1) != 0;
      uint8_t* const results = results_of(row);
      const uint8_t* const up = p.up + of * p.up_stride0;
      uint4 w[CHUNKS][F], t[PARTS];
      Words old[F] = {};
      float unit_of_row = 1;
      auto load_up = [&](uint4 (&to)[CHUNKS][F], uint32_t col0, uint32_t rank0) {
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const uint32_t col = col0 + 16 * f + r;
          const uint32_t at = (col < p.cols ? col : p.cols - 1) * (uint32_t)p.up_stride1 + 2 * (rank0 + own_rank);
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c) {
            const int exist = (int)p.rank - (int)(rank0 + 32 * c + own_rank);
            to[c][f] = make_uint4(0, 0, 0, 0);
            if constexpr (FAST) {
              if (exist > 0) to[c][f] = *(const uint4*)(up + at + 64 * c);
            } else {
              to[c][f] = last_piece_anywhere(up + at + 64 * c, exist);
            }
          }
        }
      };
      auto load_old = [&](Words (&to)[F], uint32_t col0) {
#pragma unroll
        for (int f = 0; f < F; ++f)
          if (FAST && p.accumulate && mine && col0 + 16 * f < end_col) to[f] = *four_at(results, col0 + 16 * f);
      };
      // The sums of ranks from rank0 on, as operands.
      auto take_sums = [&](uint32_t rank0) {
        // Four ranks of a row each thread. (The pitch is a multiple of 32 ranks; what lies behind it is not there.)
#pragma unroll
        for (int n = 0; n < (16 * GROUP / 4 + 255) / 256; ++n) {
          const uint32_t number = threadIdx.x + 256 * n, of_row = number / (GROUP / 4), four = 4 * (number % (GROUP / 4));
          if (of_row >= 16) continue;
          p16_v4f32 v = {0, 0, 0, 0};
          if ((same >> of_row & 1) != 0 && rank0 + four < p.pitch) {
            const float* at = p.sums + (int64_t)(first + of_row) * p.pitch + rank0 + four;
            const int64_t split = (int64_t)p.lhs.rows * p.pitch;
            for (uint32_t s = 0; s < p.splits; s += 4) {  // (four under way at a time)
              p16_v4f32 part[4];
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) part[i] = s + i < p.splits ? *(const p16_v4f32*)(at + (s + i) * split) : p16_v4f32{0, 0, 0, 0};
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) v += part[i];
            }
          }
          *(p16_v4f32*)(sums + of_row * PITCH + four) = v;
        }
        __syncthreads();
        float v[CHUNKS][8], largest = 0;
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const p16_v4f32 four = *(const p16_v4f32*)(sums + r * PITCH + 32 * c + own_rank + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              v[c][e + i] = four[i];
              const float size = __builtin_fabsf(four[i]);
              largest = size < __builtin_inff() && size > largest ? size : largest;
            }
          }
        __syncthreads();
        if constexpr (T == Float::kF16) {
          // To below 2^15, with the row's other ranks that are finite. (Zeros, and what is not finite, stay what they are.)
          largest = __builtin_fmaxf(largest, __shfl_xor(largest, 16));
          largest = __builtin_fmaxf(largest, __shfl_xor(largest, 32));
          const int field = (int)(__builtin_bit_cast(uint32_t, largest) >> 23);
          const int by = field < 24 ? 0 : 127 + 14 - field;
          unit_of_row = ldexpf(1.0f, -by);
#pragma unroll
          for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[c][e] = ldexpf(v[c][e], by);
        }
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
          uint32_t words[3][4];
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            uint16_t even[3], odd[3];
            split_sum<T>(v[c][e], even);
            split_sum<T>(v[c][e + 1], odd);
#pragma unroll
            for (int i = 0; i < 3; ++i) words[i][e / 2] = (uint32_t)even[i] | (uint32_t)odd[i] << 16;
          }
          auto operand = [&](int i) { return make_uint4(words[i][0], words[i][1], words[i][2], words[i][3]); };
          if constexpr (HALF) {
            const uint4 a = operand(0), b = operand(1), d = operand(2), none = make_uint4(0, 0, 0, 0);
            t[0] = g < 2 ? a : b;
            if constexpr (PARTS > 1) t[1] = g < 2 ? d : none;
          } else {
#pragma unroll
            for (int i = 0; i < kSumParts<T>; ++i) t[c * kSumParts<T> + i] = operand(i);
          }
        }
      };
      p16_v4f32 acc[F];
      auto multiply = [&](const uint4 (&by)[CHUNKS][F]) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i)
#pragma unroll
          for (int f = 0; f < F; ++f) acc[f] = mfma16_16<T>(by[HALF ? 0 : i / kSumParts<T>][f], t[i], acc[f]);
      };
      load_up(w, first_col < p.cols ? first_col : 0, 0);
      load_old(old, first_col);
      const float scale = p.scales ? p.scales[of] : 1;
      if constexpr (!MANY) take_sums(0);
      // (Everyone goes round as often, for the sums' sake.)
      for (uint32_t turn = 0; turn < p.turns; ++turn) {
        const uint32_t col0 = first_col + 16 * F * turn, next_col = col0 + 16 * F < end_col ? col0 + 16 * F : 0;
#pragma unroll
        for (int f = 0; f < F; ++f) acc[f] = p16_v4f32{0, 0, 0, 0};
        if constexpr (MANY) {
          p16_v4f32 total[F] = {};
          for (uint32_t rank0 = 0; rank0 < p.rank; rank0 += GROUP) {
            take_sums(rank0);
            multiply(w);
            const bool last = rank0 + GROUP >= p.rank;
            load_up(w, last ? next_col : col0 < p.cols ? col0 : 0, last ? 0 : rank0 + GROUP);
#pragma unroll
            for (int f = 0; f < F; ++f) {
              total[f] += acc[f] * unit_of_row;
              acc[f] = p16_v4f32{0, 0, 0, 0};
            }
          }
#pragma unroll
          for (int f = 0; f < F; ++f) acc[f] = total[f];
        } else {
          multiply(w);
          if (turn + 1 < p.turns) load_up(w, next_col, 0);
        }
        if (mine) {
#pragma unroll
          for (int f = 0; f < F; ++f) {
            const uint32_t col = col0 + 16 * f;
            if (col >= end_col) continue;
            p16_v4f32 v = acc[f] * (MANY ? scale : unit_of_row * scale);
            if constexpr (!FAST) {
              store_one_by_one(row, col, v);
            } else if constexpr (OUT == Float::kF32) {
              v += __builtin_bit_cast(p16_v4f32, old[f]);
              *four_at(results, col) = __builtin_bit_cast(Words, v);
            } else {
              float x[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) x[e] = v[e] + mx_widen<OUT>((uint16_t)(old[f][e / 2] >> (16 * (e & 1))));
              *four_at(results, col) = Words{mx_narrow_pair<OUT>(x[0], x[1]), mx_narrow_pair<OUT>(x[2], x[3])};
            }
          }
          if (turn + 1 < p.turns) load_old(old, col0 + 16 * F);
        }
      }
    };
    of_adapters(p, tile, slot, lane, add, [&](uint32_t without, uint32_t row) {
      if (p.accumulate || (without >> r & 1) == 0) return;
      uint8_t* const results = results_of(row);
      for (uint32_t col = first_col; col < end_col; col += 16) {
        if constexpr (!FAST) store_one_by_one(row, col, p16_v4f32{0, 0, 0, 0});
        else *four_at(results, col) = Words(0);
      }
    });
  }
}

// Whether rows are put in order, and tiles: what adapters of sixteen rows in any order have to be read, less what each adapter's own tiles
// have, is 16 MiB and more. Rows mixed at random then take what rows in runs do and 1 to 3 us for the launch (2000 x 4096 x 4096, 12 adapters, rank 64,
// 159 -> 40 us, 256 x 8192 x 4096, 40 adapters, rank 32, 35 -> 19, 4000 x 11008 x 4096, 30 adapters, rank 32, 487 -> 137); rows that come in
// runs, and no host knows whether they do, 34 -> 35, 23 -> 17 and 115 -> 108. In 40 problems of 5 to 100 MiB mixed rows take 11 us less in the
// mean from 16 MiB on, and rows in runs 0.2 more; below it is 0.7 less and 1.4 more.
struct Tiles { int64_t most; bool ordered; };
Tiles tiles_of(int64_t rows, int64_t count, int64_t depth, int64_t cols, int64_t rank) {
  const int64_t sixteens = (rows + 15) / 16, own = rows / 16 + (count + 1 < rows ? count + 1 : rows);
  if (rows <= 16 || rows > 65536 || count < 2 || count > kMostOrdered) return {sixteens, false};
  // (Of `count` adapters sixteen rows have count (1 - (1 - 1 / count)^16) in the mean.)
  double others = 1;
  for (int i = 0; i < 16; ++i) others *= 1 - 1 / (double)count;
  const double saved = (double)sixteens * (double)count * (1 - others) - (double)own;
  if (saved * 2 * (double)rank * (double)(depth + cols) < (double)(16 << 20)) return {sixteens, false};
  return {own, true};
}
// How many parts K is split into: as many as leave every wavefront four chunks, while two workgroups come to a compute unit, which its LDS
// holds of 16 ranks (64 KiB) and of more than 32 (80), but of 17 to 32 (96) one. (2000 rows, rank 64, K 4096: 3 parts 14.9 us, 4 12.6, 6 15.3.)
uint32_t splits_of(int64_t rows_of_tiles, int64_t depth, int64_t rank) {
  const int waves = rank > 32 ? kWaves<kFragments> : kWaves<1>;
  const int64_t tiles = rows_of_tiles * ((rank + 16 * kFragments - 1) / (16 * kFragments));
  const int64_t most = depth / 32 / (4 * waves), wanted = 512 / tiles;
  const int64_t s = most < wanted ? most : wanted;
  return (uint32_t)(s < 1 ? 1 : s);
}
int64_t pitch_of(int64_t rank) { return (rank + 31) / 32 * 32; }
// (Fewer than 2^31 rows, and 2^15 ranks; few splits where there are many.)
int64_t sums_bytes(int64_t rows, int64_t rank, int64_t splits) { return (rows * pitch_of(rank) * 4 * splits + 255) / 256 * 256; }

bool multiple(const void* p, int64_t to) { return (uintptr_t)p % to == 0; }

// Fragments of columns of a wavefront's turn, and turns: as many as leave some 4096 wavefronts, sixteen to a compute unit. (Both launches
// with 2048, 4096 and 8192 wavefronts: 64 rows of 64 adapters x 14336, rank 16, 18.0, 19.3, 24.4 us; 2000 rows of 12 in runs x 4096, rank 64,
// 37.9, 33.7, 33.9; 256 of 40 x 8192, rank 32, 38.2, 34.0, 36.7; 40 of 16 x 11008, rank 16, 13.7, 13.4, 15.0.)
int up_fragments(int64_t rank) { return rank <= 32 ? 4 : 2; }
uint32_t turns_of(int64_t tiles, int64_t slots, int64_t cols, int64_t rank) {
  const int64_t across = (cols + 16 * up_fragments(rank) - 1) / (16 * up_fragments(rank)), t = tiles * slots * across / 4096;
  return (uint32_t)(t < 1 ? 1 : t > 8 ? 8 : t);
}
int64_t column_parts(const AdapterProduct& p) {
  const int64_t of_group = 64 * (int64_t)up_fragments(p.rank) * p.turns;
  return (p.cols + of_group - 1) / of_group;
}

// The problem as the kernels on the matrix pipe take it; false: they do not.
bool as_product(const AdapterArgs& a, AdapterProduct* p) {
  const int64_t depth = a.K * a.K0, cols = a.N * a.N0;
  if (a.count == 0 || depth > 0x7FFFFFFF || cols > 0x7FFFFFFF - 512) return false;
  if (!as_operand16(a.lhs, a.lhs_stride0, a.M, a.M0, a.K, a.K0, &p->lhs)) return false;
  if (!multiple(a.down, 16) || (a.count > 1 && a.down_stride0 % 8 != 0) || (a.rank > 1 && a.down_stride1 % 8 != 0)) return false;
  const int64_t rows = a.M * a.M0;
  const Tiles t = tiles_of(rows, a.count, depth, cols, a.rank);
  p->tiles = (uint32_t)t.most;
  p->down = a.down; p->up = a.up;
  p->down_stride0 = 2 * a.down_stride0; p->down_stride1 = 2 * a.down_stride1;
  p->up_stride0 = 2 * a.up_stride0; p->up_stride1 = 2 * a.up_stride1;
  p->index = a.index;
  p->scales = a.scales;
  p->sums = (float*)a.workspace;
  p->out = a.out;
  p->out_at = layout_of(a.out_stride0, a.M0, a.N, a.N0);
  p->out_type = a.out_type;
  p->depth = (uint32_t)depth; p->rank = (uint32_t)a.rank; p->count = (uint32_t)a.count; p->cols = (uint32_t)cols;
  p->pitch = (uint32_t)pitch_of(a.rank);
  p->splits = splits_of(t.most, depth, a.rank);
  const int64_t sums = sums_bytes(rows, a.rank, p->splits);
  p->heads = t.ordered ? (const uint4*)(a.workspace + sums) : nullptr;
  p->ids = t.ordered ? (const uint32_t*)(a.workspace + sums + 16 * t.most) : nullptr;
  p->accumulate = a.accumulate;
  const int e = float_bytes(a.out_type);
  p->runs = runs_of(p->out_at, a.out, a.M, e, 16, 4 * e);
  // (32 bits from an adapter's start to a column of `up`.)
  if (p->up_stride1 > (1ll << 31) / cols) return false;
  // Adapters of a tile side by side where there are few tiles.
  const int64_t slots = t.ordered ? 1 : 128 / t.most, most = a.count < 16 ? a.count : 16;
  p->slots = (uint32_t)(slots < 1 ? 1 : slots > most ? most : slots);
  p->slots_reciprocal = reciprocal_of(p->slots);
  p->turns = turns_of(t.most, p->slots, cols, a.rank);
  return true;
}

// One launch over tiles * slots * parts pieces of work.
hipError_t launch_units(void (*kernel)(const AdapterProduct), AdapterProduct p, int64_t parts, unsigned threads, unsigned lds, hipStream_t stream) {
  p.parts = (uint32_t)parts;
  p.parts_reciprocal = reciprocal_of(p.parts);
  p.units = (uint32_t)(p.tiles * (int64_t)p.slots * parts);
  return launch_kernel(kernel, p.units < (1u << 22) ? p.units : 1u << 22, threads, lds, stream, p);
}

template <Float T, int RT>
hipError_t launch_down_of(const AdapterProduct& p, int64_t parts, hipStream_t stream) {
  if (kDownLds<RT> > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute((const void*)adapter_down_kernel<T, RT>, hipFuncAttributeMaxDynamicSharedMemorySize, kDownLds<RT>);
    if (e != hipSuccess) return e;
  }
  return launch_units(adapter_down_kernel<T, RT>, p, parts, 64 * kWaves<RT>, kDownLds<RT>, stream);
}
template <Float T>
hipError_t launch_down(const AdapterProduct& p, hipStream_t stream) {
  const int64_t fragments = (p.rank + 15) / 16;
  if (fragments == 1) return launch_down_of<T, 1>(p, p.splits, stream);
  if (fragments == 2) return launch_down_of<T, 2>(p, p.splits, stream);
  return launch_down_of<T, kFragments>(p, (fragments + kFragments - 1) / kFragments * p.splits, stream);
}

template <Float T, Float OUT, bool FAST>
hipError_t launch_up_of(const AdapterProduct& p, int64_t parts, hipStream_t stream) {
  if (p.rank <= 16) return launch_units(adapter_up_kernel<T, OUT, true, 1, 4, FAST, false>, p, parts, 256, 0, stream);
  if (p.rank <= 32) return launch_units(adapter_up_kernel<T, OUT, false, 1, 4, FAST, false>, p, parts, 256, 0, stream);
  if (p.rank <= 64) return launch_units(adapter_up_kernel<T, OUT, false, 2, 2, FAST, false>, p, parts, 256, 0, stream);
  return launch_units(adapter_up_kernel<T, OUT, false, 2, 2, FAST, true>, p, parts, 256, 0, stream);
}
template <Float T>
hipError_t launch_up(const AdapterProduct& p, hipStream_t stream) {
  const int64_t parts = column_parts(p);
  const bool fast = p.runs && p.cols % 16 == 0 && p.rank % 8 == 0 && multiple(p.up, 16) && (p.count <= 1 || p.up_stride0 % 16 == 0) &&
                    (p.cols <= 1 || p.up_stride1 % 16 == 0);
  if (p.out_type == Float::kF32) return fast ? launch_up_of<T, Float::kF32, true>(p, parts, stream) : launch_up_of<T, Float::kF32, false>(p, parts, stream);
  return fast ? launch_up_of<T, T, true>(p, parts, stream) : launch_up_of<T, T, false>(p, parts, stream);
}

// Whether the pieces of work of both launches are fewer than 2^31.
bool countable(const AdapterProduct& p) {
  const int64_t blocks = (p.rank + 15) / 16, most = (1ll << 31) / ((int64_t)p.tiles * p.slots);
  return blocks * p.splits < most && column_parts(p) < most;
}

}  // namespace

int64_t adapter_workspace(const AdapterArgs& a) {
  if (a.count == 0) return 0;
  const int64_t rows = a.M * a.M0, depth = a.K * a.K0, cols = a.N * a.N0;
  const Tiles t = tiles_of(rows, a.count, depth, cols, a.rank);
  // The rank sums; of rows in order 16 bytes for a tile's head and 64 for its rows.
  return sums_bytes(rows, a.rank, splits_of(t.most, depth, a.rank)) + (t.ordered ? (80 * t.most + 255) / 256 * 256 : 0);
}

hipError_t launch_adapter_mmt4d(const AdapterArgs& a, hipStream_t stream, const char** name) {
  AdapterProduct p;
  if (as_product(a, &p) && countable(p)) {
    *name = "adapter_mmt4d";
    const bool f16 = a.type == Float::kF16;
    if (p.heads) {
      const OrderArgs o = {p.index, (uint4*)p.heads, (uint32_t*)p.ids, (uint32_t*)p.sums, p.lhs.rows, p.count, p.tiles};
      const hipError_t e = launch_kernel(adapter_order_kernel, 1, kOrderThreads, 0, stream, o);
      if (e != hipSuccess) return e;
    }
    const hipError_t e = f16 ? launch_down<Float::kF16>(p, stream) : launch_down<Float::kBf16>(p, stream);
    return e != hipSuccess ? e : f16 ? launch_up<Float::kF16>(p, stream) : launch_up<Float::kBf16>(p, stream);
  }
  const int64_t rows = a.M * a.M0;
  *name = "adapter_mmt4d_generic";
  if (a.count > 0) {
    const hipError_t e = launch_over(adapter_down_generic<Float::kF16>, adapter_down_generic<Float::kBf16>, a, rows * a.rank, stream);
    if (e != hipSuccess) return e;
  }
  return launch_over(adapter_up_generic<Float::kF16>, adapter_up_generic<Float::kBf16>, a, rows * a.N * a.N0, stream);
}

}  // namespace uk
