// Microscaled products of few rows: the rhs (the weights) is streamed from memory straight into registers, once, and K is
// split over the wavefronts of a workgroup.
#include <type_traits>

#include "mx_mmt4d.h"

namespace uk {
namespace {

// Four chunks' scales of sixteen rows: lane (g, r) has loaded those of row r in chunk g, and gets block g's in chunk u as byte u,
// where the matrix instruction picks it from. One load for what takes four if every lane loads its own bytes.
__device__ __forceinline__ uint32_t scales_of_blocks(uint32_t loaded, int g) {
  typedef uint32_t v2u32 __attribute__((ext_vector_type(2)));
  const v2u32 halves = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane32_swap(loaded, loaded, false, false));
  const v2u32 low = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane16_swap(halves[0], halves[0], false, false));
  const v2u32 high = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane16_swap(halves[1], halves[1], false, false));
  const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t)g;  // byte g of the second operand, then of the first
  return __builtin_amdgcn_perm(low[1], low[0], pick) | __builtin_amdgcn_perm(high[1], high[0], pick) << 16;
}

constexpr int kWaves = 8;

extern __shared__ uint4 few_lds[];

__device__ __forceinline__ void load_pieces(uint32_t lds, uint32_t offset, const uint8_t* base) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// At most the last N loads of the wavefront are still under way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// A workgroup multiplies 16 * MT rows of the lhs with 16 * NT of the rhs; its wavefronts take four chunks of 128 of K in turn, and
// add their sums through LDS in the order of their numbers. A chunk is loaded again as soon as it is multiplied. Rows beyond
// the last are read as the last one and not stored.
//
// STAGED: the lhs goes through LDS, a wavefront's own part of it, where a row's pieces are exchanged among themselves for the
// banks' sake. Straight into registers a load's neighbouring lanes have 16 rows, 16 cache lines; to LDS four (eight) neighbouring
// lanes have one row. The best staged shape against the best without: 32 rows x 4096 columns x 14336 in 8.1 us (9.3; 8-bit lhs 9.5,
// 13.0), 128 x 4096 x 4096 in 7.4 (9.5; 8.9, 12.2), 128 x 4096 x 14336 in 14.3 (23.7; 17.9, 31.6).
template <int LBITS, int MT, int NT, bool STREAM, bool STAGED>
__global__ __launch_bounds__(64 * kWaves) void mx_mmt4d_few_kernel(const MxProduct p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t first_col = blockIdx.x * (16 * NT), first_row = blockIdx.y * (16 * MT);
  constexpr int ROW = 16 * LBITS, PIECES = ROW / 16, ROWS_OF_LOAD = 64 / PIECES;  // bytes of a row's chunk
  constexpr int CHUNK = MT * 16 * ROW, LOADS = CHUNK / 1024;                      // the lhs's, of a wavefront

  const uint8_t *rhs[NT], *rhs_scales[NT], *lhs[MT], *lhs_scales[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const uint32_t col = first_col + 16 * j + r, row = col < p.rhs.rows ? col : p.rhs.rows - 1;
    rhs[j] = p.rhs.codes + mx_row_codes<4>(p.rhs, row) + 16 * g;
    rhs_scales[j] = p.rhs.scales + mx_row_scales(p.rhs, row);
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const uint32_t at = first_row + 16 * i + r, row = at < p.lhs.rows ? at : p.lhs.rows - 1;
    lhs[i] = p.lhs.codes + mx_row_codes<LBITS>(p.lhs, row) + 16 * g;
    lhs_scales[i] = p.lhs.scales + mx_row_scales(p.lhs, row);
  }
  const int64_t rhs_step = 64 * (int64_t)p.rhs.tile_rows, lhs_step = ROW * (int64_t)p.lhs.tile_rows;
  const int64_t rhs_scales_step = 4 * (int64_t)p.rhs.tile_rows, lhs_scales_step = 4 * (int64_t)p.lhs.tile_rows;
  // Staged: load n of a chunk has rows n * ROWS_OF_LOAD + lane / PIECES; a row's piece c lies at c ^ exchanged(row).
  const uint32_t first_panel = divide(first_row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
  const uint8_t* const lhs_base = p.lhs.codes + (int64_t)first_panel * p.lhs.stride0;
  uint32_t lhs_from[STAGED ? LOADS : 1];
  auto exchanged = [](uint32_t row) { return LBITS == 4 ? ((row >> 2) & 3) ^ (row & 2) : ((row >> 1) & 7) ^ ((row & 1) << 2); };
  if constexpr (STAGED) {
#pragma unroll
    for (int n = 0; n < LOADS; ++n) {
      const uint32_t at = n * ROWS_OF_LOAD + lane / PIECES;
      const uint32_t row = first_row + at < p.lhs.rows ? first_row + at : p.lhs.rows - 1;
      const uint32_t panel = divide(row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
      lhs_from[n] = (uint32_t)((panel - first_panel) * p.lhs.stride0) + (row - panel * p.lhs.tile_rows) * ROW +
                    16 * ((lane % PIECES) ^ exchanged(at));
    }
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)few_lds + wave * (4 * CHUNK);
  const uint8_t* const staged = (const uint8_t*)few_lds + wave * (4 * CHUNK) + r * ROW;

  mx_v4f32 acc[MT][NT] = {};
  MxFragment<4> b[4][NT];
  MxFragment<LBITS> a[STAGED ? 1 : 4][MT];
  uint32_t bs[NT], as[MT], b_loaded[NT], a_loaded[MT];
  auto load_scales = [&](uint32_t first) {
    const uint32_t chunk = first + g < p.chunks ? first + g : p.chunks - 1;
#pragma unroll
    for (int j = 0; j < NT; ++j) b_loaded[j] = *(const uint32_t*)(rhs_scales[j] + chunk * rhs_scales_step);
#pragma unroll
    for (int i = 0; i < MT; ++i) a_loaded[i] = *(const uint32_t*)(lhs_scales[i] + chunk * lhs_scales_step);
  };
  auto take_scales = [&] {
#pragma unroll
    for (int j = 0; j < NT; ++j) bs[j] = scales_of_blocks(b_loaded[j], g);
#pragma unroll
    for (int i = 0; i < MT; ++i) as[i] = scales_of_blocks(a_loaded[i], g);
  };
  auto load = [&](auto number, uint32_t first) {
    constexpr int U = decltype(number)::value;
    const uint32_t chunk = first + U < p.chunks ? first + U : p.chunks - 1;
    if constexpr (STAGED) {
#pragma unroll
      for (int n = 0; n < LOADS; ++n) load_pieces(lds0 + U * CHUNK + n * 1024, lhs_from[n], lhs_base + chunk * lhs_step);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint8_t* from = rhs[j] + chunk * rhs_step;
      if constexpr (STREAM) {
        const mx_v4f32 v = __builtin_nontemporal_load((const mx_v4f32*)from);
        __builtin_memcpy(b[U][j].w, &v, 16);
      } else {
        __builtin_memcpy(b[U][j].w, __builtin_assume_aligned(from, 16), 16);
      }
    }
    if constexpr (!STAGED) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint8_t* from = lhs[i] + chunk * lhs_step;
        __builtin_memcpy(a[U][i].w, __builtin_assume_aligned(from, 16), 16);
        if constexpr (LBITS == 8) __builtin_memcpy(a[U][i].w + 4, __builtin_assume_aligned(from + 64, 16), 16);
      }
    }
  };
  auto multiply = [&](auto number) {
    constexpr int U = decltype(number)::value, HELD = STAGED ? 0 : U;
    if constexpr (STAGED) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint8_t* const row = staged + U * CHUNK + i * 16 * ROW;
        *(uint4*)a[0][i].w = *(const uint4*)(row + 16 * (g ^ exchanged(r)));
        if constexpr (LBITS == 8) *(uint4*)(a[0][i].w + 4) = *(const uint4*)(row + 16 * ((4 + g) ^ exchanged(r)));
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (LBITS == 8) {
        MxFragment<8> high, low;
        mx_split(a[HELD][i], high, low);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          acc[i][j] = mx_mfma_16<4, 8, U>(b[U][j], bs[j], high, as[i], acc[i][j]);
          acc[i][j] = mx_mfma_16<4, 8, U>(b[U][j], bs[j], low, as[i], acc[i][j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = mx_mfma_16<4, LBITS, U>(b[U][j], bs[j], a[HELD][i], as[i], acc[i][j]);
      }
    }
    // (What has been read from LDS has been read before its place is loaded again.)
    if constexpr (STAGED) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  auto of_four = [](auto f) {
    f(std::integral_constant<int, 0>{});
    f(std::integral_constant<int, 1>{});
    f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, 3>{});
  };

  // Four chunks from `first` on; where they are not all there, the last four of K, of which those before `first` are skipped.
  const uint32_t fours = (p.chunks + 3) / 4;
  auto begin = [&](uint32_t four) {
    const uint32_t last = p.chunks > 4 ? p.chunks - 4 : 0;
    return 4 * four < last ? 4 * four : last;
  };
  if ((uint32_t)wave < fours) {
    uint32_t four = wave, first = begin(four);
    load_scales(first);
    of_four([&](auto u) { load(u, first); });
    for (; four + kWaves < fours; four += kWaves) {  // (all of four chunks)
      take_scales();
      first = begin(four + kWaves);
      load_scales(first);
      of_four([&](auto u) {
        // (Behind a chunk's loads come three chunks', and of each only those to LDS are counted on: the compiler may leave out
        // or join its own.)
        if constexpr (STAGED) wait_loads<3 * LOADS>();
        multiply(u);
        load(u, first);
      });
    }
    take_scales();
    const uint32_t skip = 4 * four - first, end = p.chunks - first;
    if constexpr (STAGED) wait_loads<0>();
    of_four([&](auto u) {
      constexpr uint32_t U = decltype(u)::value;
      if (U >= skip && U < end) multiply(u);
    });
  }

  mx_v4f32* const partial = (mx_v4f32*)few_lds;  // [kWaves][MT * NT][64]
  if constexpr (STAGED) __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) partial[(wave * (MT * NT) + i * NT + j) * 64 + lane] = acc[i][j];
  __syncthreads();
  for (int f = wave; f < MT * NT; f += kWaves) {
    mx_v4f32 v = partial[f * 64 + lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v += partial[(w * (MT * NT) + f) * 64 + lane];
    const uint32_t row = first_row + 16 * (f / NT) + r, col = first_col + 16 * (f % NT) + 4 * g;
    if (row < p.lhs.rows) mx_store_four(p, mx_out_row(p, row), col, v);
  }
}

// Up to 16 rows against a rhs from memory, K up to 8192: a workgroup, one on a compute unit, keeps the lhs in registers, a wavefront
// its part of K (FOURS times four chunks, the last one over and over where K ends before them), and goes through panels of 16 rows of the rhs, AHEAD of which are under way. Sums of
// PANELS panels at a time meet in LDS, in the order of the wavefronts' numbers.
//
// Above, every workgroup loads the lhs anew, next to as many bytes of the rhs with 8-bit codes, and these loads delay the stream: 16
// rows x 28672 x 8192 take 22.7 us (4 bits) and 25.9 (8 bits), one row of 4 bits 20.4; here 21.5 (5.8 TB/s) and 25.1, of which what
// the 8-bit codes' two parts take (21.8 without). Of two workgroups on a unit, with 128 registers a lane, the second's start cost
// what it gained (4 bits). A rhs of less than 48 MiB, which the caches may hold, goes faster above: 16 x 14336 x 4096 7.1 us, here 7.7
// (8 bits 7.9, 11.0). A row-major rhs gains more: 16 x 28672 x 8192 in 26.9 us (37.8; 8 bits 30.0, 38.5).
template <int LBITS, int FOURS>
__global__ __launch_bounds__(64 * kWaves) void mx_mmt4d_resident_kernel(const MxProduct p) {
  static_assert(4 * kWaves * 2 == kMxResidentChunks, "two fours at most");
  constexpr int PANELS = 4, AHEAD = 4 / FOURS;
  constexpr int ROW = 16 * LBITS, PIECES = ROW / 16, ROWS_OF_LOAD = 64 / PIECES, CHUNK = 16 * ROW, LOADS = CHUNK / 1024;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t panels = (p.rhs.rows + 15) / 16;
  const uint32_t first = (uint32_t)((uint64_t)blockIdx.x * panels / gridDim.x),
                 end = (uint32_t)((uint64_t)(blockIdx.x + 1) * panels / gridDim.x);

  MxFragment<4> b[AHEAD][FOURS][4];
  MxFragment<LBITS> a[FOURS][4];
  uint32_t as[FOURS], b_loaded[AHEAD][FOURS];
  auto chunk_of = [&](int f, int u) { return (uint32_t)(4 * (wave + f * kWaves) + u); };
  auto inside = [&](uint32_t chunk) { return chunk < p.chunks ? chunk : p.chunks - 1; };
  // Offsets of a lane from the panel of tiles that the workgroup begins in.
  const uint32_t first_panel = divide(16 * first, p.rhs.tile_rows, p.rhs.tile_reciprocal);
  const uint8_t* const codes = p.rhs.codes + first_panel * p.rhs.stride0;
  const uint8_t* const scales = p.rhs.scales + first_panel * p.rhs.scales_stride0;
  uint32_t codes_at, scales_at;
  auto to_panel = [&](uint32_t panel) {
    const uint32_t at = 16 * panel + r, row = at < p.rhs.rows ? at : p.rhs.rows - 1;
    const uint32_t of = divide(row, p.rhs.tile_rows, p.rhs.tile_reciprocal), in = row - of * p.rhs.tile_rows;
    codes_at = (uint32_t)((of - first_panel) * p.rhs.stride0) + in * 64 + 16 * g;
    scales_at = (uint32_t)((of - first_panel) * p.rhs.scales_stride0) + in * 4;
  };
  auto load = [&](int d, int f, int u) {
    const uint8_t* const from = codes + inside(chunk_of(f, u)) * (64 * (int64_t)p.rhs.tile_rows);
    const mx_v4f32 v = __builtin_nontemporal_load((const mx_v4f32*)(from + codes_at));
    __builtin_memcpy(b[d][f][u].w, &v, 16);
  };
  auto load_scales = [&](int d, int f) {
    b_loaded[d][f] = *(const uint32_t*)(scales + scales_at + inside(chunk_of(f, 0) + g) * (4 * (int64_t)p.rhs.tile_rows));
  };

  // The lhs, by way of LDS (as above). Chunks behind the last are zeros with a scale of one.
  auto exchanged = [](uint32_t row) { return LBITS == 4 ? ((row >> 2) & 3) ^ (row & 2) : ((row >> 1) & 7) ^ ((row & 1) << 2); };
  const int64_t lhs_step = ROW * (int64_t)p.lhs.tile_rows;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)few_lds + wave * (FOURS * 4 * CHUNK);
  const uint8_t* const staged = (const uint8_t*)few_lds + wave * (FOURS * 4 * CHUNK) + r * ROW;
  uint32_t a_loaded[FOURS];
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const uint32_t at = n * ROWS_OF_LOAD + lane / PIECES;
    const uint32_t from = (uint32_t)mx_row_codes<LBITS>(p.lhs, at < p.lhs.rows ? at : p.lhs.rows - 1) + 16 * ((lane % PIECES) ^ exchanged(at));
#pragma unroll
    for (int f = 0; f < FOURS; ++f)
#pragma unroll
      for (int u = 0; u < 4; ++u)
        load_pieces(lds0 + (f * 4 + u) * CHUNK + n * 1024, from, p.lhs.codes + inside(chunk_of(f, u)) * lhs_step);
  }
  {
    const uint8_t* const lhs_scales = p.lhs.scales + mx_row_scales(p.lhs, (uint32_t)r < p.lhs.rows ? r : p.lhs.rows - 1);
#pragma unroll
    for (int f = 0; f < FOURS; ++f) {
      const uint32_t chunk = chunk_of(f, 0) + g;
      a_loaded[f] = *(const uint32_t*)(lhs_scales + inside(chunk) * (4 * (int64_t)p.lhs.tile_rows));
      if (chunk >= p.chunks) a_loaded[f] = 0x7F7F7F7Fu;
    }
  }
  // (Loads behind those to LDS, none of which is counted on.)
#pragma unroll
  for (int d = 0; d < AHEAD; ++d) {
    if (first + d >= end) break;
    to_panel(first + d);
#pragma unroll
    for (int f = 0; f < FOURS; ++f) {
      load_scales(d, f);
#pragma unroll
      for (int u = 0; u < 4; ++u) load(d, f, u);
    }
  }
  wait_loads<0>();
#pragma unroll
  for (int f = 0; f < FOURS; ++f) {
    as[f] = scales_of_blocks(a_loaded[f], g);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint8_t* const row = staged + (f * 4 + u) * CHUNK;
      *(uint4*)a[f][u].w = *(const uint4*)(row + 16 * (g ^ exchanged(r)));
      if constexpr (LBITS == 8) *(uint4*)(a[f][u].w + 4) = *(const uint4*)(row + 16 * ((4 + g) ^ exchanged(r)));
      if (chunk_of(f, u) >= p.chunks) a[f][u] = {};
    }
  }
  // Everyone's LDS writes and reads have ended. (No wait for loads: they go on.)
  auto meet = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  meet();

  mx_v4f32* const partial = (mx_v4f32*)few_lds;  // [2][PANELS][kWaves][64], the halves in turn
  uint32_t half = 0, held = 0;
  for (uint32_t group = first; group < end; group += AHEAD) {
#pragma unroll
    for (int d = 0; d < AHEAD; ++d) {
      const uint32_t panel = group + d;
      if (panel >= end) break;
      mx_v4f32 acc = {};
      const bool more = panel + AHEAD < end;
      auto multiply = [&](int f, auto number, uint32_t bs) {
        constexpr int U = decltype(number)::value;
        if constexpr (LBITS == 8) {
          MxFragment<8> whole = a[f][U], high, low;
#pragma unroll
          for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(whole.w[i]));  // (or both parts are kept in registers)
          mx_split(whole, high, low);
          acc = mx_mfma_16<4, 8, U>(b[d][f][U], bs, high, as[f], acc);
          acc = mx_mfma_16<4, 8, U>(b[d][f][U], bs, low, as[f], acc);
        } else {
          acc = mx_mfma_16<4, LBITS, U>(b[d][f][U], bs, a[f][U], as[f], acc);
        }
      };
      auto of_panel = [&](auto loads) {
#pragma unroll
        for (int f = 0; f < FOURS; ++f) {
          const uint32_t bs = scales_of_blocks(b_loaded[d][f], g);
          if constexpr (decltype(loads)::value) load_scales(d, f);
          auto one = [&](auto u) {
            multiply(f, u, bs);
            if constexpr (decltype(loads)::value) load(d, f, decltype(u)::value);
          };
          one(std::integral_constant<int, 0>{});
          one(std::integral_constant<int, 1>{});
          one(std::integral_constant<int, 2>{});
          one(std::integral_constant<int, 3>{});
        }
      };
      if (more) {
        to_panel(panel + AHEAD);
        of_panel(std::true_type{});
      } else {
        of_panel(std::false_type{});
      }
      partial[((half * PANELS + held) * kWaves + wave) * 64 + lane] = acc;
      if (++held == PANELS || panel + 1 == end) {
        meet();
        for (uint32_t n = wave; n < held; n += kWaves) {
          const mx_v4f32* const of = partial + (half * PANELS + n) * kWaves * 64 + lane;
          mx_v4f32 v = of[0];
#pragma unroll
          for (int w = 1; w < kWaves; ++w) v += of[w * 64];
          if ((uint32_t)r < p.lhs.rows) mx_store_four(p, mx_out_row(p, r), 16 * (panel + 1 - held + n) + 4 * g, v);
        }
        half ^= 1;
        held = 0;
      }
    }
  }
}

template <int LBITS, int MT, int NT, bool STAGED>
hipError_t launch(const MxProduct& p, hipStream_t stream) {
  const dim3 grid((p.rhs.rows + 16 * NT - 1) / (16 * NT), (p.lhs.rows + 16 * MT - 1) / (16 * MT));
  void* args[] = {const_cast<MxProduct*>(&p)};
  const bool stream_rhs = comes_from_hbm((int64_t)p.rhs.rows * p.chunks * 64);
  const void* kernel = stream_rhs ? (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, true, STAGED>
                                  : (const void*)mx_mmt4d_few_kernel<LBITS, MT, NT, false, STAGED>;
  constexpr int SUMS = kWaves * MT * NT * 1024, LHS = STAGED ? kWaves * 4 * MT * 256 * LBITS : 0, LDS = SUMS > LHS ? SUMS : LHS;
  static_assert(LDS <= 160 * 1024, "LDS");
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return e;
  }
  return hipLaunchKernel(kernel, grid, dim3(64 * kWaves), args, LDS, stream);
}

template <int LBITS, int FOURS>
hipError_t launch_resident(const MxProduct& p, hipStream_t stream) {
  const void* kernel = (const void*)mx_mmt4d_resident_kernel<LBITS, FOURS>;
  constexpr int SUMS = 2 * 4 * kWaves * 1024, LHS = kWaves * FOURS * 4 * 256 * LBITS, LDS = SUMS > LHS ? SUMS : LHS;
  if (LDS > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
    if (e != hipSuccess) return e;
  }
  const uint32_t panels = (p.rhs.rows + 15) / 16;
  void* args[] = {const_cast<MxProduct*>(&p)};
  return hipLaunchKernel(kernel, dim3(panels < kMxResidentGroups ? panels : kMxResidentGroups), dim3(64 * kWaves), args, LDS, stream);
}

template <int LBITS>
hipError_t launch_of(const MxProduct& p, int shape, hipStream_t stream) {
  switch (shape) {  // kMxFewShapes
    case 0: return launch<LBITS, 1, 1, false>(p, stream);
    case 1: return launch<LBITS, 1, 2, false>(p, stream);
    case 2: return launch<LBITS, 1, 4, false>(p, stream);
    case 3: return launch<LBITS, 1, 1, true>(p, stream);
    case 4: return launch<LBITS, 1, 2, true>(p, stream);
    case 5: return launch<LBITS, 1, 4, true>(p, stream);
    case 6: return launch<LBITS, 2, 1, true>(p, stream);
    case 7: return launch<LBITS, 2, 2, true>(p, stream);
    case 8: return launch<LBITS, 2, 4, true>(p, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_mx_few(const MxProduct& p, int lhs_bits, int shape, hipStream_t stream) {
  return lhs_bits == 4 ? launch_of<4>(p, shape, stream) : launch_of<8>(p, shape, stream);
}

hipError_t launch_mx_resident(const MxProduct& p, int lhs_bits, hipStream_t stream) {
  if (p.chunks <= 32) return lhs_bits == 4 ? launch_resident<4, 1>(p, stream) : launch_resident<8, 1>(p, stream);
  return lhs_bits == 4 ? launch_resident<4, 2>(p, stream) : launch_resident<8, 2>(p, stream);
}

}  // namespace uk
