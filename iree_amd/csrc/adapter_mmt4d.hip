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

constexpr int kWaves = 8;      // of a workgroup that multiplies by `down`
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
  uint32_t slots, units;    // of a launch: workgroups' pieces of work
  uint32_t parts, parts_reciprocal, slots_reciprocal;
  int32_t accumulate, runs;
};

// f(adapter, which of the sixteen rows have it) for every `slots`-th adapter of the rows from `first` on. -> The rows that have none.
template <typename F>
__device__ __forceinline__ uint32_t of_adapters(const AdapterProduct& p, uint32_t first, uint32_t slot, int lane, F f) {
  const uint32_t row = first + (lane & 15);
  const int32_t named = row < p.lhs.rows ? p.index[row] : -1;
  uint32_t left = (uint32_t)__builtin_amdgcn_ballot_w64(named >= 0 && (uint32_t)named < p.count) & 0xFFFF;
  const uint32_t without = ~left & 0xFFFF;
  while (left != 0) {
    const int32_t of = __builtin_amdgcn_readlane(named, __builtin_ctz(left));
    const uint32_t same = (uint32_t)__builtin_amdgcn_ballot_w64(named == of) & left;
    left &= ~same;
    if (slot == 0) f((uint32_t)of, same);
    slot = slot == 0 ? p.slots - 1 : slot - 1;
  }
  return without;
}

// Sums of 16 rows with 16 * RT ranks over a split's part of K, which the wavefronts share four chunks of 32 at a time; they meet in
// LDS, in the order of the wavefronts' numbers.
template <Float T, int RT>
__global__ __launch_bounds__(64 * kWaves) void adapter_down_kernel(const AdapterProduct p) {
  __shared__ p16_v4f32 partial[kWaves][RT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t full = p.depth >> 5, rest = p.depth & 31;
  for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    // unit = (tile * slots + slot) * parts + (block of ranks * splits + split)
    const uint32_t upper = divide(unit, p.parts, p.parts_reciprocal), part = unit - upper * p.parts;
    const uint32_t tile = divide(upper, p.slots, p.slots_reciprocal), slot = upper - tile * p.slots;
    const uint32_t block = part / p.splits, split = part - block * p.splits;
    const uint32_t first = tile * 16, first_rank = block * (16 * RT);
    // (Splits begin with whole fours.)
    const uint32_t fours = (full + 3) / 4;
    const uint32_t from = (uint32_t)((uint64_t)fours * split / p.splits), to = (uint32_t)((uint64_t)fours * (split + 1) / p.splits);
    const uint32_t row = first + r < p.lhs.rows ? first + r : p.lhs.rows - 1;
    const uint32_t panel = divide(row, p.lhs.tile_rows, p.lhs.tile_reciprocal);
    const uint8_t* const lhs = p.lhs.data + (int64_t)panel * p.lhs.stride0 + (row - panel * p.lhs.tile_rows) * p.lhs.row_bytes +
                               (g & 1) * p.lhs.piece1 + (g >> 1) * p.lhs.piece2;
    const int64_t lhs_step = 64 * (int64_t)p.lhs.tile_rows;
    of_adapters(p, first, slot, lane, [&](uint32_t of, uint32_t same) {
      const uint8_t* down[RT];
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        const uint32_t rank = first_rank + 16 * j + r;
        down[j] = p.down + of * p.down_stride0 + (int64_t)(rank < p.rank ? rank : p.rank - 1) * p.down_stride1 + 16 * g;
      }
      p16_v4f32 acc[RT] = {};
      uint4 a[4], b[4][RT];
      auto load = [&](int u, uint32_t four) {
        const uint32_t chunk = 4 * four + u < full ? 4 * four + u : full - 1;
        a[u] = *(const uint4*)(lhs + chunk * lhs_step);
#pragma unroll
        for (int j = 0; j < RT; ++j) b[u][j] = *(const uint4*)(down[j] + (int64_t)chunk * 64);
      };
      auto multiply = [&](int u) {
#pragma unroll
        for (int j = 0; j < RT; ++j) acc[j] = mfma16_16<T>(b[u][j], a[u], acc[j]);
      };
      uint32_t four = from + wave;
      if (four < to) {
#pragma unroll
        for (int u = 0; u < 4; ++u) load(u, four);
        for (; four + kWaves < to; four += kWaves) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            multiply(u);
            load(u, four + kWaves);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (4 * four + u < full) multiply(u);
      }
      // What K has behind its last whole chunk, zeros behind it.
      if (rest != 0 && split == p.splits - 1 && wave == (int)((to - from) % kWaves)) {
        const int exist = (int)rest - 8 * g;
        a[0] = last_piece(lhs + full * lhs_step, exist);
#pragma unroll
        for (int j = 0; j < RT; ++j) b[0][j] = last_piece(down[j] + (int64_t)full * 64, exist);
        multiply(0);
      }
#pragma unroll
      for (int j = 0; j < RT; ++j) partial[wave][j][lane] = acc[j];
      __syncthreads();
      for (int j = wave; j < RT; j += kWaves) {
        p16_v4f32 v = partial[0][j][lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += partial[w][j][lane];
        const uint32_t rank = first_rank + 16 * j + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = rank + e < p.rank ? v[e] : 0;  // (ranks behind the last meet zeros, and are finite)
        if ((same >> r & 1) != 0 && rank < p.pitch) *(p16_v4f32*)(p.sums + ((int64_t)split * p.lhs.rows + first + r) * p.pitch + rank) = v;
      }
      __syncthreads();
    });
  }
}

// 16 rows times 16 * kFragments columns a wavefront. Sums and products are f32: v_mfma_f32_16x16x4, lane (r, g) with V ranks from V g on
// of each 4 V, of row r of the sums and of column r.
template <Float T, int V, bool ALIGNED>
__global__ __launch_bounds__(256) void adapter_up_kernel(const AdapterProduct p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  for (uint32_t unit = blockIdx.x; unit < p.units; unit += gridDim.x) {
    // unit = (tile * slots + slot) * parts + block of columns
    const uint32_t upper = divide(unit, p.parts, p.parts_reciprocal), part = unit - upper * p.parts;
    const uint32_t tile = divide(upper, p.slots, p.slots_reciprocal), slot = upper - tile * p.slots;
    const uint32_t first = tile * 16, first_col = (part * 4 + wave) * (16 * kFragments);
    if (first_col >= p.cols) continue;
    const uint32_t row = first + r < p.lhs.rows ? first + r : p.lhs.rows - 1;
    const int64_t out_row = layout_row(p.out_at, row);
    auto store = [&](int f, p16_v4f32 v) {
      const uint32_t col = first_col + 16 * f + 4 * g;
      if (p.runs && col + 4 <= p.cols) {
        const int64_t at = out_row + layout_col(p.out_at, col);
        float x[4] = {v[0], v[1], v[2], v[3]}, old[4];
        if (p.out_type == Float::kF32) {
          if (p.accumulate) {
            load_run<Float::kF32, 4>(p.out, at, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += old[e];
          }
          store_run<Float::kF32, 4>(p.out, at, x);
        } else {
          if (p.accumulate) {
            load_run<T, 4>(p.out, at, old);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] += old[e];
          }
          store_run<T, 4>(p.out, at, x);
        }
        return;
      }
#pragma unroll 1
      for (int e = 0; e < 4; ++e) {
        if (col + e >= p.cols) continue;
        const int64_t at = out_row + layout_col(p.out_at, col + e);
        const float old = !p.accumulate ? 0 : p.out_type == Float::kF32 ? element<Float::kF32>(p.out, at) : element<T>(p.out, at);
        if (p.out_type == Float::kF32) ((float*)p.out)[at] = old + v[e];
        else ((uint16_t*)p.out)[at] = mx_narrow<T>(old + v[e]);
      }
    };
    const uint32_t without = of_adapters(p, first, slot, lane, [&](uint32_t of, uint32_t same) {
      const uint8_t* up[kFragments];
#pragma unroll
      for (int f = 0; f < kFragments; ++f) {
        const uint32_t col = first_col + 16 * f + r;
        up[f] = p.up + of * p.up_stride0 + (int64_t)(col < p.cols ? col : p.cols - 1) * p.up_stride1;
      }
      p16_v4f32 acc[kFragments] = {};
      for (uint32_t from = 0; from < p.rank; from += 4 * V) {
        const uint32_t rank = from + V * g;
        float sum[V] = {};
        for (uint32_t s = 0; s < p.splits; ++s) {
          const float* at = p.sums + ((int64_t)s * p.lhs.rows + row) * p.pitch + rank;
#pragma unroll
          for (int e = 0; e < V; e += 4) {
            const p16_v4f32 v = *(const p16_v4f32*)(at + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[e + i] += v[i];
          }
        }
#pragma unroll
        for (int f = 0; f < kFragments; ++f) {
          uint16_t w[V];
          if (ALIGNED && rank + V <= p.rank) {
            __builtin_memcpy(w, __builtin_assume_aligned(up[f] + 2 * rank, 2 * V), 2 * V);
          } else {
#pragma unroll
            for (int e = 0; e < V; ++e) w[e] = rank + e < p.rank ? ((const uint16_t*)up[f])[rank + e] : 0;
          }
#pragma unroll
          for (int e = 0; e < V; ++e) acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(mx_widen<T>(w[e]), sum[e], acc[f], 0, 0, 0);
        }
      }
      const float scale = p.scales ? p.scales[of] : 1;
      if ((same >> r & 1) != 0) {
#pragma unroll
        for (int f = 0; f < kFragments; ++f) store(f, acc[f] * scale);
      }
    });
    if (!p.accumulate && slot == 0 && (without >> r & 1) != 0 && first + r < p.lhs.rows) {
#pragma unroll
      for (int f = 0; f < kFragments; ++f) store(f, p16_v4f32{0, 0, 0, 0});
    }
  }
}

// How many parts K is split into: as many as leave every wavefront four chunks, while there are fewer workgroups than compute units.
uint32_t splits_of(int64_t rows, int64_t depth, int64_t rank) {
  const int64_t tiles = (rows + 15) / 16 * ((rank + 16 * kFragments - 1) / (16 * kFragments));
  const int64_t most = depth / 32 / (4 * kWaves), wanted = (256 + tiles - 1) / tiles;
  const int64_t s = most < wanted ? most : wanted;
  return (uint32_t)(s < 1 ? 1 : s);
}
int64_t pitch_of(int64_t rank) { return (rank + 31) / 32 * 32; }

bool multiple(const void* p, int64_t to) { return (uintptr_t)p % to == 0; }

// The problem as the kernels on the matrix pipe take it; false: they do not.
bool as_product(const AdapterArgs& a, AdapterProduct* p) {
  const int64_t depth = a.K * a.K0, cols = a.N * a.N0;
  if (a.count == 0 || depth > 0x7FFFFFFF || cols > 0x7FFFFFFF - 512) return false;
  if (!as_operand16(a.lhs, a.lhs_stride0, a.M, a.M0, a.K, a.K0, &p->lhs)) return false;
  if (!multiple(a.down, 16) || (a.count > 1 && a.down_stride0 % 8 != 0) || (a.rank > 1 && a.down_stride1 % 8 != 0)) return false;
  const int64_t rows = a.M * a.M0, tiles = (rows + 15) / 16;
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
  p->splits = splits_of(rows, depth, a.rank);
  p->accumulate = a.accumulate;
  const int e = float_bytes(a.out_type);
  p->runs = runs_of(p->out_at, a.out, a.M, e, 4, 4 * e);
  // Adapters of a tile side by side where there are few tiles.
  const int64_t slots = 128 / tiles, most = a.count < 16 ? a.count : 16;
  p->slots = (uint32_t)(slots < 1 ? 1 : slots > most ? most : slots);
  p->slots_reciprocal = reciprocal_of(p->slots);
  return true;
}

// One launch over tiles * slots * parts pieces of work.
hipError_t launch_units(void (*kernel)(const AdapterProduct), AdapterProduct p, int64_t parts, unsigned threads, hipStream_t stream) {
  const int64_t tiles = ((int64_t)p.lhs.rows + 15) / 16;
  p.parts = (uint32_t)parts;
  p.parts_reciprocal = reciprocal_of(p.parts);
  p.units = (uint32_t)(tiles * p.slots * parts);
  return launch_kernel(kernel, p.units < (1u << 22) ? p.units : 1u << 22, threads, 0, stream, p);
}

template <Float T>
hipError_t launch_down(const AdapterProduct& p, hipStream_t stream) {
  const int64_t fragments = (p.rank + 15) / 16;
  if (fragments == 1) return launch_units(adapter_down_kernel<T, 1>, p, p.splits, 64 * kWaves, stream);
  if (fragments == 2) return launch_units(adapter_down_kernel<T, 2>, p, p.splits, 64 * kWaves, stream);
  return launch_units(adapter_down_kernel<T, kFragments>, p, (fragments + kFragments - 1) / kFragments * p.splits, 64 * kWaves, stream);
}

template <Float T>
hipError_t launch_up(const AdapterProduct& p, hipStream_t stream) {
  const int64_t parts = ((int64_t)p.cols + 64 * kFragments - 1) / (64 * kFragments);
  const int v = p.rank <= 16 ? 4 : 8;
  const bool aligned = multiple(p.up, 2 * v) && (p.count <= 1 || p.up_stride0 % (2 * v) == 0) && (p.cols <= 1 || p.up_stride1 % (2 * v) == 0);
  if (v == 4) return launch_units(aligned ? adapter_up_kernel<T, 4, true> : adapter_up_kernel<T, 4, false>, p, parts, 256, stream);
  return launch_units(aligned ? adapter_up_kernel<T, 8, true> : adapter_up_kernel<T, 8, false>, p, parts, 256, stream);
}

// Whether the pieces of work of both launches are fewer than 2^31.
bool countable(const AdapterProduct& p) {
  const int64_t tiles = ((int64_t)p.lhs.rows + 15) / 16, blocks = (p.rank + 15) / 16;
  const int64_t parts = ((int64_t)p.cols + 64 * kFragments - 1) / (64 * kFragments), most = (1ll << 31) / (tiles * p.slots);
  return blocks * p.splits < most && parts < most;
}

}  // namespace

int64_t adapter_workspace(const AdapterArgs& a) {
  if (a.count == 0) return 0;
  const int64_t rows = a.M * a.M0;  // fewer than 2^31, and 2^15 ranks
  int64_t bytes;
  if (__builtin_mul_overflow(rows * pitch_of(a.rank) * 4, (int64_t)splits_of(rows, a.K * a.K0, a.rank), &bytes) || bytes > INT64_MAX - 256) return -1;
  return (bytes + 255) / 256 * 256;
}

hipError_t launch_adapter_mmt4d(const AdapterArgs& a, hipStream_t stream, const char** name) {
  AdapterProduct p;
  if (as_product(a, &p) && countable(p)) {
    *name = "adapter_mmt4d";
    const bool f16 = a.type == Float::kF16;
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
