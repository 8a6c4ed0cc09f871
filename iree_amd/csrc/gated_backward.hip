// The backward pass of gated products: the gradients of the two products, rounded to the operands' type, into the workspace, then
// the products that give the gradients of lhs, gate and up.
#include "gated_backward.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

// dg and du of f16 operands are held as multiples of a power of two, the call's `unit`, which brings the largest of them (that is finite)
// to between 2^14 and 2^15. As they are, 65504 and more would be infinite, which gradients of a scaled loss come to, and 2^-25 and less
// zero; like this what is 2^-28 of the largest or more has all bits of an f16, and only what is less than 2^-39 of it is zero. A pass over
// the inputs in front of the first step finds the largest, each of its workgroups one of some; the first step makes the unit of these, and
// the products' results are multiplied by it in f32. (bf16 has f32's range.) The pass takes 26 us of 2048 x 8192, f16 throughout, 100 MB,
// where the whole backward pass takes 600, and 4 of 130 x 1000.
struct Scaling {
  float* largest;  // [kMostLargest]
  float* unit;     // or null: there is no dg
  uint32_t count;  // of the largest
};
constexpr int kMostLargest = 8 * kThreads, kScalingBytes = 4 * kMostLargest + 256;

// In the first step, by all of a workgroup: one over the unit.
__device__ __forceinline__ float one_over_unit(const Scaling& s) {
  __shared__ float of_wave[kThreads / 64];
  float v = 0;
#pragma unroll
  for (uint32_t i = 0; i < kMostLargest / kThreads; ++i) {
    const uint32_t at = i * kThreads + threadIdx.x;
    v = __builtin_fmaxf(v, at < s.count ? s.largest[at] : 0);
  }
  for (int by = 32; by > 0; by /= 2) v = __builtin_fmaxf(v, __shfl_xor(v, by));
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) v = __builtin_fmaxf(v, of_wave[w]);
  // (Of subnormals, and zeros, as large as a float's exponent has it.)
  const int by = v == 0 ? 0 : 127 + 14 - (int)(__builtin_bit_cast(uint32_t, v) >> 23), power = by < 126 ? by : 126;
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.unit = __builtin_bit_cast(float, (uint32_t)(127 - power) << 23);
  return __builtin_bit_cast(float, (uint32_t)(127 + power) << 23);
}
// In the pass in front of it: the larger one.
__device__ __forceinline__ float larger(float largest, float v) {
  v = __builtin_fabsf(v);
  return v < __builtin_inff() && v > largest ? v : largest;
}
__device__ __forceinline__ void put_largest(const Scaling& s, float v) {
  __shared__ float of_wave[kThreads / 64];
  for (int by = 32; by > 0; by /= 2) v = __builtin_fmaxf(v, __shfl_xor(v, by));
  if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = v;
  __syncthreads();
  for (int w = 0; w < kThreads / 64; ++w) v = __builtin_fmaxf(v, of_wave[w]);
  if (threadIdx.x == 0) s.largest[blockIdx.x] = v;
}

// The workspace: [rows][2 * cols] of the operands' type, a row's dg then its du, each filled up with zeros to a multiple of eight;
// behind it, of f16, what Scaling has, and where lhs_grad's sums over the columns are split, [splits][rows][depth] of f32.
struct Sizes {
  int64_t rows, cols, depth, pitch;
  explicit Sizes(const GatedBackwardArgs& a)
      : rows(a.M * a.M0), cols(a.N * a.N0), depth(a.K * a.K0), pitch(2 * ((cols + 7) / 8 * 8)) {}
};

struct BackwardArgs {
  GatedBackwardArgs p;
  Curve curve;
  Scaling scaling;
  int64_t rows, cols, depth, pitch, results;
};

// LARGEST: the pass in front that finds it.
template <Float T, bool LARGEST>
__global__ __launch_bounds__(kThreads) void gated_backward_generic(const BackwardArgs g) {
  const GatedBackwardArgs& a = g.p;
  const int64_t half = g.pitch / 2;
  const float times = T == Float::kF16 && !LARGEST ? one_over_unit(g.scaling) : 1;
  float largest = 0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t row = n / half, col = n % half;
    float dg = 0, du = 0;
    if (col < g.cols) {
      const int64_t i = row / a.M0, in_row = ((col / a.N0) * a.M0 + row % a.M0) * a.N0 + col % a.N0;
      const float grad = element(a.out_type, a.out_grad, i * a.out_grad_stride0 + in_row);
      const float u = element(a.pre_type, a.up_pre, i * a.up_pre_stride0 + in_row);
      float slope;
      du = grad * activated_and_slope(g.curve, element(a.pre_type, a.gate_pre, i * a.gate_pre_stride0 + in_row), &slope);
      dg = grad * u * slope;
    }
    if constexpr (LARGEST) {
      largest = larger(larger(largest, dg), du);
      continue;
    }
    uint16_t* to = (uint16_t*)a.workspace + row * g.pitch + col;
    to[0] = mx_narrow<T>(dg * times);
    to[half] = mx_narrow<T>(du * times);
  }
  if constexpr (LARGEST) put_largest(g.scaling, largest);
}

template <Float T>
__device__ __forceinline__ float unit_of(const Scaling& s) {
  return T == Float::kF16 && s.unit ? *s.unit : 1;
}

// lhs_grad: a thread for each result, which goes over the columns.
template <Float T>
__global__ __launch_bounds__(kThreads) void gated_lhs_grad_generic(const BackwardArgs g) {
  const GatedBackwardArgs& a = g.p;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t row = n / g.depth, k = n % g.depth;
    const uint16_t* from = (const uint16_t*)a.workspace + row * g.pitch;
    float sum = 0;
    for (int64_t j = 0; j < a.N; ++j) {
      for (int j0 = 0; j0 < a.N0; ++j0) {
        const int64_t col = j * a.N0 + j0, at = (k / a.K0 * a.N0 + j0) * a.K0 + k % a.K0;
        sum += mx_widen<T>(from[col]) * element<T>(a.gate, j * a.gate_stride0 + at);
        sum += mx_widen<T>(from[g.pitch / 2 + col]) * element<T>(a.up, j * a.up_stride0 + at);
      }
    }
    put_element(a.out_type, a.lhs_grad, row / a.M0 * a.lhs_grad_stride0 + (k / a.K0 * a.M0 + row % a.M0) * a.K0 + k % a.K0,
                sum * unit_of<T>(g.scaling));
  }
}

// gate_grad and up_grad: a thread for each place, which goes over the rows.
template <Float T>
__global__ __launch_bounds__(kThreads) void gated_weight_grad_generic(const BackwardArgs g) {
  const GatedBackwardArgs& a = g.p;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t col = n / g.depth, k = n % g.depth;
    float sum_g = 0, sum_u = 0;
    for (int64_t row = 0; row < g.rows; ++row) {
      const float x = element<T>(a.lhs, row / a.M0 * a.lhs_stride0 + (k / a.K0 * a.M0 + row % a.M0) * a.K0 + k % a.K0);
      const uint16_t* from = (const uint16_t*)a.workspace + row * g.pitch + col;
      sum_g += mx_widen<T>(from[0]) * x;
      sum_u += mx_widen<T>(from[g.pitch / 2]) * x;
    }
    sum_g *= unit_of<T>(g.scaling);
    sum_u *= unit_of<T>(g.scaling);
    const int64_t panel = col / a.N0, in_panel = (k / a.K0 * a.N0 + col % a.N0) * a.K0 + k % a.K0;
    if (a.gate_grad) {
      const int64_t at = panel * a.gate_grad_stride0 + in_panel;
      put_element(a.out_type, a.gate_grad, at, a.accumulate ? element(a.out_type, a.gate_grad, at) + sum_g : sum_g);
    }
    if (a.up_grad) {
      const int64_t at = panel * a.up_grad_stride0 + in_panel;
      put_element(a.out_type, a.up_grad, at, a.accumulate ? element(a.out_type, a.up_grad, at) + sum_u : sum_u);
    }
  }
}

// The first step where eight columns at a time lie next to each other, aligned: a thread for eight. Memory bounds it: 2048 x 8192, bf16
// throughout, 33 to 36 us, 168 MB at 4.7 to 5.1 TB/s. dg and du are rounded to the operands' type here since the products' matrix
// instructions take that; with the gradients' own rounding that is two roundings in all (errors of 0.0023 of a bf16 gradient's size, and
// 0.0017 with one), and as 32-bit sums of two parts they would double both products.
struct FirstStep {
  const uint8_t *gate_pre, *up_pre, *out_grad;
  uint8_t* grads;
  Layout gate_at, up_at, out_at;
  Curve curve;
  Scaling scaling;
  int64_t results;  // eights
  uint32_t half, half_reciprocal;  // eights of a row's dg
  int64_t pitch;
  Float pre_type, out_type;
};
template <Float T, bool LARGEST>
__global__ __launch_bounds__(kThreads) void gated_backward_first(const FirstStep p) {
  const float times = T == Float::kF16 && !LARGEST ? one_over_unit(p.scaling) : 1;
  float largest = 0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < p.results; n += (int64_t)gridDim.x * kThreads) {
    const uint32_t row = p.results < (1ll << 32) ? divide((uint32_t)n, p.half, p.half_reciprocal) : (uint32_t)(n / p.half);
    const uint32_t col = 8 * (uint32_t)(n - (int64_t)row * p.half);
    auto load = [&](Float type, const uint8_t* from, const Layout& l, float (&v)[8]) {
      const int64_t at = layout_row(l, row) + layout_col(l, col);
      if (type == Float::kF32) load_run<Float::kF32, 8>(from, at, v);
      else load_run<T, 8>(from, at, v);
    };
    float g[8], u[8], grad[8];
    load(p.pre_type, p.gate_pre, p.gate_at, g);
    load(p.pre_type, p.up_pre, p.up_at, u);
    load(p.out_type, p.out_grad, p.out_at, grad);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float slope;
      const float value = activated_and_slope(p.curve, g[e], &slope);
      g[e] = grad[e] * u[e] * slope;
      u[e] = grad[e] * value;
      if constexpr (LARGEST) {
        largest = larger(larger(largest, g[e]), u[e]);
      } else {
        g[e] *= times;
        u[e] *= times;
      }
    }
    if constexpr (LARGEST) continue;
    const int64_t to = (int64_t)row * p.pitch + col;
    store_run<T, 8>(p.grads, to, g);
    store_run<T, 8>(p.grads, to + p.pitch / 2, u);
  }
  if constexpr (LARGEST) put_largest(p.scaling, largest);
}

hipError_t launch_over(void (*f16)(const BackwardArgs), void (*bf16)(const BackwardArgs), BackwardArgs& g, int64_t results, hipStream_t stream) {
  if (results == 0) return hipSuccess;
  g.results = results;
  const int64_t groups = (results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  return launch_kernel(g.p.type == Float::kF16 ? f16 : bf16, grid, kThreads, 0, stream, g);
}

// The first step, of f16 behind the pass that finds the largest.
template <typename P>
hipError_t launch_step(void (*largest)(const P), void (*f16)(const P), void (*bf16)(const P), Float type, const P& p, hipStream_t stream) {
  if (p.results == 0) return hipSuccess;
  const int64_t groups = (p.results + kThreads - 1) / kThreads;
  if (type == Float::kF16) {
    const hipError_t e = launch_kernel(largest, p.scaling.count, kThreads, 0, stream, p);
    if (e != hipSuccess) return e;
  }
  return launch_kernel(type == Float::kF16 ? f16 : bf16, (unsigned)(groups < (1 << 22) ? groups : 1 << 22), kThreads, 0, stream, p);
}

GradResults results_of(const GatedBackwardArgs& a, const Layout& at, uint8_t* first, uint8_t* second, int64_t stride0, int64_t stride1,
                       int64_t rows, int64_t panels, const float* unit, bool accumulate) {
  GradResults r;
  r.out[0] = first; r.out[1] = second;
  r.stride0[0] = stride0; r.stride0[1] = stride1;
  r.at = at;
  r.type = a.out_type;
  r.unit = unit;
  r.accumulate = accumulate;
  const int e = float_bytes(a.out_type);
  Layout other = at;
  other.stride0 = stride1;
  r.runs = runs_of(at, first, panels, e, 16 / e, 16) && (!second || runs_of(other, second, panels, e, 16 / e, 16));
  r.rows = (uint32_t)rows;
  r.apart = 0;
  r.copies = second ? 2 : 1;
  r.tile_rows_of_copy = r.tile_rows_reciprocal = 0;
  return r;
}

// Which tile, and how many parts K is split into: the least of the times that a model gives, in microseconds: a start, and chunks of K
// times what one of them takes with one workgroup on a compute unit and, where LDS and registers hold two, with two; more than that
// follow each other. With all compute units busy, clocks and memory hold a chunk to `busy` for each 256 workgroups at least. Fitted to
// the times of every tile in 260 problems from 16 to 4096 rows, 64 to 28672 columns, K of 64 to 14336, and, for lhs_grad, of every tile
// with up to ten numbers of parts in 120 of 1 to 4096 rows; over these what is taken is slower than the best by 0.7 % (lhs) and 1.3 %
// (weights) in the mean. lhs_grad's K is both weights' rows, and its results are few where the rows are: 19 x 18592 x 448 takes 25.7 us
// in 28 parts and 188 in one, 100 x 12176 x 3504 45 and 125, 508 x 9526 x 325 33 and 105, 2048 x 8192 x 4096 245 in two and 283 in one
// (of smaller tiles). tile -1: none can.
struct Times { float start, one, two, start_again, busy; };  // two = 0: one workgroup on a compute unit
struct Choice { int tile, splits; float cost; };
// The parts of sums are written and read, in a launch more.
float parts_time(int64_t rows, int64_t cols, int64_t splits) { return splits == 1 ? 0 : 2 + (float)splits * (float)(rows * cols) * 1.5e-6f; }
Choice choose(const Times* times, int64_t rows, int64_t cols, int64_t chunks, int64_t copies, int64_t most_splits) {
  Choice best = {-1, 1, 0};
  for (int i = 0; i < (int)(sizeof kGradTiles / sizeof kGradTiles[0]); ++i) {
    const GradTile& t = kGradTiles[i];
    const int64_t of_one = (rows + t.rows - 1) / t.rows * ((cols + t.cols - 1) / t.cols) * copies;
    const Times& of = times[i];
    for (int64_t splits = 1; splits <= most_splits; ++splits) {
      if (splits > 1 && of_one * (splits - 1) > 512) break;  // (all compute units had two)
      const int64_t tiles = of_one * splits, rounds = (tiles + 255) / 256;
      if (tiles > (1 << 23)) continue;  // (a grid has fewer than 2^32 threads)
      const float in_turn = (float)chunks / (float)splits * (of.two == 0 ? rounds * of.one : (rounds >> 1) * of.two + (rounds & 1) * of.one);
      const float busy = (float)of_one * (float)chunks / 256 * of.busy, steps = in_turn > busy ? in_turn : busy;
      const float cost = of.start + (rounds - 1) * of.start_again + steps + parts_time(rows, cols, splits);
      if (best.tile < 0 || cost < best.cost) best = {i, (int)splits, cost};
    }
  }
  return best;
}
constexpr Times kLhsGradTimes[] = {{16.2f, .491f, 0, 21.5f, .45f},   {11.3f, .299f, 0, 11.7f, .66f},   {11.4f, .334f, .834f, 4.3f, .53f},
                                   {9.1f, .220f, .555f, 2.3f, .24f}, {7.7f, .157f, .418f, 1.1f, .29f}, {7.6f, .159f, .361f, 1.3f, .17f},
                                   {6.6f, .137f, .246f, .9f, .13f}};
constexpr Times kWeightGradTimes[] = {{17.3f, .522f, 0, 15.6f, .92f},   {11.9f, .323f, 0, 8.5f, .57f},    {11.6f, .303f, .747f, 4.1f, .49f},
                                      {8.8f, .196f, .448f, 2.4f, .27f}, {7.4f, .171f, .303f, 1.6f, .10f}, {7.3f, .164f, .313f, 1.6f, .17f},
                                      {6.3f, .141f, .210f, 1.1f, .12f}};

// lhs_grad's. A split has sixteen chunks at least, and all of them 64 MiB of sums at most.
int64_t most_splits(const Sizes& s) {
  const int64_t whole = 2 * (s.cols / 32), of_sums = s.rows > (1 << 24) / s.depth ? 1 : (1 << 24) / (s.rows * s.depth);
  const int64_t most = whole / 16 < of_sums ? whole / 16 : of_sums;
  return most < 1 ? 1 : most > 32 ? 32 : most;
}
bool choosable(const Sizes& s) {
  return s.rows > 0 && s.cols > 0 && s.depth > 0 && s.rows <= INT32_MAX && s.cols <= INT32_MAX && s.depth <= INT32_MAX;
}
Choice choose_lhs_grad(const Sizes& s) {
  if (!choosable(s)) return {-1, 1, 0};
  return choose(kLhsGradTimes, s.rows, s.depth, 2 * ((s.cols + 31) / 32), 1, most_splits(s));
}
// Both products in one launch of 64x64 tiles: the longer of them, or all chunks of all tiles, as many as the machine has at a time. Over
// 120 problems of 1 to 2048 rows, 64 to 12000 columns, K of 64 to 6000 a backward pass takes 1.23 times less in the mean where this is
// chosen for the less time (130 x 1000 x 500 15.5 us and not 20, 37 x 1338 x 1001 13.8 and 18.9; but 30 x 8567 x 3462 94 and 68 apart); what is
// chosen is slower than the better by 0.1 % in the mean.
constexpr float kBothStart = 5.6f, kBothOne = .150f, kBothTwo = .155f, kBothAgain = 2.34f, kBothBusy = .15f;
Choice choose_both(const Sizes& s, int64_t copies) {
  Choice best = {-1, 1, 0};
  if (!choosable(s)) return best;
  const int64_t of_lhs = (s.rows + 63) / 64 * ((s.depth + 63) / 64), of_weights = (s.cols + 63) / 64 * ((s.depth + 63) / 64) * copies;
  const int64_t lhs_chunks = 2 * ((s.cols + 31) / 32), weight_chunks = (s.rows + 31) / 32, most = most_splits(s);
  if (of_lhs * most + of_weights > (1 << 23)) return best;
  const float all = ((float)of_lhs * (float)lhs_chunks + (float)of_weights * (float)weight_chunks) / 256 * kBothBusy;
  for (int64_t splits = 1; splits <= most; ++splits) {
    if (splits > 1 && of_lhs * (splits - 1) + of_weights > 1024) break;
    const int64_t tiles = of_lhs * splits + of_weights;
    const float longer = lhs_chunks > splits * weight_chunks ? (float)lhs_chunks / (float)splits : (float)weight_chunks;
    const float in_turn = longer * (tiles > 256 ? kBothTwo : kBothOne), steps = in_turn > all ? in_turn : all;
    const float cost = kBothStart + (float)((tiles + 511) / 512 - 1) * kBothAgain + steps + parts_time(s.rows, s.depth, splits);
    if (best.tile < 0 || cost < best.cost) best = {kSmallestGradTile, (int)splits, cost};
  }
  return best;
}
Choice choose_weight_grads(const Sizes& s, int64_t copies) {
  if (!choosable(s)) return {-1, 1, 0};
  return choose(kWeightGradTimes, s.cols, s.depth, (s.rows + 31) / 32, copies, 1);
}
int64_t copies_of(const GatedBackwardArgs& a) { return (a.gate_grad != nullptr) + (a.up_grad != nullptr); }
int64_t grads_bytes(const Sizes& s) { return (s.rows * s.pitch * 2 + 255) / 256 * 256; }
// Where the parts of sums begin.
int64_t sums_at(const Sizes& s, Float type) { return grads_bytes(s) + (type == Float::kF16 && s.rows > 0 && s.cols > 0 ? kScalingBytes : 0); }
// Of a first step of so many pieces of work, a thread for each or more.
Scaling scaling_of(const GatedBackwardArgs& a, const Sizes& s, int64_t results) {
  if (a.type != Float::kF16 || s.rows == 0 || s.cols == 0) return {nullptr, nullptr, 0};
  float* const largest = (float*)(a.workspace + grads_bytes(s));
  const int64_t groups = (results + kThreads - 1) / kThreads;
  return {largest, largest + kMostLargest, (uint32_t)(groups < kMostLargest ? groups : kMostLargest)};
}

// The sums of lhs_grad's splits, in their order: a thread for four of a row. (2048 x 4096 in two parts: 15 us, 84 MB at 5.6 TB/s.)
struct SumArgs {
  const float* parts;
  uint8_t* out;
  Layout at;
  int64_t results, apart;  // fours; floats from a split to the next
  uint32_t cols, fours;    // of a row
  int32_t splits, runs;
  Float type;
};
template <Float T>
__global__ __launch_bounds__(kThreads) void gated_lhs_grad_sums(const SumArgs p) {
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < p.results; n += (int64_t)gridDim.x * kThreads) {
    const uint32_t row = (uint32_t)(n / p.fours), col = 4 * (uint32_t)(n - (int64_t)row * p.fours);
    const float* const from = p.parts + (int64_t)row * p.cols + col;
    float v[4];
    load_run<Float::kF32, 4>((const uint8_t*)from, 0, v);
    for (int32_t s = 1; s < p.splits; ++s) {
      float more[4];
      load_run<Float::kF32, 4>((const uint8_t*)(from + s * p.apart), 0, more);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += more[e];
    }
    const int64_t row_at = layout_row(p.at, row);
    if (p.runs) {
      if (p.type == Float::kF32) store_run<Float::kF32, 4>(p.out, row_at + layout_col(p.at, col), v);
      else store_run<T, 4>(p.out, row_at + layout_col(p.at, col), v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) put_element(p.type, p.out, row_at + layout_col(p.at, col + e), v[e]);
    }
  }
}

// false: the general kernel takes it.
bool as_lhs_grad(const GatedBackwardArgs& a, const Sizes& s, LhsGradProduct* p) {
  Strided16 up;
  if (s.rows == 0 || s.cols == 0 || s.cols > 0x7FFFFFFF - 512) return false;
  if (!as_operand16(a.workspace, s.pitch, s.rows, 1, s.cols, 1, &p->grads) || !near16(p->grads, 256) ||
      !as_strided16(a.gate, a.gate_stride0, a.N, a.N0, a.K, a.K0, &p->gate) || !as_strided16(a.up, a.up_stride0, a.N, a.N0, a.K, a.K0, &up))
    return false;
  p->up = up.data;
  p->up_stride0 = up.stride0;
  p->lhs_second = s.pitch;  // (half of a row's bytes)
  p->depth = (uint32_t)s.cols;
  p->results = results_of(a, layout_of(a.lhs_grad_stride0, a.M0, a.K, a.K0), a.lhs_grad, nullptr, a.lhs_grad_stride0, 0, s.rows, a.M,
                          scaling_of(a, s, 0).unit, false);
  return true;
}
// (The depth is a multiple of eight.)
void split_sums(const GatedBackwardArgs& a, const Sizes& s, int splits, GradResults* r) {
  r->out[0] = a.workspace + sums_at(s, a.type);
  r->at = layout_of(s.depth, 1, s.depth, 1);
  r->stride0[0] = s.depth;
  r->type = Float::kF32;
  r->runs = 1;
  r->apart = s.rows * s.depth * 4;
  r->copies = (uint32_t)splits;
}
hipError_t launch_sums(const GatedBackwardArgs& a, const Sizes& s, int splits, hipStream_t stream) {
  SumArgs g;
  g.parts = (const float*)(a.workspace + sums_at(s, a.type));
  g.out = a.lhs_grad;
  g.at = layout_of(a.lhs_grad_stride0, a.M0, a.K, a.K0);
  g.cols = (uint32_t)s.depth;
  g.fours = g.cols / 4;
  g.results = s.rows * g.fours;
  g.apart = s.rows * s.depth;
  g.splits = splits;
  const int size = float_bytes(a.out_type);
  g.runs = runs_of(g.at, a.lhs_grad, a.M, size, 4, 4 * size);
  g.type = a.out_type;
  const int64_t groups = (g.results + kThreads - 1) / kThreads;
  return launch_kernel(a.type == Float::kF16 ? gated_lhs_grad_sums<Float::kF16> : gated_lhs_grad_sums<Float::kBf16>,
                       (unsigned)(groups < (1 << 22) ? groups : 1 << 22), kThreads, 0, stream, g);
}
bool as_weight_grads(const GatedBackwardArgs& a, const Sizes& s, WeightGradProduct* p) {
  if (s.rows == 0 || s.cols == 0 || s.rows > 0x7FFFFFFF || s.cols > 0x7FFFFFFF - 512) return false;
  const uint8_t* const grads = a.workspace + (a.gate_grad ? 0 : s.pitch);
  // (As many columns of dg as there are with the zeros that fill up an eight.)
  if (!as_strided16(grads, s.pitch, s.rows, 1, s.pitch / 2, 1, &p->grads) || !as_strided16(a.lhs, a.lhs_stride0, a.M, a.M0, a.K, a.K0, &p->lhs))
    return false;
  p->lhs_second = s.pitch;
  p->depth = (uint32_t)s.rows;
  uint8_t* const first = a.gate_grad ? a.gate_grad : a.up_grad;
  uint8_t* const second = a.gate_grad ? a.up_grad : nullptr;
  const int64_t stride0 = a.gate_grad ? a.gate_grad_stride0 : a.up_grad_stride0;
  p->results = results_of(a, layout_of(stride0, a.N0, a.K, a.K0), first, second, stride0, a.up_grad_stride0, s.cols, a.N,
                          scaling_of(a, s, 0).unit, a.accumulate);
  return true;
}

bool launch_first(const GatedBackwardArgs& a, const Sizes& s, hipStream_t stream, hipError_t* e) {
  if (s.rows == 0 || s.cols == 0 || s.rows > 0x7FFFFFFF || s.cols > 0x7FFFFFFF || s.cols % 8 != 0) return false;
  FirstStep p;
  p.gate_at = layout_of(a.gate_pre_stride0, a.M0, a.N, a.N0);
  p.up_at = layout_of(a.up_pre_stride0, a.M0, a.N, a.N0);
  p.out_at = layout_of(a.out_grad_stride0, a.M0, a.N, a.N0);
  const int pe = float_bytes(a.pre_type), oe = float_bytes(a.out_type);
  if (!runs_of(p.gate_at, a.gate_pre, a.M, pe, 8, 16) || !runs_of(p.up_at, a.up_pre, a.M, pe, 8, 16) ||
      !runs_of(p.out_at, a.out_grad, a.M, oe, 8, 16))
    return false;
  p.gate_pre = a.gate_pre; p.up_pre = a.up_pre; p.out_grad = a.out_grad;
  p.grads = a.workspace;
  p.curve = curve_of(a.activation);
  p.half = (uint32_t)(s.cols / 8);
  p.half_reciprocal = reciprocal_of(p.half);
  p.results = s.rows * p.half;
  p.pitch = s.pitch;
  p.pre_type = a.pre_type; p.out_type = a.out_type;
  p.scaling = scaling_of(a, s, p.results);
  *e = launch_step(gated_backward_first<Float::kF16, true>, gated_backward_first<Float::kF16, false>, gated_backward_first<Float::kBf16, false>,
                   a.type, p, stream);
  return true;
}

}  // namespace

int64_t gated_backward_workspace(const GatedBackwardArgs& a) {
  const Sizes s(a);
  int64_t bytes;
  if (__builtin_mul_overflow(s.rows, 2 * s.pitch, &bytes) || bytes > INT64_MAX - (1ll << 30)) return -1;
  bytes = sums_at(s, a.type);
  if (a.lhs_grad) {
    int splits = choose_lhs_grad(s).splits;
    if (const int64_t copies = copies_of(a)) {
      const int both = choose_both(s, copies).splits;
      splits = splits < both ? both : splits;
    }
    if (splits > 1) bytes += splits * s.rows * s.depth * 4;
  }
  return bytes;
}

hipError_t launch_gated_backward(const GatedBackwardArgs& a, hipStream_t stream, const char** name) {
  const Sizes s(a);
  BackwardArgs g;
  g.p = a;
  g.curve = curve_of(a.activation);
  g.rows = s.rows; g.cols = s.cols; g.depth = s.depth; g.pitch = s.pitch;
  *name = "gated_backward";
  hipError_t e = hipSuccess;
  g.results = s.rows * (s.pitch / 2);
  g.scaling = scaling_of(a, s, g.results);
  if (!launch_first(a, s, stream, &e))
    e = launch_step(gated_backward_generic<Float::kF16, true>, gated_backward_generic<Float::kF16, false>,
                    gated_backward_generic<Float::kBf16, false>, a.type, g, stream);
  if (e != hipSuccess) return e;
  LhsGradProduct lhs;
  WeightGradProduct weights;
  const int64_t copies = copies_of(a);
  const bool f16 = a.type == Float::kF16;
  bool lhs_fast = a.lhs_grad && as_lhs_grad(a, s, &lhs), weights_fast = copies && as_weight_grads(a, s, &weights);
  Choice of_lhs = lhs_fast ? choose_lhs_grad(s) : Choice{-1, 1, 0};
  const Choice of_weights = weights_fast ? choose_weight_grads(s, copies) : Choice{-1, 1, 0};
  lhs_fast = of_lhs.tile >= 0;
  weights_fast = of_weights.tile >= 0;
  const Choice both = lhs_fast && weights_fast ? choose_both(s, copies) : Choice{-1, 1, 0};
  const bool together = both.tile >= 0 && both.cost < of_lhs.cost + of_weights.cost;
  if (together) of_lhs = both;
  if (of_lhs.splits > 1) split_sums(a, s, of_lhs.splits, &lhs.results);
  if (together) {
    e = f16 ? launch_both_grads_f16(lhs, weights, stream) : launch_both_grads_bf16(lhs, weights, stream);
  } else {
    if (lhs_fast) e = f16 ? launch_lhs_grad_f16(lhs, of_lhs.tile, stream) : launch_lhs_grad_bf16(lhs, of_lhs.tile, stream);
    if (e == hipSuccess && weights_fast)
      e = f16 ? launch_weight_grad_f16(weights, of_weights.tile, stream) : launch_weight_grad_bf16(weights, of_weights.tile, stream);
  }
  if (e == hipSuccess && of_lhs.splits > 1) e = launch_sums(a, s, of_lhs.splits, stream);
  if (e == hipSuccess && a.lhs_grad && !lhs_fast)
    e = launch_over(gated_lhs_grad_generic<Float::kF16>, gated_lhs_grad_generic<Float::kBf16>, g, s.rows * s.depth, stream);
  if (e == hipSuccess && copies && !weights_fast)
    e = launch_over(gated_weight_grad_generic<Float::kF16>, gated_weight_grad_generic<Float::kBf16>, g, s.cols * s.depth, stream);
  return e;
}

}  // namespace uk
