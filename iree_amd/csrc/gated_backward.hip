// The backward pass of gated products: the gradients of the two products, rounded to the operands' type, into the workspace, then
// the products that give the gradients of lhs, gate and up.
#include "gated_backward.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

// The workspace: [rows][2 * cols] of the operands' type, a row's dg then its du, each filled up with zeros to a multiple of eight.
struct Sizes {
  int64_t rows, cols, depth, pitch;
  explicit Sizes(const GatedBackwardArgs& a)
      : rows(a.M * a.M0), cols(a.N * a.N0), depth(a.K * a.K0), pitch(2 * ((cols + 7) / 8 * 8)) {}
};

struct BackwardArgs {
  GatedBackwardArgs p;
  Curve curve;
  int64_t rows, cols, depth, pitch, results;
};

template <Float T>
__global__ __launch_bounds__(kThreads) void gated_backward_generic(const BackwardArgs g) {
  const GatedBackwardArgs& a = g.p;
  const int64_t half = g.pitch / 2;
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
    uint16_t* to = (uint16_t*)a.workspace + row * g.pitch + col;
    to[0] = mx_narrow<T>(dg);
    to[half] = mx_narrow<T>(du);
  }
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
    put_element(a.out_type, a.lhs_grad, row / a.M0 * a.lhs_grad_stride0 + (k / a.K0 * a.M0 + row % a.M0) * a.K0 + k % a.K0, sum);
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

// The first step where eight columns at a time lie next to each other, aligned: a thread for eight.
struct FirstStep {
  const uint8_t *gate_pre, *up_pre, *out_grad;
  uint8_t* grads;
  Layout gate_at, up_at, out_at;
  Curve curve;
  int64_t results;  // eights
  uint32_t half, half_reciprocal;  // eights of a row's dg
  int64_t pitch;
  Float pre_type, out_type;
};
template <Float T>
__global__ __launch_bounds__(kThreads) void gated_backward_first(const FirstStep p) {
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
    }
    const int64_t to = (int64_t)row * p.pitch + col;
    store_run<T, 8>(p.grads, to, g);
    store_run<T, 8>(p.grads, to + p.pitch / 2, u);
  }
}

hipError_t launch_over(void (*f16)(const BackwardArgs), void (*bf16)(const BackwardArgs), BackwardArgs& g, int64_t results, hipStream_t stream) {
  if (results == 0) return hipSuccess;
  g.results = results;
  const int64_t groups = (results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  return launch_kernel(g.p.type == Float::kF16 ? f16 : bf16, grid, kThreads, 0, stream, g);
}

GradResults results_of(const GatedBackwardArgs& a, const Layout& at, uint8_t* first, uint8_t* second, int64_t stride0, int64_t stride1,
                       int64_t rows, int64_t panels, bool accumulate) {
  GradResults r;
  r.out[0] = first; r.out[1] = second;
  r.stride0[0] = stride0; r.stride0[1] = stride1;
  r.at = at;
  r.type = a.out_type;
  r.accumulate = accumulate;
  const int e = float_bytes(a.out_type);
  Layout other = at;
  other.stride0 = stride1;
  r.runs = runs_of(at, first, panels, e, 16 / e, 16) && (!second || runs_of(other, second, panels, e, 16 / e, 16));
  r.rows = (uint32_t)rows;
  r.tile_rows_of_first = 0;
  r.results = second ? 2 : 1;
  return r;
}

// Which tile: the least of the times that a model gives, in microseconds: a start, and chunks of K times what one of them takes with one
// workgroup on a compute unit and, where LDS and registers hold two, with two; more than that follow each other. Fitted to the times of
// every tile in 260 problems from 16 to 4096 rows, 64 to 28672 columns, K of 64 to 14336; over these the tile taken is slower than the
// best one by 0.6 % (lhs) and 1.6 % (weights) in the mean. -1: none can.
struct Times { float start, one, two, start_again; };  // two = 0: one workgroup on a compute unit
int choose_tile(const Times* times, int64_t rows, int64_t cols, int64_t chunks, int64_t results) {
  int best = -1;
  float least = 0;
  for (int i = 0; i < (int)(sizeof kGradTiles / sizeof kGradTiles[0]); ++i) {
    const GradTile& t = kGradTiles[i];
    const int64_t tiles = (rows + t.rows - 1) / t.rows * ((cols + t.cols - 1) / t.cols) * results, rounds = (tiles + 255) / 256;
    if (tiles > (1 << 23)) continue;  // (a grid has fewer than 2^32 threads)
    const Times& of = times[i];
    const float steps = (float)chunks * (of.two == 0 ? rounds * of.one : (rounds >> 1) * of.two + (rounds & 1) * of.one);
    const float cost = of.start + (rounds - 1) * of.start_again + steps;
    if (best < 0 || cost < least) {
      least = cost;
      best = i;
    }
  }
  return best;
}
constexpr Times kLhsGradTimes[] = {{16.2f, .491f, 0, 21.5f},   {11.3f, .299f, 0, 11.7f},  {11.4f, .334f, .834f, 4.3f}, {9.1f, .220f, .555f, 2.3f},
                                   {7.7f, .157f, .418f, 1.1f}, {7.6f, .159f, .361f, 1.3f}, {6.6f, .137f, .246f, .9f}};
constexpr Times kWeightGradTimes[] = {{17.3f, .522f, 0, 15.6f},   {11.9f, .323f, 0, 8.5f},   {11.6f, .303f, .747f, 4.1f}, {8.8f, .196f, .448f, 2.4f},
                                      {7.4f, .171f, .303f, 1.6f}, {7.3f, .164f, .313f, 1.6f}, {6.3f, .141f, .210f, 1.1f}};

// false: the general kernel takes it.
bool launch_lhs_grad(const GatedBackwardArgs& a, const Sizes& s, hipStream_t stream, hipError_t* e) {
  LhsGradProduct p;
  Strided16 up;
  if (s.rows == 0 || s.cols == 0 || s.cols > 0x7FFFFFFF - 512) return false;
  if (!as_operand16(a.workspace, s.pitch, s.rows, 1, s.cols, 1, &p.grads) || !near16(p.grads, 256) ||
      !as_strided16(a.gate, a.gate_stride0, a.N, a.N0, a.K, a.K0, &p.gate) || !as_strided16(a.up, a.up_stride0, a.N, a.N0, a.K, a.K0, &up))
    return false;
  p.up = up.data;
  p.up_stride0 = up.stride0;
  p.lhs_second = s.pitch;  // (half of a row's bytes)
  p.depth = (uint32_t)s.cols;
  p.results = results_of(a, layout_of(a.lhs_grad_stride0, a.M0, a.K, a.K0), a.lhs_grad, nullptr, a.lhs_grad_stride0, 0, s.rows, a.M, false);
  const int tile = choose_tile(kLhsGradTimes, s.rows, s.depth, 2 * ((s.cols + 31) / 32), 1);
  if (tile < 0) return false;
  *e = a.type == Float::kF16 ? launch_lhs_grad_f16(p, tile, stream) : launch_lhs_grad_bf16(p, tile, stream);
  return true;
}
bool launch_weight_grads(const GatedBackwardArgs& a, const Sizes& s, hipStream_t stream, hipError_t* e) {
  WeightGradProduct p;
  if (s.rows == 0 || s.cols == 0 || s.rows > 0x7FFFFFFF || s.cols > 0x7FFFFFFF - 512) return false;
  const uint8_t* const grads = a.workspace + (a.gate_grad ? 0 : s.pitch);
  // (As many columns of dg as there are with the zeros that fill up an eight.)
  if (!as_strided16(grads, s.pitch, s.rows, 1, s.pitch / 2, 1, &p.grads) || !as_strided16(a.lhs, a.lhs_stride0, a.M, a.M0, a.K, a.K0, &p.lhs))
    return false;
  p.lhs_second = s.pitch;
  p.depth = (uint32_t)s.rows;
  uint8_t* const first = a.gate_grad ? a.gate_grad : a.up_grad;
  uint8_t* const second = a.gate_grad ? a.up_grad : nullptr;
  const int64_t stride0 = a.gate_grad ? a.gate_grad_stride0 : a.up_grad_stride0;
  p.results = results_of(a, layout_of(stride0, a.N0, a.K, a.K0), first, second, stride0, a.up_grad_stride0, s.cols, a.N, a.accumulate);
  const int tile = choose_tile(kWeightGradTimes, s.cols, s.depth, (s.rows + 31) / 32, p.results.results);
  if (tile < 0) return false;
  *e = a.type == Float::kF16 ? launch_weight_grad_f16(p, tile, stream) : launch_weight_grad_bf16(p, tile, stream);
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
  const int64_t groups = (p.results + kThreads - 1) / kThreads;
  *e = launch_kernel(a.type == Float::kF16 ? gated_backward_first<Float::kF16> : gated_backward_first<Float::kBf16>,
                     (unsigned)(groups < (1 << 22) ? groups : 1 << 22), kThreads, 0, stream, p);
  return true;
}

}  // namespace

int64_t gated_backward_workspace(const GatedBackwardArgs& a) {
  const Sizes s(a);
  int64_t bytes;
  if (__builtin_mul_overflow(s.rows, 2 * s.pitch, &bytes) || bytes > INT64_MAX - 256) return -1;
  return (bytes + 255) / 256 * 256;
}

hipError_t launch_gated_backward(const GatedBackwardArgs& a, hipStream_t stream, const char** name) {
  const Sizes s(a);
  BackwardArgs g;
  g.p = a;
  g.curve = curve_of(a.activation);
  g.rows = s.rows; g.cols = s.cols; g.depth = s.depth; g.pitch = s.pitch;
  *name = "gated_backward";
  hipError_t e = hipSuccess;
  if (!launch_first(a, s, stream, &e))
    e = launch_over(gated_backward_generic<Float::kF16>, gated_backward_generic<Float::kBf16>, g, s.rows * (s.pitch / 2), stream);
  if (e == hipSuccess && a.lhs_grad && !launch_lhs_grad(a, s, stream, &e))
    e = launch_over(gated_lhs_grad_generic<Float::kF16>, gated_lhs_grad_generic<Float::kBf16>, g, s.rows * s.depth, stream);
  if (e == hipSuccess && (a.gate_grad || a.up_grad) && !launch_weight_grads(a, s, stream, &e))
    e = launch_over(gated_weight_grad_generic<Float::kF16>, gated_weight_grad_generic<Float::kBf16>, g, s.cols * s.depth, stream);
  return e;
}

}  // namespace uk
