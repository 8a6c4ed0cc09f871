// The backward pass of gated products: the gradients of the two products, rounded to the operands' type, into the workspace, then
// the products that give the gradients of lhs, gate and up.
#include "gated_device.h"

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

hipError_t launch_over(void (*f16)(const BackwardArgs), void (*bf16)(const BackwardArgs), BackwardArgs& g, int64_t results, hipStream_t stream) {
  if (results == 0) return hipSuccess;
  g.results = results;
  const int64_t groups = (results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  return launch_kernel(g.p.type == Float::kF16 ? f16 : bf16, grid, kThreads, 0, stream, g);
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
  *name = "gated_backward_generic";
  hipError_t e = launch_over(gated_backward_generic<Float::kF16>, gated_backward_generic<Float::kBf16>, g, s.rows * (s.pitch / 2), stream);
  if (e == hipSuccess && a.lhs_grad)
    e = launch_over(gated_lhs_grad_generic<Float::kF16>, gated_lhs_grad_generic<Float::kBf16>, g, s.rows * s.depth, stream);
  if (e == hipSuccess && (a.gate_grad || a.up_grad))
    e = launch_over(gated_weight_grad_generic<Float::kF16>, gated_weight_grad_generic<Float::kBf16>, g, s.cols * s.depth, stream);
  return e;
}

}  // namespace uk
