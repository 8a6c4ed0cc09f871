// Gated products: the choice of kernel, and the kernel with one thread for each result, which takes every tile shape, stride and
// alignment.
#include "gated_device.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

struct GenericArgs {
  GatedArgs p;
  Curve curve;
  int64_t results;
};

template <Float T>
__global__ __launch_bounds__(kThreads) void gated_mmt4d_generic(const GenericArgs g) {
  const GatedArgs& a = g.p;
  const int64_t tile = (int64_t)a.M0 * a.N0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t o = n / tile, within = n % tile;
    const int64_t i = o / a.N, j = o % a.N;
    const int64_t i0 = within / a.N0, j0 = within % a.N0;
    const uint16_t* lhs = (const uint16_t*)a.lhs + i * a.lhs_stride0 + i0 * a.K0;
    const uint16_t* gate = (const uint16_t*)a.gate + j * a.gate_stride0 + j0 * a.K0;
    const uint16_t* up = (const uint16_t*)a.up + j * a.up_stride0 + j0 * a.K0;
    float sum_g = 0, sum_u = 0;
    for (int64_t k = 0; k < a.K; ++k) {
      for (int k0 = 0; k0 < a.K0; ++k0) {
        const float x = mx_widen<T>(lhs[k * a.M0 * a.K0 + k0]);
        sum_g += x * mx_widen<T>(gate[k * a.N0 * a.K0 + k0]);
        sum_u += x * mx_widen<T>(up[k * a.N0 * a.K0 + k0]);
      }
    }
    const int64_t in_row = j * tile + within;
    const int64_t gate_at = i * a.gate_pre_stride0 + in_row, up_at = i * a.up_pre_stride0 + in_row;
    if (a.pre_load) {
      sum_g += element(a.pre_type, a.gate_pre, gate_at);
      sum_u += element(a.pre_type, a.up_pre, up_at);
    }
    if (a.pre_store) {
      put_element(a.pre_type, a.gate_pre, gate_at, sum_g);
      put_element(a.pre_type, a.up_pre, up_at, sum_u);
    }
    put_element(a.out_type, a.out, i * a.out_stride0 + in_row, activated(g.curve, sum_g) * sum_u);
  }
}

hipError_t launch_generic(const GatedArgs& a, hipStream_t stream, const char** name) {
  GenericArgs g;
  g.p = a;
  g.curve = curve_of(a.activation);
  g.results = a.M * a.N * a.M0 * a.N0;
  const int64_t groups = (g.results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  *name = "gated_mmt4d_generic";
  return a.type == Float::kF16 ? launch_kernel(gated_mmt4d_generic<Float::kF16>, grid, kThreads, 0, stream, g)
                               : launch_kernel(gated_mmt4d_generic<Float::kBf16>, grid, kThreads, 0, stream, g);
}

}  // namespace

hipError_t launch_gated_mmt4d(const GatedArgs& a, hipStream_t stream, const char** name) { return launch_generic(a, stream, name); }

}  // namespace uk
