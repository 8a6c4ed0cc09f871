// Low-rank adapters of many requests at once: each row of the lhs times the `down` of its adapter, rank sums of f32 in the
// workspace, then those times its `up`.
#include "gated_device.h"

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

}  // namespace

int64_t adapter_workspace(const AdapterArgs& a) {
  if (a.count == 0) return 0;
  return (a.M * a.M0 * a.rank * 4 + 255) / 256 * 256;  // (fewer than 2^31 rows, 2^15 ranks)
}

hipError_t launch_adapter_mmt4d(const AdapterArgs& a, hipStream_t stream, const char** name) {
  const int64_t rows = a.M * a.M0;
  *name = "adapter_mmt4d_generic";
  if (a.count > 0) {
    const hipError_t e = launch_over(adapter_down_generic<Float::kF16>, adapter_down_generic<Float::kBf16>, a, rows * a.rank, stream);
    if (e != hipSuccess) return e;
  }
  return launch_over(adapter_up_generic<Float::kF16>, adapter_up_generic<Float::kBf16>, a, rows * a.N * a.N0, stream);
}

}  // namespace uk
