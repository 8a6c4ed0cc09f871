// Products of microscaled operands: the choice of kernel, and the kernel with one thread for each result, which takes
// every tile shape, stride and alignment.
#include <type_traits>

#include "mx_device.h"

namespace uk {
namespace {

constexpr int kThreads = 256;

struct MxGenericArgs {
  MxMmt4dArgs p;
  int64_t results;
};

// A block's 32 products are summed in f32, exactly (E2M1 times E2M1) or nearly so, then scaled and added to the total.
template <int LBITS>
__global__ __launch_bounds__(kThreads) void mx_mmt4d_generic(const MxGenericArgs g) {
  const MxMmt4dArgs& a = g.p;
  const int64_t tile = (int64_t)a.M0 * a.N0;
  for (int64_t n = (int64_t)blockIdx.x * kThreads + threadIdx.x; n < g.results; n += (int64_t)gridDim.x * kThreads) {
    const int64_t o = n / tile, within = n % tile;
    const int64_t i = o / a.N, j = o % a.N;
    const int64_t i0 = within / a.N0, j0 = within % a.N0;
    const int blocks = a.K0 / 32;
    const uint8_t* lhs = a.lhs + i * a.lhs_stride0;
    const uint8_t* rhs = a.rhs + j * a.rhs_stride0;
    const uint8_t* lhs_scales = a.lhs_scales + i * a.lhs_scales_stride0;
    const uint8_t* rhs_scales = a.rhs_scales + j * a.rhs_scales_stride0;
    float sum = 0;
    for (int64_t k = 0; k < a.K; ++k) {
      for (int b = 0; b < blocks; ++b) {
        const int64_t l_at = (k * a.M0 + i0) * blocks + b, r_at = (k * a.N0 + j0) * blocks + b;
        float part = 0;
        for (int s = 0; s < 4; ++s) {  // eight values at a time
          uint32_t lw[LBITS / 4], rw[1];
          __builtin_memcpy(lw, lhs + l_at * (4 * LBITS) + s * LBITS, LBITS);
          __builtin_memcpy(rw, rhs + r_at * 16 + s * 4, 4);
          float x[8], y[8];
          mx_values<LBITS>(lw, 127, x);
          mx_values<4>(rw, 127, y);
          for (int e = 0; e < 8; ++e) part += x[e] * y[e];
        }
        const int ls = lhs_scales[l_at], rs = rhs_scales[r_at];
        sum += ls == 255 || rs == 255 ? __builtin_nanf("") : ldexpf(part, ls + rs - 254);
      }
    }
    const int64_t at = i * a.out_stride0 + j * tile + within;
    if (a.out_type == Float::kF32) {
      float* out = (float*)a.out + at;
      *out = a.accumulate ? *out + sum : sum;
    } else if (a.out_type == Float::kF16) {
      uint16_t* out = (uint16_t*)a.out + at;
      *out = mx_narrow<Float::kF16>(a.accumulate ? mx_widen<Float::kF16>(*out) + sum : sum);
    } else {
      uint16_t* out = (uint16_t*)a.out + at;
      *out = mx_narrow<Float::kBf16>(a.accumulate ? mx_widen<Float::kBf16>(*out) + sum : sum);
    }
  }
}

hipError_t launch_generic(const MxMmt4dArgs& a, hipStream_t stream, const char** name) {
  MxGenericArgs g;
  g.p = a;
  g.results = a.M * a.N * a.M0 * a.N0;
  const int64_t groups = (g.results + kThreads - 1) / kThreads;
  const unsigned grid = (unsigned)(groups < (1 << 22) ? groups : 1 << 22);
  *name = "mx_mmt4d_generic";
  return a.lhs_bits == 4 ? launch_kernel(mx_mmt4d_generic<4>, grid, kThreads, 0, stream, g)
                         : launch_kernel(mx_mmt4d_generic<8>, grid, kThreads, 0, stream, g);
}

}  // namespace

hipError_t launch_mx_mmt4d(const MxMmt4dArgs& a, hipStream_t stream, const char** name) {
  return launch_generic(a, stream, name);
}

}  // namespace uk
