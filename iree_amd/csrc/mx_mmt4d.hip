// Products of microscaled operands: the choice of kernel, and the kernel with one thread for each result, which takes
// every tile shape, stride and alignment.
#include <type_traits>

#include "mx_mmt4d.h"

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

// Whether a row of an operand's tiles has its K in chunks of 128 that lie a tile apart.
bool in_chunks(int32_t tile_rows, int32_t k0) { return tile_rows == 1 || k0 == 128; }

bool aligned(const void* p, int64_t stride, int64_t rows, int64_t to) {
  return (uintptr_t)p % to == 0 && (rows == 1 || stride % to == 0);
}

// The problem as the fast kernels take it; false: they do not.
bool as_product(const MxMmt4dArgs& a, MxProduct* p) {
  const int64_t rows = a.M * a.M0, cols = a.N * a.N0, depth = a.K * a.K0;
  if (depth == 0 || depth % 128 != 0 || depth / 128 > 0x7FFFFFFF || !in_chunks(a.M0, a.K0) || !in_chunks(a.N0, a.K0)) return false;
  if (rows > 0x7FFFFFFF - 256 || cols > 0x7FFFFFFF - 256) return false;
  if (!aligned(a.lhs, a.lhs_stride0, a.M, 16) || !aligned(a.rhs, a.rhs_stride0, a.N, 16) ||
      !aligned(a.lhs_scales, a.lhs_scales_stride0, a.M, 4) || !aligned(a.rhs_scales, a.rhs_scales_stride0, a.N, 4))
    return false;
  const int out_bytes = float_bytes(a.out_type);
  p->lhs = {a.lhs, a.lhs_scales, a.lhs_stride0, a.lhs_scales_stride0, (uint32_t)rows, (uint32_t)a.M0, reciprocal_of((uint32_t)a.M0)};
  p->rhs = {a.rhs, a.rhs_scales, a.rhs_stride0, a.rhs_scales_stride0, (uint32_t)cols, (uint32_t)a.N0, reciprocal_of((uint32_t)a.N0)};
  p->out = a.out;
  p->out_stride0 = a.out_stride0;
  p->chunks = (uint32_t)(depth / 128);
  p->n0 = (uint32_t)a.N0;
  p->n0_reciprocal = reciprocal_of((uint32_t)a.N0);
  p->out_tile = (uint32_t)a.M0 * (uint32_t)a.N0;
  p->out_type = a.out_type;
  p->accumulate = a.accumulate;
  // (Tiles one row tall and one column wide are a row-major result.)
  if (a.M0 == 1 && a.N0 == 1) {
    p->n0 = p->rhs.rows;
    p->n0_reciprocal = reciprocal_of(p->n0);
    p->out_tile = 0;
  }
  p->fours = (p->n0 % 4 == 0 || (a.M0 == 1 && a.N0 == 1)) && aligned(a.out, a.out_stride0 * out_bytes, a.M, 4 * out_bytes);
  return true;
}

}  // namespace

hipError_t launch_mx_mmt4d(const MxMmt4dArgs& a, hipStream_t stream, const char** name) {
  MxProduct p;
  if (as_product(a, &p)) return launch_mx_few(p, a.lhs_bits, stream, name);
  return launch_generic(a, stream, name);
}

}  // namespace uk
