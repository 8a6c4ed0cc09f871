// Device-side helpers of the gated products and their backward pass: the activations, and results on their way to memory.
#ifndef IREE_AMD_CSRC_GATED_DEVICE_H_
#define IREE_AMD_CSRC_GATED_DEVICE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mx_device.h"
#include "uk_device.h"

namespace uk {

// act(x) = x s(z) or s(z), s(z) = 1 / (1 + e^-z), z = x (linear + cubic x^2); the coefficients times -log2 e, so that e^-z is one
// instruction. One formula for the three activations costs the epilogues no branch.
struct Curve {
  float linear, cubic, slope_cubic;  // slope_cubic: of dz/dx = 1 or, cubic, linear' + slope_cubic x^2
  float slope_linear;
  int32_t times;                     // whether s is multiplied by x
};
inline Curve curve_of(Activation a) {
  constexpr double kLog2e = 1.4426950408889634, kTwoRoot = 1.5957691216057308;  // 2 sqrt(2 / pi)
  if (a == Activation::kGelu)
    return {(float)(-kLog2e * kTwoRoot), (float)(-kLog2e * kTwoRoot * 0.044715), (float)(3 * kTwoRoot * 0.044715), (float)kTwoRoot, 1};
  return {(float)-kLog2e, 0, 0, 1, a == Activation::kSilu};
}

// e^-z: from 2^128 on (z below -88.7) infinite, which gives s = 0. Where x^2 is beyond f32, z is an infinity of x's sign (or, not
// cubic, 0 x infinity is kept out).
__device__ __forceinline__ float exp_minus_z(const Curve& c, float x) {
  const float square = __builtin_fminf(x * x, 1e30f);
  return __builtin_amdgcn_exp2f(x * __builtin_fmaf(c.cubic, square, c.linear));
}
__device__ __forceinline__ float activated(const Curve& c, float x) {
  const float s = __builtin_amdgcn_rcpf(1 + exp_minus_z(c, x));
  return c.times ? x * s : s;
}
// act(x) and act'(x) = s + x s (1 - s) z' or s (1 - s) z', with 1 - s = e^-z s, which loses no bits where s is near one. (Where e^-z
// is beyond 2^126, s is zero, and the limit keeps zero times infinity away.)
__device__ __forceinline__ float activated_and_slope(const Curve& c, float x, float* slope) {
  const float e = exp_minus_z(c, x), s = __builtin_amdgcn_rcpf(1 + e);
  const float rest = __builtin_fminf(e, 0x1p126f) * s;
  const float inner = __builtin_fmaf(c.slope_cubic, __builtin_fminf(x * x, 1e6f), c.slope_linear);
  const float bend = s * rest * inner;
  *slope = c.times ? __builtin_fmaf(x, bend, s) : bend;
  return c.times ? x * s : s;
}

// One element of a buffer of either kind.
template <Float T>
__device__ __forceinline__ float element(const uint8_t* p, int64_t at) {
  if constexpr (T == Float::kF32) return ((const float*)p)[at];
  else return mx_widen<T>(((const uint16_t*)p)[at]);
}
__device__ __forceinline__ float element(Float type, const uint8_t* p, int64_t at) {
  return type == Float::kF32 ? element<Float::kF32>(p, at) : type == Float::kF16 ? element<Float::kF16>(p, at) : element<Float::kBf16>(p, at);
}
__device__ __forceinline__ void put_element(Float type, uint8_t* p, int64_t at, float v) {
  if (type == Float::kF32) ((float*)p)[at] = v;
  else ((uint16_t*)p)[at] = type == Float::kF16 ? mx_narrow<Float::kF16>(v) : mx_narrow<Float::kBf16>(v);
}

}  // namespace uk

#endif  // IREE_AMD_CSRC_GATED_DEVICE_H_
