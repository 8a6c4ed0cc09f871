// Root-mean-square norm with the residual's addition, into 8-bit integers or microscaled codes: iree_uk_mi355x_rms_norm_p.
//
// Bound by memory: a value is read once with its residual, its sum written, its code written. A row stays in registers
// between the sum of its squares and its codes; rows of up to 32768 values do. A lane takes eight consecutive values at a
// time and four neighbouring lanes a block of 32, as in mx_pack.hip.
//
// Squares are summed in f64: the square of an f32 is exact there and the order of the sum does not show in r, which is
// rounded to f32 once. So a row's codes depend on the row alone, not on how many lanes share it: y = (s r) w has two f32
// roundings, and the codes one.
#include <type_traits>

#include "mx_device.h"

namespace uk {
namespace {

// The sum over the lanes of a wavefront, the same bits in every lane: an exchange adds the same two numbers on both sides.
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
    v = o > v ? o : v;
  }
  return v;
}

// The eight values of s at `col` of a row, of which `left` exist; with STORE they go to the sum.
template <Float T, bool STORE>
__device__ __forceinline__ void norm_sum(const RmsNormArgs& a, int64_t row, int64_t col, int64_t left, float s[8]) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  MxEight<T> x;
  mx_load<T>(x, a.in + (row * a.in_stride0 + col) * SIZE, left);
  mx_widen_eight<T>(x, s);
  if (!a.residual) return;
  MxEight<T> old;
  mx_load<T>(old, a.residual + (row * a.residual_stride0 + col) * SIZE, left);
  float o[8];
  mx_widen_eight<T>(old, o);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    s[i] += o[i];
    if constexpr (T != Float::kF32) s[i] = mx_widen<T>(mx_narrow<T>(s[i]));
  }
  if (STORE && a.sum && left > 0) mx_store_eight<T>(a.sum + (row * a.sum_stride0 + col) * SIZE, s, left);
}

__device__ __forceinline__ void norm_weight(const RmsNormArgs& a, int64_t col, int64_t left, float w[8]) {
  if (!a.weight) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.0f;
  } else if (a.weight_type == Float::kF32) {
    MxEight<Float::kF32> v;
    mx_load<Float::kF32>(v, a.weight + col * 4, left);
    mx_widen_eight<Float::kF32>(v, w);
  } else if (a.weight_type == Float::kF16) {
    MxEight<Float::kF16> v;
    mx_load<Float::kF16>(v, a.weight + col * 2, left);
    mx_widen_eight<Float::kF16>(v, w);
  } else {
    MxEight<Float::kBf16> v;
    mx_load<Float::kBf16>(v, a.weight + col * 2, left);
    mx_widen_eight<Float::kBf16>(v, w);
  }
}

// y, with zeros where there is no value (r may be an infinity or NaN).
__device__ __forceinline__ void norm_scaled(float s[8], const float w[8], float r, int64_t left) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i] = i < left ? s[i] * r * w[i] : 0.0f;
}

__device__ __forceinline__ uint32_t largest_of(const float y[8]) {
  MxEight<Float::kF32> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.w[i] = __builtin_bit_cast(uint32_t, y[i]);
  return mx_largest<Float::kF32>(v);
}

template <NormOut OUT>
__device__ __forceinline__ void norm_store_mx(const RmsNormArgs& a, int64_t row, int64_t col, const float y[8]) {
  constexpr int BITS = OUT == NormOut::kE2M1 ? 4 : 8;
  MxEight<Float::kF32> v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v.w[i] = __builtin_bit_cast(uint32_t, y[i]);
  const uint32_t b = mx_scale_byte<BITS>(mx_largest_of_block(mx_largest<Float::kF32>(v)));
  uint32_t codes[BITS / 4];
  mx_codes<BITS, Float::kF32>(v, b, codes);
  __builtin_memcpy(a.out + row * a.out_stride0 + col / 8 * BITS, codes, BITS);
  if (threadIdx.x % 4 == 0) a.scales[row * a.scales_stride0 + col / 32] = (uint8_t)b;
}

// A row's scale from its largest magnitude: a NaN where that is not finite.
__device__ __forceinline__ float s8_scale(uint32_t largest) {
  if (largest >= 0x7F800000u) return __builtin_nanf("");
  const float scale = __builtin_bit_cast(float, largest) / 127.0f;
  return scale < 0x1p-126f ? 0x1p-126f : scale;
}

__device__ __forceinline__ void norm_store_s8(const RmsNormArgs& a, int64_t row, int64_t col, const float y[8], float scale,
                                              float inverse) {
  uint32_t q[2] = {0, 0};
  if (scale == scale) {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i / 4] |= ((uint32_t)(int)rintf(y[i] * inverse) & 0xFFu) << (8 * (i % 4));
  }
  uint8_t* out = a.out + row * a.out_stride0 + col;
  const int64_t left = a.out_size1 - col;
  if (left >= 8) {
    __builtin_memcpy(out, q, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) out[i] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
  }
}

// LANES lanes (64, or the workgroup) to a row of up to 8 * LANES * PIECES values.
template <Float T, NormOut OUT, int LANES, int PIECES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void rms_norm_row(const RmsNormArgs a) {
  constexpr int WAVES = LANES / 64, ROWS = LANES < 256 ? 256 / LANES : 1;
  // Two of each, used in turn: who writes the next row's is past the barrier behind which the last row's were read.
  __shared__ double sums[2][WAVES];
  __shared__ uint32_t largest[2][WAVES];
  const int lane = threadIdx.x % LANES, wave = lane / 64;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < a.size0; row += (int64_t)gridDim.x * ROWS) {
    float s[PIECES][8];
    double squares = 0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t col = (int64_t)(p * LANES + lane) * 8;
      norm_sum<T, true>(a, row, col, a.size1 - col, s[p]);
#pragma unroll
      for (int i = 0; i < 8; ++i) squares += (double)s[p][i] * (double)s[p][i];
    }
    squares = wave_sum(squares);
    if constexpr (WAVES > 1) {
      if (lane % 64 == 0) sums[turn][wave] = squares;
      __syncthreads();
      squares = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) squares += sums[turn][w];
    }
    const float r = (float)(1.0 / sqrt(squares / (double)a.size1 + (double)a.epsilon));

    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t col = (int64_t)(p * LANES + lane) * 8, left = a.size1 - col;
      float w[8];
      norm_weight(a, col, left, w);
      norm_scaled(s[p], w, r, left);
      if constexpr (OUT != NormOut::kS8) {
        if (col < a.out_size1) norm_store_mx<OUT>(a, row, col, s[p]);
      } else {
        const uint32_t m = largest_of(s[p]);
        top = m > top ? m : top;
      }
    }
    if constexpr (OUT == NormOut::kS8) {
      top = wave_largest(top);
      if constexpr (WAVES > 1) {
        if (lane % 64 == 0) largest[turn][wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = largest[turn][w] > top ? largest[turn][w] : top;
      }
      const float scale = s8_scale(top), inverse = 1.0f / scale;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int64_t col = (int64_t)(p * LANES + lane) * 8;
        if (col < a.out_size1) norm_store_s8(a, row, col, s[p], scale, inverse);
      }
      if (lane == 0) *(float*)(a.scales + row * a.scales_stride0) = scale;
    }
    turn ^= 1;
  }
}

// Rows of any length, read again for each step. (The sum may lie where `in` or the residual does: once it is written, it
// is what is read.)
template <Float T, NormOut OUT>
__global__ __launch_bounds__(1024) void rms_norm_long(const RmsNormArgs a) {
  constexpr int LANES = 1024, WAVES = LANES / 64;
  __shared__ double sums[2][WAVES];
  __shared__ uint32_t largest[2][WAVES];
  const int lane = threadIdx.x, wave = lane / 64;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.size0; row += gridDim.x, turn ^= 1) {
    double squares = 0;
    for (int64_t col = lane * 8; col < a.size1; col += LANES * 8) {
      float s[8];
      norm_sum<T, true>(a, row, col, a.size1 - col, s);
  #pragma unroll
      for (int i = 0; i < 8; ++i) squares += (double)s[i] * (double)s[i];
    }
    squares = wave_sum(squares);
    if (lane % 64 == 0) sums[turn][wave] = squares;
    __syncthreads();
    squares = 0;
  #pragma unroll
    for (int w = 0; w < WAVES; ++w) squares += sums[turn][w];
    const float r = (float)(1.0 / sqrt(squares / (double)a.size1 + (double)a.epsilon));

    RmsNormArgs again = a;  // (a lane reads back what it has written itself)
    if (a.sum) {
      again.in = a.sum;
      again.in_stride0 = a.sum_stride0;
      again.residual = nullptr;
    }
    auto y_at = [&](int64_t col, float y[8]) {
      const int64_t left = a.size1 - col;
      float w[8];
      norm_sum<T, false>(again, row, col, left, y);
      norm_weight(a, col, left, w);
      norm_scaled(y, w, r, left);
    };
    if constexpr (OUT != NormOut::kS8) {
      for (int64_t col = lane * 8; col < a.out_size1; col += LANES * 8) {
        float y[8];
        y_at(col, y);
        norm_store_mx<OUT>(a, row, col, y);
      }
    } else {
      uint32_t top = 0;
      for (int64_t col = lane * 8; col < a.size1; col += LANES * 8) {
        float y[8];
        y_at(col, y);
        const uint32_t m = largest_of(y);
        top = m > top ? m : top;
      }
      top = wave_largest(top);
      if (lane % 64 == 0) largest[turn][wave] = top;
      __syncthreads();
  #pragma unroll
      for (int w = 0; w < WAVES; ++w) top = largest[turn][w] > top ? largest[turn][w] : top;
      const float scale = s8_scale(top), inverse = 1.0f / scale;
      for (int64_t col = lane * 8; col < a.out_size1; col += LANES * 8) {
        float y[8];
        y_at(col, y);
        norm_store_s8(a, row, col, y, scale, inverse);
      }
      if (lane == 0) *(float*)(a.scales + row * a.scales_stride0) = scale;
    }
  }
}

template <Float T, NormOut OUT>
hipError_t launch(const RmsNormArgs& a, hipStream_t stream, const char** name) {
  *name = "rms_norm_row";
  const int64_t cols = a.out_size1;
  // (Workgroups beyond these numbers take the rows that are left one after the other.)
  auto at_most = [](int64_t n) { return (unsigned)(n < (1 << 20) ? n : 1 << 20); };
  const unsigned rows = at_most(a.size0), rows_by_four = at_most((a.size0 + 3) / 4);
  if (cols <= 512) return launch_kernel(rms_norm_row<T, OUT, 64, 1>, rows_by_four, 256, 0, stream, a);
  if (cols <= 1024) return launch_kernel(rms_norm_row<T, OUT, 64, 2>, rows_by_four, 256, 0, stream, a);
  if (cols <= 2048) return launch_kernel(rms_norm_row<T, OUT, 256, 1>, rows, 256, 0, stream, a);
  if (cols <= 4096) return launch_kernel(rms_norm_row<T, OUT, 256, 2>, rows, 256, 0, stream, a);
  if (cols <= 8192) {
    // Few rows: what counts is how long one takes.
    if (rows <= 256) return launch_kernel(rms_norm_row<T, OUT, 1024, 1>, rows, 1024, 0, stream, a);
    return launch_kernel(rms_norm_row<T, OUT, 256, 4>, rows, 256, 0, stream, a);
  }
  if (cols <= 16384) return launch_kernel(rms_norm_row<T, OUT, 1024, 2>, rows, 1024, 0, stream, a);
  if (cols <= 32768) return launch_kernel(rms_norm_row<T, OUT, 1024, 4>, rows, 1024, 0, stream, a);
  *name = "rms_norm_long";
  return launch_kernel(rms_norm_long<T, OUT>, rows, 1024, 0, stream, a);
}

template <Float T>
hipError_t launch_of(const RmsNormArgs& a, hipStream_t stream, const char** name) {
  switch (a.out_type) {
    case NormOut::kS8: return launch<T, NormOut::kS8>(a, stream, name);
    case NormOut::kE4M3: return launch<T, NormOut::kE4M3>(a, stream, name);
    default: return launch<T, NormOut::kE2M1>(a, stream, name);
  }
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& a, hipStream_t stream, const char** name) {
  switch (a.type) {
    case Float::kF32: return launch_of<Float::kF32>(a, stream, name);
    case Float::kF16: return launch_of<Float::kF16>(a, stream, name);
    default: return launch_of<Float::kBf16>(a, stream, name);
  }
}

}  // namespace uk
