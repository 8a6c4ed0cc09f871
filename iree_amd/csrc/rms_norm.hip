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

// Exchanges that leave every lane of 16 (2, 4, 8 of them before) with the same value when both sides combine what they have.
template <int STEP>
__device__ __forceinline__ uint32_t exchanged(uint32_t v) {
  constexpr int PATTERN = STEP == 0 ? 0xB1 : STEP == 1 ? 0x4E : STEP == 2 ? 0x141 : 0x140;  // pairs, pairs of pairs, mirrored 8, 16
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, PATTERN, 0xF, 0xF, true);
}
template <int STEP>
__device__ __forceinline__ double exchanged(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)exchanged<STEP>((uint32_t)(w >> 32)) << 32 | exchanged<STEP>((uint32_t)w));
}
// What the rows of 16 lanes below and above (16 or 32 lanes apart) have, the same two in both.
template <bool FAR>
__device__ __forceinline__ void both(uint32_t v, uint32_t* low, uint32_t* high) {
  typedef uint32_t v2u32 __attribute__((ext_vector_type(2)));
  v2u32 p;
  if constexpr (FAR) p = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane32_swap(v, v, false, false));
  else p = __builtin_bit_cast(v2u32, __builtin_amdgcn_permlane16_swap(v, v, false, false));
  *low = p[0];
  *high = p[1];
}
template <bool FAR>
__device__ __forceinline__ double sum_of_both(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  uint32_t l0, l1, h0, h1;
  both<FAR>((uint32_t)w, &l0, &l1);
  both<FAR>((uint32_t)(w >> 32), &h0, &h1);
  return __builtin_bit_cast(double, (uint64_t)h0 << 32 | l0) + __builtin_bit_cast(double, (uint64_t)h1 << 32 | l1);
}

// The sum over the lanes of a wavefront, the same bits in every lane: both sides of an exchange add the same two numbers.
__device__ __forceinline__ double wave_sum(double v) {
  v += exchanged<0>(v);
  v += exchanged<1>(v);
  v += exchanged<2>(v);
  v += exchanged<3>(v);
  return sum_of_both<true>(sum_of_both<false>(v));
}
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  v = larger(v, exchanged<0>(v));
  v = larger(v, exchanged<1>(v));
  v = larger(v, exchanged<2>(v));
  v = larger(v, exchanged<3>(v));
  uint32_t a, b;
  both<false>(v, &a, &b);
  both<true>(larger(a, b), &a, &b);
  return larger(a, b);
}

// 1 / sqrt(v) to the last bits of f64, from the hardware's estimate: y (1 + e / 2 + 3 e^2 / 8) with e = 1 - v y^2, below 1e-7. (A
// division behind a square root is twice as many dependent steps, for every row.) Zero, infinity and NaN: the estimate's.
__device__ __forceinline__ double reciprocal_root(double v) {
  const double y = __builtin_amdgcn_rsq(v);
  const double e = __builtin_fma(-v * y, y, 1.0);
  const double better = __builtin_fma(y * e, __builtin_fma(e, 0.375, 0.5), y);
  return better == better ? better : y;
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

// Eight values at `col` of a row of `size` at `row`, all of them loaded from inside the row whether they exist or not: loads
// follow each other without a branch, and the lanes (one of a row, mostly) that begin less than eight values from its end are
// put right behind all of them.
template <Float T>
__device__ __forceinline__ void load_inside(MxEight<T>& v, const uint8_t* row, int col, int size) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  __builtin_memcpy(v.w, row + (col < size - 8 ? col : size - 8) * SIZE, MxEight<T>::kBytes);
}
template <Float T>
__device__ __forceinline__ void load_end(MxEight<T>& v, const uint8_t* row, int col, int size) {
  constexpr int SIZE = T == Float::kF32 ? 4 : 2;
  if (size - col < 8) mx_load<T>(v, row + (int64_t)col * SIZE, size - col);
}

// LANES lanes (64, or the workgroup) to a row of up to 8 * LANES * PIECES values; WEIGHT: the weight's type.
//
// 4096 rows of 8192 bf16 values, with a residual, to E4M3 (236 MB): 47.0 us, 5.0 TB/s. With the sum stored through the caches 52.4; of
// that form, 256 lanes of four pieces took 55.0 (140 registers, three wavefronts on a SIMD), 1024 of one 54.7, and a branch in
// front of every load 59.7.
//
// Sums of 16-bit types of more than 24 MiB go past the caches: also where 100 MB of other traffic and then a kernel that reads the
// sum follow, 96 us instead of 104 (2048 rows 55 and 59; 512 rows, the other way, 25.3 and 24.9). Of f32 a lane's eight values
// are two stores with gaps between the lanes, which lose more past the caches than there is to gain.
template <Float T, Float WEIGHT, NormOut OUT, int LANES, int PIECES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void rms_norm_row(const RmsNormArgs a) {
  constexpr int WAVES = LANES / 64, ROWS = LANES < 256 ? 256 / LANES : 1, SIZE = T == Float::kF32 ? 4 : 2;
  // Two of each, used in turn: who writes the next row's is past the barrier behind which the last row's were read.
  __shared__ double sums[2][WAVES];
  __shared__ uint32_t largest[2][WAVES];
  const int lane = threadIdx.x % LANES, wave = lane / 64;
  const int size = (int)a.size1, out_size = (int)a.out_size1;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x / LANES); row < a.size0;
       row += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const uint8_t* const in = a.in + row * a.in_stride0 * SIZE;
    const uint8_t* const residual = a.residual + (a.residual ? row * a.residual_stride0 * SIZE : 0);
    MxEight<T> x[PIECES], old[PIECES];
    MxEight<WEIGHT> weight[PIECES];
    if (size >= 8) {
#pragma unroll
      for (int p = 0; p < PIECES; ++p) load_inside<T>(x[p], in, (p * LANES + lane) * 8, size);
      if (a.residual) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) load_inside<T>(old[p], residual, (p * LANES + lane) * 8, size);
      }
      if (a.weight) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) load_inside<WEIGHT>(weight[p], a.weight, (p * LANES + lane) * 8, size);
      }
    }
    float s[PIECES][8];
    double part[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (p * LANES + lane) * 8;
      load_end<T>(x[p], in, col, size);
      mx_widen_eight<T>(x[p], s[p]);
      if (a.residual) {
        load_end<T>(old[p], residual, col, size);
        float o[8];
        mx_widen_eight<T>(old[p], o);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[p][i] += o[i];
        MxEight<T> rounded;
        if constexpr (T != Float::kF32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) rounded.w[i] = mx_narrow_pair<T>(s[p][2 * i], s[p][2 * i + 1]);
          mx_widen_eight<T>(rounded, s[p]);
        }
        if (a.sum && col < size) {
          uint8_t* const to = a.sum + (row * a.sum_stride0 + col) * SIZE;
          if constexpr (T != Float::kF32) {
            if (a.stream_sum && size - col >= 8) mx_store_sixteen<true>(to, rounded.w);
            else mx_store_eight<T>(to, s[p], size - col);
          } else {
            mx_store_eight<T>(to, s[p], size - col);
          }
        }
      }
      part[p] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) part[p] = __builtin_fma((double)s[p][i], (double)s[p][i], part[p]);
    }
    double squares = part[0];
#pragma unroll
    for (int p = 1; p < PIECES; ++p) squares += part[p];
    squares = wave_sum(squares);
    if constexpr (WAVES > 1) {
      if (lane % 64 == 0) sums[turn][wave] = squares;
      __syncthreads();
      squares = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) squares += sums[turn][w];
    }
    const float r = (float)reciprocal_root(squares / (double)size + (double)a.epsilon);

    uint32_t top = 0;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int col = (p * LANES + lane) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) s[p][i] *= r;
      if (a.weight) {
        load_end<WEIGHT>(weight[p], a.weight, col, size);
        float w[8];
        mx_widen_eight<WEIGHT>(weight[p], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[p][i] *= w[i];
      }
      if (size - col < 8) {  // (r may be an infinity or NaN: what does not exist is zero all the same)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[p][i] = i < size - col ? s[p][i] : 0.0f;
      }
      if constexpr (OUT != NormOut::kS8) {
        if (col < out_size) norm_store_mx<OUT>(a, row, col, s[p]);
      } else {
        top = larger(top, largest_of(s[p]));
      }
    }
    if constexpr (OUT == NormOut::kS8) {
      top = wave_largest(top);
      if constexpr (WAVES > 1) {
        if (lane % 64 == 0) largest[turn][wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = larger(top, largest[turn][w]);
      }
      const float scale = s8_scale(top), inverse = 1.0f / scale;
#pragma unroll
      for (int p = 0; p < PIECES; ++p) {
        const int col = (p * LANES + lane) * 8;
        if (col < out_size) norm_store_s8(a, row, col, s[p], scale, inverse);
      }
      if (lane == 0) *(float*)(a.scales + row * a.scales_stride0) = scale;
    }
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
    const float r = (float)reciprocal_root(squares / (double)a.size1 + (double)a.epsilon);

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

template <Float T, Float WEIGHT, NormOut OUT>
hipError_t launch(const RmsNormArgs& a, hipStream_t stream, const char** name) {
  *name = "rms_norm_row";
  const int64_t cols = a.out_size1;
  // (Workgroups beyond these numbers take the rows that are left one after the other.)
  auto at_most = [](int64_t n) { return (unsigned)(n < (1 << 20) ? n : 1 << 20); };
  const unsigned rows = at_most(a.size0), rows_by_four = at_most((a.size0 + 3) / 4);
  if (cols <= 512) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 64, 1>, rows_by_four, 256, 0, stream, a);
  // (Few rows: what counts is how long one takes.)
  if (cols <= 1024 && a.size0 > 512) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 64, 2>, rows_by_four, 256, 0, stream, a);
  if (cols <= 2048) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 256, 1>, rows, 256, 0, stream, a);
  if (cols <= 4096) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 512, 1>, rows, 512, 0, stream, a);
  if (cols <= 8192) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 512, 2>, rows, 512, 0, stream, a);
  if (cols <= 16384) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 1024, 2>, rows, 1024, 0, stream, a);
  if (cols <= 32768) return launch_kernel(rms_norm_row<T, WEIGHT, OUT, 1024, 4>, rows, 1024, 0, stream, a);
  *name = "rms_norm_long";
  return launch_kernel(rms_norm_long<T, OUT>, rows, 1024, 0, stream, a);
}

template <Float T, Float WEIGHT>
hipError_t launch_of(const RmsNormArgs& a, hipStream_t stream, const char** name) {
  switch (a.out_type) {
    case NormOut::kS8: return launch<T, WEIGHT, NormOut::kS8>(a, stream, name);
    case NormOut::kE4M3: return launch<T, WEIGHT, NormOut::kE4M3>(a, stream, name);
    default: return launch<T, WEIGHT, NormOut::kE2M1>(a, stream, name);
  }
}

}  // namespace

hipError_t launch_rms_norm(const RmsNormArgs& given, hipStream_t stream, const char** name) {
  RmsNormArgs a = given;
  const int e = float_bytes(a.type);
  a.stream_sum = a.size0 * a.size1 * e > (24ll << 20) && (uintptr_t)a.sum % 16 == 0 && a.sum_stride0 * e % 16 == 0;
  const bool f32 = a.weight_type == Float::kF32;
  switch (a.type) {
    case Float::kF32: return launch_of<Float::kF32, Float::kF32>(a, stream, name);
    case Float::kF16:
      return f32 ? launch_of<Float::kF16, Float::kF32>(a, stream, name) : launch_of<Float::kF16, Float::kF16>(a, stream, name);
    default:
      return f32 ? launch_of<Float::kBf16, Float::kF32>(a, stream, name) : launch_of<Float::kBf16, Float::kBf16>(a, stream, name);
  }
}

}  // namespace uk
