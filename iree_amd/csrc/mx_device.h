// Device-side helpers of the microscaled kernels: eight values of a block at a time, on their way into or out of codes.
//
// Microscaling: 32 consecutive values along K share a scale 2^(b - 127), b a byte (E8M0), and are codes of E2M1 (sign, 2
// exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or E4M3 (up to 448). Four neighbouring lanes hold a block.
#ifndef IREE_AMD_CSRC_MX_DEVICE_H_
#define IREE_AMD_CSRC_MX_DEVICE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "uk_internal.h"

namespace uk {

typedef float mx_v2f32 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_v2bf16 __attribute__((ext_vector_type(2)));
typedef _Float16 mx_v2f16 __attribute__((ext_vector_type(2)));
typedef short mx_v2s16 __attribute__((ext_vector_type(2)));
typedef unsigned short mx_v2u16 __attribute__((ext_vector_type(2)));

// IEEE widening and narrowing, subnormals kept (the conversions of the reference's own types, which flush them, are
// uk_device.h's; these operators have no counterpart there).
template <Float T>
__device__ __forceinline__ float mx_widen(uint16_t h) {
  if constexpr (T == Float::kBf16) return __builtin_bit_cast(float, (uint32_t)h << 16);
  else return (float)__builtin_bit_cast(_Float16, h);
}
template <Float T>
__device__ __forceinline__ uint16_t mx_narrow(float f) {
  if constexpr (T == Float::kBf16) return __builtin_bit_cast(uint16_t, (__bf16)f);
  else return __builtin_bit_cast(uint16_t, (_Float16)f);
}
// Two of them in a word.
template <Float T>
__device__ __forceinline__ uint32_t mx_narrow_pair(float a, float b) {
  if constexpr (T == Float::kBf16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_v2f32{a, b}, mx_v2bf16));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(mx_v2f32{a, b}, mx_v2f16));
}

// Eight consecutive values as they lie in memory: 4 words of a 16-bit type, 8 of f32.
template <Float T>
struct MxEight {
  static constexpr int kWords = T == Float::kF32 ? 8 : 4, kBytes = kWords * 4;
  uint32_t w[kWords];
};

// STREAM: past the caches.
template <Float T, bool STREAM>
__device__ __forceinline__ void mx_load_eight(MxEight<T>& v, const uint8_t* p) {
  if constexpr (STREAM) {
    typedef uint32_t unaligned_v4u32 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
    for (int i = 0; i < MxEight<T>::kBytes / 16; ++i) {
      const unaligned_v4u32 q = __builtin_nontemporal_load((const unaligned_v4u32*)p + i);
      __builtin_memcpy(v.w + 4 * i, &q, 16);
    }
  } else {
    __builtin_memcpy(v.w, p, MxEight<T>::kBytes);
  }
}

// `count` of them exist (any number, also none or more); the others are zero. The address is a multiple of the element's
// size and of nothing more: a row of an odd length starts anywhere, and loads of 16 bytes need no alignment here.
template <Float T, bool STREAM = false>
__device__ __forceinline__ void mx_load(MxEight<T>& v, const uint8_t* p, int64_t count) {
  if (count >= 8) {
    mx_load_eight<T, STREAM>(v, p);
    return;
  }
#pragma unroll
  for (int i = 0; i < MxEight<T>::kWords; ++i) {
    if constexpr (T == Float::kF32) {
      v.w[i] = i < count ? ((const uint32_t*)p)[i] : 0;
    } else {
      v.w[i] = (2 * i < count ? ((const uint16_t*)p)[2 * i] : 0u) |
               (2 * i + 1 < count ? (uint32_t)((const uint16_t*)p)[2 * i + 1] << 16 : 0u);
    }
  }
}

template <Float T>
__device__ __forceinline__ void mx_widen_eight(const MxEight<T>& v, float f[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (T == Float::kF32) f[i] = __builtin_bit_cast(float, v.w[i]);
    else f[i] = mx_widen<T>((uint16_t)(v.w[i / 2] >> (16 * (i & 1))));
  }
}

// 16 bytes to an address of any alignment; STREAM: past the caches.
template <bool STREAM>
__device__ __forceinline__ void mx_store_sixteen(uint8_t* p, const uint32_t w[4]) {
  typedef uint32_t unaligned_v4u32 __attribute__((ext_vector_type(4), aligned(1)));
  if constexpr (STREAM) __builtin_nontemporal_store(unaligned_v4u32{w[0], w[1], w[2], w[3]}, (unaligned_v4u32*)p);
  else __builtin_memcpy(p, w, 16);
}

// Eight f32 values to memory as T, the first `count` of them.
template <Float T>
__device__ __forceinline__ void mx_store_eight(uint8_t* p, const float f[8], int64_t count) {
  if (count >= 8) {
    uint32_t w[MxEight<T>::kWords];
#pragma unroll
    for (int i = 0; i < MxEight<T>::kWords; ++i) {
      if constexpr (T == Float::kF32) w[i] = __builtin_bit_cast(uint32_t, f[i]);
      else w[i] = mx_narrow_pair<T>(f[2 * i], f[2 * i + 1]);
    }
    __builtin_memcpy(p, w, sizeof w);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (i >= count) continue;
    if constexpr (T == Float::kF32) ((float*)p)[i] = f[i];
    else ((uint16_t*)p)[i] = mx_narrow<T>(f[i]);
  }
}

// The largest magnitude of eight values, as the bits of an f32. Magnitudes compare as integers do, an infinity and NaNs
// above every number, so that a block with one of them is known by its maximum.
template <Float T>
__device__ __forceinline__ uint32_t mx_largest(const MxEight<T>& v) {
  if constexpr (T == Float::kF32) {
    uint32_t m = v.w[0] & 0x7FFFFFFFu;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      const uint32_t x = v.w[i] & 0x7FFFFFFFu;
      m = x > m ? x : m;
    }
    return m;
  } else {
    mx_v2u16 m = __builtin_bit_cast(mx_v2u16, v.w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(mx_v2u16, v.w[i] & 0x7FFF7FFFu));
    const uint16_t both = m[0] > m[1] ? m[0] : m[1];
    return __builtin_bit_cast(uint32_t, mx_widen<T>(both));
  }
}

// The maximum over the four lanes of a block (lanes 4i to 4i + 3, all of them active).
__device__ __forceinline__ uint32_t mx_largest_of_block(uint32_t m) {
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true);  // lanes 1 0 3 2
  m = o > m ? o : m;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true);           // lanes 2 3 0 1
  return o > m ? o : m;
}

// floor(log2) of a normal f32 is its exponent field; below 2^-126 the scale is the least one whatever it is.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t largest) {
  constexpr int EMAX = BITS == 4 ? 2 : 8;
  const int field = (int)(largest >> 23);
  const int b = field > EMAX ? field - EMAX : 0;
  return field == 255 ? 255u : (uint32_t)b;
}
// 2^(b - 127), b below 255; 2^-127 is subnormal.
__device__ __forceinline__ float mx_scale_value(uint32_t b) {
  return __builtin_bit_cast(float, b == 0 ? 0x00400000u : b << 23);
}

// Eight values over 2^(b - 127) -> their codes: one word of 4-bit ones, two of 8-bit ones; the first lowest. The conversion
// instructions round to nearest even and keep the sign of zero; E2M1 saturates, E4M3 (NaN from 464 on) has to be kept
// below 448. All zero where b is 255.
template <int BITS, Float T>
__device__ __forceinline__ void mx_codes(const MxEight<T>& v, uint32_t b, uint32_t codes[BITS / 4]) {
  const float scale = mx_scale_value(b);
  if constexpr (BITS == 4) {
    uint32_t c = 0;
    auto pair = [&](uint32_t old, int i, auto sel) {
      constexpr int SEL = decltype(sel)::value;
      if constexpr (T == Float::kF32)
        return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, __builtin_bit_cast(float, v.w[2 * i]),
                                                                  __builtin_bit_cast(float, v.w[2 * i + 1]), scale, SEL);
      else if constexpr (T == Float::kF16)
        return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_f16(old, __builtin_bit_cast(mx_v2f16, v.w[i]), scale, SEL);
      else
        return (uint32_t)__builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(old, __builtin_bit_cast(mx_v2bf16, v.w[i]), scale, SEL);
    };
    c = pair(c, 0, std::integral_constant<int, 0>{});
    c = pair(c, 1, std::integral_constant<int, 1>{});
    c = pair(c, 2, std::integral_constant<int, 2>{});
    c = pair(c, 3, std::integral_constant<int, 3>{});
    codes[0] = b == 255 ? 0 : c;
  } else {
    const float top = scale * 448.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx_v2s16 c = {0, 0};
      if constexpr (T == Float::kF32) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_fmed3f(__builtin_bit_cast(float, v.w[4 * h + i]), -top, top);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, f[0], f[1], scale, false);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(c, f[2], f[3], scale, true);
      } else {
        // (A limit that f16 has to round, below 14 * 2^-24, rounds up to what its block's values do not exceed.)
        const uint16_t limit = mx_narrow<T>(top);
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = v.w[2 * h + i];
          const mx_v2u16 m = __builtin_elementwise_min(__builtin_bit_cast(mx_v2u16, x & 0x7FFF7FFFu), mx_v2u16{limit, limit});
          w[i] = __builtin_bit_cast(uint32_t, m) | (x & 0x80008000u);
        }
        if constexpr (T == Float::kF16) {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(mx_v2f16, w[0]), scale, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(c, __builtin_bit_cast(mx_v2f16, w[1]), scale, true);
        } else {
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(mx_v2bf16, w[0]), scale, false);
          c = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(c, __builtin_bit_cast(mx_v2bf16, w[1]), scale, true);
        }
      }
      codes[h] = b == 255 ? 0 : __builtin_bit_cast(uint32_t, c);
    }
  }
}

// The values of eight codes times 2^(b - 127), in f32 (b = 255 and the NaN codes of E4M3: NaN).
template <int BITS>
__device__ __forceinline__ void mx_values(const uint32_t codes[BITS / 4], uint32_t b, float f[8]) {
  const float scale = mx_scale_value(b);
  mx_v2f32 p[4];
  if constexpr (BITS == 4) {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 0);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 1);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 2);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[0], scale, 3);
  } else {
    p[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], scale, false);
    p[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[0], scale, true);
    p[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], scale, false);
    p[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(codes[1], scale, true);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = b == 255 ? __builtin_nanf("") : p[i / 2][i % 2];
}

}  // namespace uk

#endif  // IREE_AMD_CSRC_MX_DEVICE_H_
