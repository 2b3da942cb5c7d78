// latent_device.h -- what the operators around the paged latent cache share:
// element types, 8-element loads and stores, rotation angles, the quantised
// group's scale, and the cache's addressing.
#pragma once

#include <type_traits>

#include "fdm_internal.h"

namespace fdm {

constexpr int kLatDim = 512;   // latent values of a row (keys and values)
constexpr int kRotDim = 64;    // rotary values of a row (keys only)
constexpr int kLatGroup = 128; // latent values that share a scale in an FP8 row

// Eight consecutive elements <-> fp32.  `vec` (16-byte aligned, uniform over
// the launch): one or two 16-byte accesses; else one access an element.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float* v) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const f32x4 a = reinterpret_cast<const f32x4*>(p)[0], b = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
    } else {
      typedef T tx8 __attribute__((ext_vector_type(8)));
      const tx8 a = *reinterpret_cast<const tx8*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)p[i];
  }
}

// fp32 -> the element type, to nearest even.
template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, const float* v) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<f32x4*>(p)[0] = f32x4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<f32x4*>(p)[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      typedef T tx8 __attribute__((ext_vector_type(8)));
      tx8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
      *reinterpret_cast<tx8*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (T)v[i];
  }
}

// Sine and cosine of a fraction of a turn in 64-bit fixed point.  A rotary
// angle is position x (frequency / 2 pi): with the frequency held as that
// fraction, the wrapping 64-bit product is already reduced to one turn, exact
// for every 32-bit position, where a float angle has lost 2e-3 radians at
// position 32768.  The nearest quarter turn is taken off (|x| <= pi / 4) and
// the Taylor series cut where the next term is below 2^-24: x^11 / 11! <
// 2e-9 for the sine, x^10 / 10! < 2.5e-8 for the cosine.
__device__ __forceinline__ void turn_sincos(uint64_t turns, float* sin_out, float* cos_out) {
  const uint32_t q = (uint32_t)((turns + (1ull << 61)) >> 62);
  const int32_t r = (int32_t)((int64_t)(turns - ((uint64_t)q << 62)) >> 30);  // 2^-34 of a turn
  const float x = (float)r * (6.283185307179586f / 17179869184.0f);
  const float z = x * x;
  const float s = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320))));
  const float a = q & 1 ? c : s, b = q & 1 ? s : c;
  *sin_out = q & 2 ? -a : a;
  *cos_out = ((q + 1) & 2) ? -b : b;
}

// The scale byte of an FP8 group: e + 127 with e the smallest exponent for
// which amax <= 448 * 2^e (448 = 1.75 * 2^8, the largest e4m3 value), inside
// [-100, 119]: below, the codes' steps would leave the normal range of the
// 16-bit types; above, 448 * 2^e is no fp32 number.  255 (no number) for a
// group that holds an infinity or a NaN: amax is not finite then.
constexpr int kScaleMin = -100, kScaleMax = 119, kScaleNan = 255;
__device__ __forceinline__ int fp8_scale_byte(float amax) {
  const uint32_t b = __builtin_bit_cast(uint32_t, amax) & 0x7FFFFFFFu;
  if (b >= 0x7F800000u) return kScaleNan;
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kScaleMin), kScaleMax) + 127;
}
// 2^(byte - 127); NaN for 255
__device__ __forceinline__ float scale_value(int byte) {
  return __builtin_bit_cast(float, byte == kScaleNan ? 0x7FC00000u : (uint32_t)max(byte, 1) << 23);
}

// e4m3 codes of eight values of a group with that scale byte, four a word.
__device__ __forceinline__ void fp8_codes8(const float* v, int byte, uint32_t* code) {
  const float up = scale_value(byte == kScaleNan ? 127 : 254 - byte);  // 2^-e
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = fminf(fmaxf(v[4 * k + j] * up, -448.0f), 448.0f);
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    code[k] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  }
  if (byte == kScaleNan) code[0] = code[1] = 0x7F7F7F7Fu;  // e4m3's NaN
}

// max over |v| that keeps infinities and NaN (a NaN's bits, sign cleared, are
// above every number's)
__device__ __forceinline__ float amax_bits(float m, float v) {
  const uint32_t a = __builtin_bit_cast(uint32_t, m), b = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
  return __builtin_bit_cast(float, max(a, b));
}

}  // namespace fdm
