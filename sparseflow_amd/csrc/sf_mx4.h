// The microscaled 4-bit format on the device: blocks of 32 values, a byte 127 + e
// (255: not a number) and 32 codes of 4 bits, +-{0, .5, 1, 1.5, 2, 3, 4, 6} 2^e.
// gfx950 only: its conversions take the block's scale along and round to nearest
// even, for every scale byte; a value of the format below 2^128 is a bf16 one exactly.
#pragma once

#include "sf_seq.h"

namespace sf {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMx4Block = 32;

// The scale as the conversions take it: they read the exponent's field alone, so that
// byte 0 is 2^-127 and byte 255 makes NaN.
__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// Eight values from eight codes.
__device__ __forceinline__ bf16x8 mx4_bf16(uint32_t codes, float scale) {
  const u32x4 u = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
  return __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ void mx4_f32(uint32_t codes, float scale, float (&v)[8]) {
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0);
  const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2);
  const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
}

// The scale's byte of a block whose largest magnitude has the bits `top`: its exponent's
// field less 2 (6 2^e is the largest value), at least 0; infinities and NaN have field 255.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) {
  const uint32_t f = top >> 23;
  return f == 255 ? 255 : f < 2 ? 0 : f - 2;
}

// Eight values of a block that four lanes in a row hold, eight each: their codes, and the
// block's scale byte in all four lanes.
__device__ __forceinline__ uint32_t mx4_encode(const float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __builtin_bit_cast(uint32_t, v[i]) & 0x7fffffffu;
    top = a > top ? a : top;  // (the bits of magnitudes are in the order of their values, NaN last)
  }
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const uint32_t o = __shfl_xor(top, d, kWave);
    top = o > top ? o : top;
  }
  byte = mx4_scale_byte(top);
  const float s = mx4_scale(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
  return byte == 255 ? 0 : c;
}

// Elements k .. k + 7 of a row of `size`; zeros behind its end.
template <typename T, bool ONCE = false>
__device__ __forceinline__ void load8(const T* __restrict__ row, int64_t k, int64_t size, float (&v)[8]) {
  if (k + 8 <= size) {
    load_any_f32<T, 8, ONCE>(row + k, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < size ? to_f32<T>(row[k + i]) : 0.f;
  }
}

// A float as a sum of bf16 parts of 8 bits each: exact in three (float32 from 2^-109 on; bf16 numbers
// are multiples of 2^-133) and two (f16).
// Cut off, not rounded: nothing overflows.  An infinity is the first part alone.
template <typename T>
struct Parts {
  static constexpr int n = sizeof(T) == 4 ? 3 : 2;
};
template <>
struct Parts<__hip_bfloat16> {
  static constexpr int n = 1;
};
__device__ __forceinline__ uint32_t pack_high(float lo, float hi) {  // the upper halves of two floats
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo), 0x07060302u);
}
template <int NP>
__device__ __forceinline__ void split8(const float (&v)[8], bf16x8 (&p)[NP]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = v[i];
#pragma unroll
  for (int k = 0; k < NP; ++k) {
    const u32x4 u = {pack_high(r[0], r[1]), pack_high(r[2], r[3]), pack_high(r[4], r[5]), pack_high(r[6], r[7])};
    p[k] = __builtin_bit_cast(bf16x8, u);
    if (k + 1 < NP) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, r[i]) & 0xffff0000u);
        r[i] = r[i] == h ? 0.f : r[i] - h;
      }
    }
  }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

}  // namespace
}  // namespace sf
