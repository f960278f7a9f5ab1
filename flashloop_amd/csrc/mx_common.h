// Microscaled (MX) rows: values of 4 bits (e2m1) or 8 bits (e4m3) with one power-of-two scale for
// every 32 of them.  The scale of a block is the smallest 2^e with which no value of the block lies
// past the format's largest (6, 448), so nothing saturates; e >= -126, stored as e + 127; 255 marks
// a block that held a NaN or an infinity (its values read as NaN).  Rows are padded with zeros to
// whole steps of the matrix instruction, 128 values.
#pragma once

#include "fl_common.h"

namespace fl {

constexpr int kMxBlock = FL_MX_BLOCK;
constexpr int kMxPad = FL_MX_PAD;

__host__ __device__ __forceinline__ int64_t mx_padded(int64_t k) { return (k + kMxPad - 1) / kMxPad * kMxPad; }

typedef short mx_i16x2_t __attribute__((ext_vector_type(2)));

// 16 bytes at an element's alignment (one load or store, as global memory takes any alignment)
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Bytes16 {
  u32x4_t v;
};

// Stored scale of a block from the largest magnitude of its values, as f32 bits without the sign
// (compared as integers, so that a NaN counts as the largest).  1.m > 1.5 (6 = 1.5 * 2^2) or > 1.75
// (448 = 1.75 * 2^8) takes the next power.
template <int BITS>
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t peak) {
  const int e = static_cast<int>(peak >> 23);
  const uint32_t frac = peak & 0x7FFFFFu;
  const int code = BITS == 4 ? e - 2 + (frac > 0x400000u) : e - 8 + (frac > 0x600000u);
  return e == 255 ? 255u : static_cast<uint32_t>(max(code, 1));
}
// the scale as the float that the conversion instructions take (only its exponent counts: code 0,
// which nothing here writes, is 2^-127 to them, and 255 gives NaN)
__device__ __forceinline__ float mx_scale(uint32_t code) { return __uint_as_float(code << 23); }

// Eight values over their scale, rounded to the nearest code, ties to the even one: the hardware's
// conversions, equal to a search over the format's values on every bf16 value and at every border.
__device__ __forceinline__ uint32_t mx_encode4(const float* f, float scale) {
  uint32_t u = 0;
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, f[0], f[1], scale, 0);
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, f[2], f[3], scale, 1);
  u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, f[4], f[5], scale, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, f[6], f[7], scale, 3);
}
__device__ __forceinline__ uint2 mx_encode8(const float* f, float scale) {
  mx_i16x2_t a = {0, 0}, b = {0, 0};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, f[0], f[1], scale, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, f[2], f[3], scale, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, f[4], f[5], scale, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, f[6], f[7], scale, true);
  return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
}

// Eight 4-bit codes as packed bf16 values (exact: two bits of fraction and an exponent).
__device__ __forceinline__ uint4 mx_decode4(uint32_t u, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 0)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 1)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 2)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 3)));
}
__device__ __forceinline__ uint4 mx_decode8(uint2 u, float scale) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.x, scale, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, scale, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u.y, scale, true)));
}

// A 64-bit value as f32, rounded to odd: the last bit is set where anything was cut off.  A later
// rounding to fewer bits (bf16, e4m3), and any comparison with a value of fewer bits, then gives
// what it would give for the 64-bit value itself.  Past f32's range it is an infinity, as of a conversion.
__device__ __forceinline__ float round_odd(double v) {
  const float f = static_cast<float>(v);
  const double d = static_cast<double>(f);
  const uint32_t u = __float_as_uint(f);
  const uint32_t cut = (u - (fabs(d) > fabs(v) ? 1u : 0u)) | 1u;
  return __uint_as_float(d == v || __builtin_isinf(f) ? u : cut);
}

}  // namespace fl
