// What the attention kernels share (attention.hip, paged_attention.hip): operand types, the tiles of
// keys in LDS, and the running softmax's base-2 arithmetic.
#pragma once

#include <cfloat>

#include "fl_common.h"

namespace fl {
namespace {

constexpr int kKeys = 64;                  // per tile
// LDS rows: K padded by 16 bytes (the 16 lanes of a ds_read_b128 phase cover all banks), V
// by 64 (the four rows of a transposed 16-lane read lie 16 banks apart)
constexpr int kKRow = kDim + 8;
constexpr int kVRow = kDim + 32;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t attn_bf16_pair(float lo, float hi) {
  const f32x2_t f = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2_t));
}

// acc + both values of a packed bf16 pair (v_dot2_f32_bf16 with ones): the fp32 sum of the
// probabilities as the second product sees them, so that their roundings cancel in the quotient.
// The sum of the unrounded ones is 1-3% faster and errs more: against 64 bits 2.00e-3 instead of
// 1.99e-3 at 2048 dense queries, 2.03e-3 and 2.02e-3 at 8192 (the SDPA: 2.03e-3 and 2.08e-3).
__device__ __forceinline__ float add_pair(uint32_t w, float acc) {
  const bf16x2_t one = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), one, acc, false);
}

// the other half-wave's value of the same query
__device__ __forceinline__ float swap_half(float v) { return __shfl_xor(v, 32, kWave); }

struct AttnLds {
  uint16_t k[2][kKeys * kKRow];
  uint16_t v[2][kKeys * kVRow];
};

// Base-2 logits past kFar: their products with the scale are no longer exact to a small part of 1, so
// that exp2(fma(s, scale, -m)) would be off by a power of two, or overflow.  There the differences
// are taken before the scale.  kNone: the maximum of a query that has seen no key.
constexpr float kFar = 4096.0f;
constexpr float kNone = -FLT_MAX;
__device__ __forceinline__ float scaled_max(float r, float scale) { return fmaxf(r * scale, -FLT_MAX); }
// 2^(scale (a - b)) of two raw maxima, a <= b; sa, sb: their scaled_max
__device__ __forceinline__ float exp2_between(float a, float b, float sa, float sb, float scale) {
  return fast_exp2(fabsf(sa) > kFar || fabsf(sb) > kFar ? (a - b) * scale : sa - sb);
}

// 4 keys (rows of the tile) of one d per lane: lane i of each 16-lane group passes the
// address of V[key + i / 4][d + 4 (i % 4)] and receives V[key .. key + 3][d + i].
__device__ __forceinline__ bf16x4_t read_v_tr(const uint16_t* p) {
  typedef __attribute__((address_space(3))) bf16x4_t lds_t;
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
      reinterpret_cast<lds_t*>(reinterpret_cast<uintptr_t>(p)));
}

}  // namespace
}  // namespace fl
