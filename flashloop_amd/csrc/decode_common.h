// What the decode-step products share (decode_ops.hip, mx_gemv.hip): epilogues, bf16 helpers, buffer
// loads, and the residual / RMSNorm chain of their input rows.
#pragma once

#include "fl_common.h"

namespace fl {
namespace {

constexpr int kMaxM = 8;

enum GemvEpi : int { kEpiPlain = 0, kEpiF32 = 1, kEpiAdd = 2, kEpiSwiGlu = 3, kEpiRope = 4 };

__device__ __forceinline__ float bf16_round(float v) { return round_bf16(v); }

// A raw buffer resource over `bytes` bytes at p (wave-uniform): loads past the end (or
// from a resource of size 0) return zero.  Word 3 is the gfx9 raw-buffer format.
using BufRes = __amdgpu_buffer_rsrc_t;
__device__ __forceinline__ BufRes buf_res(const void* p, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, static_cast<int>(bytes), 0x00020000);
}
__device__ __forceinline__ uint4 buf_load16(BufRes r, uint32_t off) {
  return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(off), 0, 0));
}

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------
// Residual / RMSNorm chain of one row (one workgroup per row).  Thread t owns the
// 8-value chunks t, t + 256, ... of the row; every global load (x, r and the three
// weight rows) is issued before the first reduction, so the chain costs one memory
// round trip plus its block reductions.
// RMSNorm(x) = bf16(w * (x * rsqrt(mean(x^2) + eps))) in fp32, as the model's module.
constexpr int kNormThreads = 256;
constexpr int kNormChunks = 4;  // 8-value chunks per thread: D <= 8192

struct NormArgs {
  int D;
  float eps;
  const uint16_t* x;   // [M, D] or null (then h = r)
  const uint16_t* r;   // [M, D] residual / input
  const uint16_t* wa;  // norm of x
  const uint16_t* wf;  // optional norm of h (replaces h)
  const uint16_t* wb;  // optional norm of h -> z
  uint16_t* h_out;     // optional
  uint16_t* z_out;     // optional
  int64_t stride;      // row stride of every [M, D] tensor
};

constexpr int kNormWaves = kNormThreads / kWave;

// Block sums through two LDS buffers used in turn: reduction k writes buffer k & 1 and
// every wave reads it before it reaches the barrier of reduction k + 1, so buffer k & 1 is
// free again for reduction k + 2 -- one barrier per sum.  Waves past the first kNormWaves
// of a larger workgroup take part in the barriers only.
struct BlockSum {
  float (*red)[kNormWaves];
  int phase;
  __device__ __forceinline__ float operator()(float v) {
    float* r = red[phase & 1];
    ++phase;
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0 && threadIdx.x < kNormThreads) r[threadIdx.x >> 6] = v;
    lds_barrier();  // (a global fence would wait for a caller's weight loads)
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kNormWaves; ++i) s += r[i];
    return s;
  }
};

// v <- RMSNorm(v) with weight chunks w (8 values per chunk), rounded to bf16
template <int NC>
__device__ __forceinline__ void rms_apply(float (*v)[8], const uint4* w, int nc, int D, float eps, BlockSum& bs) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if (i < nc)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  const float inv = rsqrtf(bs(ss) / static_cast<float>(D) + eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float wf[8];
    unpack_bf16x8(w[i], wf);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = bf16_round(wf[e] * (v[i][e] * inv));
  }
}

__device__ __forceinline__ uint4 pack8(const float* f) {
  uint4 u;
  u.x = static_cast<uint32_t>(f32_to_bf16_rne(f[0])) | (static_cast<uint32_t>(f32_to_bf16_rne(f[1])) << 16);
  u.y = static_cast<uint32_t>(f32_to_bf16_rne(f[2])) | (static_cast<uint32_t>(f32_to_bf16_rne(f[3])) << 16);
  u.z = static_cast<uint32_t>(f32_to_bf16_rne(f[4])) | (static_cast<uint32_t>(f32_to_bf16_rne(f[5])) << 16);
  u.w = static_cast<uint32_t>(f32_to_bf16_rne(f[6])) | (static_cast<uint32_t>(f32_to_bf16_rne(f[7])) << 16);
  return u;
}

// The chain of row `base` (element offset): h = r (+ n_a(x)), optionally h = n_f(h),
// written to h_out when write_h; then z = n_b(h) when n_b is given.  chain_load issues the
// loads of this thread's chunks t, t + 256, ...; chain_finish leaves z (or h without n_b)
// in v as bf16 values.  All kNormThreads threads must call chain_finish (block reductions).
template <int NC>
struct ChainIn {
  uint4 xr[NC], rr[NC], wa[NC], wf[NC], wb[NC];
};

template <int NC>
__device__ __forceinline__ void chain_load(const NormArgs& a, int64_t base, ChainIn<NC>& in) {
  const int nq = a.D / 8;
  const int nc = (nq - static_cast<int>(threadIdx.x) + kNormThreads - 1) / kNormThreads;  // my chunks
  // Buffer loads sized to each operand (size 0 when absent): chunks past the row read as
  // zero without a branch.  A load under a branch would make the compiler's wait at the
  // join drain every outstanding load, including a caller's loads issued after these.
  (void)nc;
  const uint32_t row = static_cast<uint32_t>(a.D) * 2u;
  const BufRes r = buf_res(a.r + base, row);
  const BufRes x = buf_res(a.x ? a.x + base : nullptr, a.x ? row : 0u);
  const BufRes wa = buf_res(a.x ? a.wa : nullptr, a.x ? row : 0u);
  const BufRes wf = buf_res(a.wf, a.wf ? row : 0u);
  const BufRes wb = buf_res(a.wb, a.wb ? row : 0u);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const uint32_t off = 16u * static_cast<uint32_t>(threadIdx.x + i * kNormThreads);
    in.rr[i] = buf_load16(r, off);
    in.xr[i] = buf_load16(x, off);
    in.wa[i] = buf_load16(wa, off);
    in.wf[i] = buf_load16(wf, off);
    in.wb[i] = buf_load16(wb, off);
  }
}

template <int NC>
__device__ __forceinline__ void chain_finish(const NormArgs& a, int64_t base, bool write_h, const ChainIn<NC>& in,
                                             float (*h)[8], BlockSum& bs) {
  const int nc = (a.D / 8 - static_cast<int>(threadIdx.x) + kNormThreads - 1) / kNormThreads;
#pragma unroll
  for (int i = 0; i < NC; ++i) unpack_bf16x8(in.rr[i], h[i]);
  if (a.x != nullptr) {
    float xv[NC][8];
#pragma unroll
    for (int i = 0; i < NC; ++i) unpack_bf16x8(in.xr[i], xv[i]);
    rms_apply<NC>(xv, in.wa, nc, a.D, a.eps, bs);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = bf16_round(h[i][e] + xv[i][e]);
  }
  if (a.wf != nullptr) rms_apply<NC>(h, in.wf, nc, a.D, a.eps, bs);
  if (write_h && a.h_out != nullptr) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (i < nc) reinterpret_cast<uint4*>(a.h_out + base)[threadIdx.x + i * kNormThreads] = pack8(h[i]);
  }
  if (a.wb != nullptr) rms_apply<NC>(h, in.wb, nc, a.D, a.eps, bs);
}

template <int NC>
__device__ __forceinline__ void chain_row(const NormArgs& a, int64_t base, bool write_h, float (*h)[8], BlockSum& bs) {
  ChainIn<NC> in;
  chain_load<NC>(a, base, in);
  chain_finish<NC>(a, base, write_h, in, h, bs);
}

// One row's chain by one wave: lane l holds chunks l + 64 j, and the four partial sums of
// a norm are those of norm_chain_kernel's four waves (thread 64 w + l: chunks 64 w + l and
// 256 + 64 w + l), added in its order.
template <int CH>
struct WaveChainIn {
  uint4 x[CH], r[CH], wa[CH], wb[CH];
};

template <int CH>
__device__ __forceinline__ void wave_chain_load(const NormArgs& c, int64_t base, WaveChainIn<CH>& in) {
  const uint32_t row = static_cast<uint32_t>(c.D) * 2u;
  const BufRes r = buf_res(c.r + base, row);
  const BufRes x = buf_res(c.x ? c.x + base : nullptr, c.x ? row : 0u);
  const BufRes wa = buf_res(c.x ? c.wa : nullptr, c.x ? row : 0u);
  const BufRes wb = buf_res(c.wb, c.wb ? row : 0u);
  const uint32_t o = 16u * (threadIdx.x & 63u);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    in.x[j] = buf_load16(x, o + 1024u * j);
    in.r[j] = buf_load16(r, o + 1024u * j);
    in.wa[j] = buf_load16(wa, o + 1024u * j);
    in.wb[j] = buf_load16(wb, o + 1024u * j);
  }
}

template <int CH>
__device__ __forceinline__ void wave_rms(uint4 (&v)[CH], const uint4 (&w)[CH], int D, float eps) {
  float ss[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    float f[8];
    unpack_bf16x8(v[j], f);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss[j & 3] = fmaf(f[e], f[e], ss[j & 3]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) ss[i] = wave_sum(ss[i]);
  const float inv = rsqrtf((((ss[0] + ss[1]) + ss[2]) + ss[3]) / static_cast<float>(D) + eps);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    float f[8], g[8];
    unpack_bf16x8(v[j], f);
    unpack_bf16x8(w[j], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = g[e] * (f[e] * inv);
    v[j] = pack_bf16x8(f);
  }
}

// z (or h without n_b) of the row, as packed bf16, in in.r; h is written to h_out when asked
template <int CH>
__device__ __forceinline__ void wave_chain(const NormArgs& c, int64_t base, bool write_h, WaveChainIn<CH>& in) {
  if (c.x != nullptr) {
    wave_rms<CH>(in.x, in.wa, c.D, c.eps);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float f[8], g[8];
      unpack_bf16x8(in.r[j], f);
      unpack_bf16x8(in.x[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += g[e];
      in.r[j] = pack_bf16x8(f);
    }
  }
  if (c.wf != nullptr) {  // the last chain of a loop only: loaded here, so that the others keep the registers
    const BufRes res = buf_res(c.wf, static_cast<uint32_t>(c.D) * 2u);
#pragma unroll
    for (int j = 0; j < CH; ++j) in.x[j] = buf_load16(res, 16u * (threadIdx.x & 63u) + 1024u * j);
    wave_rms<CH>(in.r, in.x, c.D, c.eps);
  }
  if (write_h && c.h_out != nullptr) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      const int q = static_cast<int>(threadIdx.x & 63u) + 64 * j;
      if (q < c.D / 8) reinterpret_cast<uint4*>(c.h_out + base)[q] = in.r[j];
    }
  }
  if (c.wb != nullptr) wave_rms<CH>(in.r, in.wb, c.D, c.eps);
}

}  // namespace
}  // namespace fl
