// Rows in microscaled formats: quantisation of bf16 or f32 rows to 4 or 8 bits, the values back as
// bf16, and the residual / RMSNorm chain between two products with its last norm in 8 bits.
//
// Quantisation moves 2 or 4 bytes a value in and 1 or 1/2 out, with a maximum over 32 neighbours and a
// conversion that the hardware has, so it is bound by HBM.  A thread holds 8 neighbouring values (one
// 16-byte load of bf16), a block of 32 lies in a quad of lanes, whose maximum is two DPP moves.
#include "mx_common.h"

namespace fl {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kNormGrid = 256 * 5;  // workgroups of a norm: what the CUs hold at once

__device__ __forceinline__ uint32_t quad_max_u(uint32_t v) {
  v = max(v, static_cast<uint32_t>(dpp_i<kDppXor1>(static_cast<int>(v))));
  return max(v, static_cast<uint32_t>(dpp_i<kDppXor2>(static_cast<int>(v))));
}

struct QuantArgs {
  const void* x;
  int64_t x_stride;  // elements between rows
  int64_t pieces;    // rows * (padded K / 8)
  int k, per_row;    // pieces of a row
  uint8_t* codes;
  uint8_t* scales;
};

template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  return __builtin_bit_cast(uint4, reinterpret_cast<const Bytes16*>(p)->v);
}

// values [8 c, 8 c + 8) of a row, zero from k on
template <bool F32>
__device__ __forceinline__ void load8(const QuantArgs& a, int64_t row, int c, float* f) {
  const int64_t at = row * a.x_stride + 8 * static_cast<int64_t>(c);
  const int left = a.k - 8 * c;
  if (left >= 8) {
    if constexpr (F32) {
      const float* p = static_cast<const float*>(a.x) + at;
      const uint4 u = load16(p), v = load16(p + 4);
      const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(w[e]);
    } else {
      unpack_bf16x8(load16(static_cast<const uint16_t*>(a.x) + at), f);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = 0.0f;
    if (e < left)
      f[e] = F32 ? static_cast<const float*>(a.x)[at + e] : bf16_to_f32(static_cast<const uint16_t*>(a.x)[at + e]);
  }
}

// This thread's piece: its row and its place in it.  Rows are whole quads of pieces, so the lanes of a block
// are all inside or all past the end.
struct Piece {
  int64_t at, row;
  int c;
};
__device__ __forceinline__ Piece piece_of(int per_row) {
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads;
  const int64_t row0 = first / per_row;  // (uniform)
  const uint32_t in = static_cast<uint32_t>(first - row0 * per_row) + threadIdx.x;
  const uint32_t over = in / static_cast<uint32_t>(per_row);
  return Piece{first + threadIdx.x, row0 + over, static_cast<int>(in - over * static_cast<uint32_t>(per_row))};
}

// Eight values of a block, whose four lanes call this together, to their codes and the block's scale.
template <int BITS>
__device__ __forceinline__ void store_codes(const float* f, int64_t piece, uint8_t* codes, uint8_t* scales) {
  uint32_t peak = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) peak = max(peak, __float_as_uint(f[e]) & 0x7FFFFFFFu);
  peak = quad_max_u(peak);
  const uint32_t code = mx_scale_code<BITS>(peak);
  const float s = mx_scale(code);
  if constexpr (BITS == 4) {
    const uint32_t q = mx_encode4(f, s);
    reinterpret_cast<uint32_t*>(codes)[piece] = code == 255u ? 0u : q;
  } else {
    const uint2 q = mx_encode8(f, s);
    reinterpret_cast<uint2*>(codes)[piece] = code == 255u ? make_uint2(0u, 0u) : q;
  }
  if ((piece & 3) == 0) scales[piece >> 2] = static_cast<uint8_t>(code);
}

template <int BITS, bool F32>
__global__ __launch_bounds__(kThreads) void mx_quantize_kernel(QuantArgs a) {
  const Piece p = piece_of(a.per_row);
  if (p.at >= a.pieces) return;
  float f[8];
  load8<F32>(a, p.row, p.c, f);
  store_codes<BITS>(f, p.at, a.codes, a.scales);
}

// SwiGLU rows in 8 bits: bf16(bf16(silu(gate)) * up), as swiglu_kernel rounds, quantised without a trip
// through memory (8192 x 5632: 55 us where the two calls take 44 + 25).
struct SwigluMxArgs {
  QuantArgs gate;
  const uint16_t* up;
};

__global__ __launch_bounds__(kThreads) void mx_swiglu_kernel(SwigluMxArgs a) {
  const Piece p = piece_of(a.gate.per_row);
  if (p.at >= a.gate.pieces) return;
  QuantArgs up = a.gate;
  up.x = a.up;
  float g[8], u[8];
  load8<false>(a.gate, p.row, p.c, g);
  load8<false>(up, p.row, p.c, u);
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] = g[e] / (1.0f + expf(-g[e]));
  unpack_bf16x8(pack_bf16x8(g), g);
#pragma unroll
  for (int e = 0; e < 8; ++e) g[e] *= u[e];
  unpack_bf16x8(pack_bf16x8(g), g);
  store_codes<8>(g, p.at, a.gate.codes, a.gate.scales);
}

struct DequantArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  uint16_t* out;
  int64_t out_stride, pieces;
  int k, per_row;
};

template <int BITS>
__global__ __launch_bounds__(kThreads) void mx_dequantize_kernel(DequantArgs a) {
  const Piece p = piece_of(a.per_row);
  const int64_t piece = p.at;
  const int left = a.k - 8 * p.c;
  if (piece >= a.pieces || left <= 0) return;
  const float s = mx_scale(a.scales[piece >> 2]);
  uint4 v;
  if constexpr (BITS == 4)
    v = mx_decode4(reinterpret_cast<const uint32_t*>(a.codes)[piece], s);
  else
    v = mx_decode8(reinterpret_cast<const uint2*>(a.codes)[piece], s);
  uint16_t* out = a.out + p.row * a.out_stride + 8 * static_cast<int64_t>(p.c);
  if (left >= 8) {
    reinterpret_cast<Bytes16*>(out)->v = __builtin_bit_cast(u32x4_t, v);
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < left) out[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
}

// ---------------------------------------------------------------------------------
// h = r + norm_a(x), optionally h = norm_f(h), rounded to bf16; z = norm_b(h) in 8 bits, with
// norm_w(v) = w * v / sqrt(mean(v^2) + eps).
//
// A value of z that lies next to a border of e4m3 must not be moved over it by the rounding of what
// came before (a step of e4m3 is 1/16 of the value), so the sums and the products are in 64 bits: h
// becomes bf16 as torch converts a 64-bit value (by way of f32), and z, from that h, e4m3 in one
// rounding.  (A 64-bit FMA costs here what a 32-bit one does.)  The order of the sums shows in no output.
//
// ~260 instructions for 8 values and ~80 for each sum of a wave, which two pieces a lane halve (8192 rows of
// 4096: 53 -> 42 us, of 8192 with 8 waves a row 152 -> 117, of 1000 18 -> 15).  8192 x 2048 takes 26 us, 118 MB at
// 4.6 TB/s, where a large copy reaches 5.0 and the VALU is busy 59% of the time (norm_chain_kernel with bf16 z
// 31); 2051 x 1000 with the final norm 7.0, of which 2.8 are instructions, in waves that wait 45% of their time for
// r and x; a few rows 4-5 (one trip to memory and two sums).
struct NormMxArgs {
  int64_t rows, stride;
  int d, per_row;  // values; 8-value pieces of a padded row
  double eps;
  const uint16_t* x;
  const uint16_t* r;
  const uint16_t* wa;
  const uint16_t* wf;
  const uint16_t* wb;
  uint16_t* h_out;
  uint8_t* codes;
  uint8_t* scales;
};

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(dpp_i<CTRL>(static_cast<int>(u)));
  const uint32_t hi = static_cast<uint32_t>(dpp_i<CTRL>(static_cast<int>(u >> 32)));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double lane64(double v, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane));
  const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<kDppXor1>(v);
  v += dpp64<kDppXor2>(v);
  v += dpp64<kDppHalfMirror>(v);
  v += dpp64<kDppMirror>(v);
  return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}

// sum over the lanes of a row: W waves (two LDS buffers in turn, one barrier a sum)
template <int W>
struct RowSum64 {
  double (*red)[W < 4 ? 4 : W];
  int phase;
  __device__ __forceinline__ double operator()(double v) {
    v = wave_sum64(v);
    if constexpr (W == 1) return v;
    double* r = red[phase & 1];
    ++phase;
    const int wave = threadIdx.x >> 6, first = wave / W * W;
    if ((threadIdx.x & 63) == 0) r[wave] = v;
    lds_barrier();
    double s = r[first];
#pragma unroll
    for (int i = 1; i < W; ++i) s += r[first + i];
    return s;
  }
};

// Eight 64-bit values as f32 that round on to e4m3 as the 64-bit ones do.  The nearest f32 does unless it
// has reached a border (between two codes, or two scales: its last 19 bits are zero there), where the
// value rounded to odd takes its place.
typedef float f32x8_t __attribute__((ext_vector_type(8)));
__device__ __forceinline__ f32x8_t round8_for_codes(const double (&v)[8]) {
  f32x8_t f;
  uint32_t least = 0xFFFFFFFFu;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    f[e] = static_cast<float>(v[e]);
    least = min(least, __float_as_uint(f[e]) & 0x7FFFFu);
  }
  if (least == 0) f = f32x8_t{round_odd(v[0]), round_odd(v[1]), round_odd(v[2]), round_odd(v[3]),
                              round_odd(v[4]), round_odd(v[5]), round_odd(v[6]), round_odd(v[7])};
  return f;
}

// W waves share a row, a lane holds its pieces t, t + 64 W, ... (NC of them).  A workgroup takes one row, or as
// many as 4 waves hold, and goes on to further ones, whose r and x are requested before the sums of the
// ones in hand.
template <int W>
constexpr int kNormThreads = W < 4 ? 256 : 64 * W;

template <int NC, int W, bool ADD, bool FINAL>
__global__ __launch_bounds__(kNormThreads<W>) void norm_chain_mx_kernel(NormMxArgs a) {
  __shared__ double red[2][W < 4 ? 4 : W];
  constexpr int kLanes = 64 * W, kRows = kNormThreads<W> / kLanes;
  const int t = threadIdx.x % kLanes, nq = a.d / 8;
  RowSum64<W> sum{red, 0};
  uint4 r[NC], x[NC], wa[NC], wf[NC], wb[NC];
  const auto piece = [&](const uint16_t* p, int i) {
    const int c = t + i * kLanes;
    return p != nullptr && c < nq ? reinterpret_cast<const uint4*>(p)[c] : make_uint4(0, 0, 0, 0);
  };
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    if constexpr (ADD) wa[i] = piece(a.wa, i);
    if constexpr (FINAL) wf[i] = piece(a.wf, i);
    wb[i] = piece(a.wb, i);
  }
  const double inv_d = 1.0 / static_cast<double>(a.d);
  const auto inv_rms = [&](double ss) { return rsqrt(fma(sum(ss), inv_d, a.eps)); };
  const auto request = [&](int64_t row, uint4(&rr)[NC], uint4(&xx)[NC]) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      rr[i] = piece(a.r + row * a.stride, i);
      if constexpr (ADD) xx[i] = piece(a.x + row * a.stride, i);
    }
  };
  const auto squares = [&](const uint4(&v)[NC]) {
    double ss[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float f[8];
      unpack_bf16x8(v[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss[e & 1] = fma(static_cast<double>(f[e]), static_cast<double>(f[e]), ss[e & 1]);
    }
    return ss[0] + ss[1];
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes;
  request(min(row, a.rows - 1), r, x);
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * kRows; first < a.rows; first += step, row += step) {
    const bool live = row < a.rows;  // (a row past the last is the last again, not stored)
    uint4 nr[NC], nx[NC];
    if (first + step < a.rows) request(min(row + step, a.rows - 1), nr, nx);
    if constexpr (ADD || FINAL) {
      const double ia = ADD ? inv_rms(squares(x)) : 0.0;
      double h[NC][8];  // r + norm_a(x)
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float f[8], w[8];
        unpack_bf16x8(r[i], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = static_cast<double>(f[e]);
        if constexpr (ADD) {
          unpack_bf16x8(x[i], f);
          unpack_bf16x8(wa[i], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) h[i][e] = fma(static_cast<double>(w[e]) * static_cast<double>(f[e]), ia, h[i][e]);
        }
      }
      double fi = 1.0;
      if constexpr (FINAL) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = fma(h[i][e], h[i][e], ss);
        fi = inv_rms(ss);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float o[8], w[8];
        if constexpr (FINAL) unpack_bf16x8(wf[i], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(FINAL ? h[i][e] * (static_cast<double>(w[e]) * fi) : h[i][e]);
        r[i] = pack_bf16x8(o);
      }
    }
    if (a.h_out != nullptr && live) {
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if (t + i * kLanes < nq) reinterpret_cast<uint4*>(a.h_out + row * a.stride)[t + i * kLanes] = r[i];
    }
    if (a.wb != nullptr) {
      const double ib = inv_rms(squares(r));
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int c = t + i * kLanes;
        // (0 past the row, also where the row's statistics are not finite)
        const double scale = c < nq ? ib : 0.0;
        float fh[8], fw[8], z[8];
        double v[8];
        unpack_bf16x8(r[i], fh);
        unpack_bf16x8(wb[i], fw);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = static_cast<double>(fw[e]) * static_cast<double>(fh[e]) * scale;
        const f32x8_t rounded = round8_for_codes(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = rounded[e];
        if (c < a.per_row && live) store_codes<8>(z, row * a.per_row + c, a.codes, a.scales);  // (whole quads)
      }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      r[i] = nr[i];
      if constexpr (ADD) x[i] = nx[i];
    }
  }
}

template <int NC, int W>
void launch_norm(const NormMxArgs& a, hipStream_t st) {
  constexpr int kRows = kNormThreads<W> / (64 * W);
  const int64_t groups = (a.rows + kRows - 1) / kRows, most = kNormGrid * 256 / kNormThreads<W>;
  const dim3 g(static_cast<unsigned>(groups < most ? groups : most)), t(kNormThreads<W>);
  if (a.x != nullptr) {
    if (a.wf != nullptr)
      hipLaunchKernelGGL((norm_chain_mx_kernel<NC, W, true, true>), g, t, 0, st, a);
    else
      hipLaunchKernelGGL((norm_chain_mx_kernel<NC, W, true, false>), g, t, 0, st, a);
  } else if (a.wf != nullptr) {
    hipLaunchKernelGGL((norm_chain_mx_kernel<NC, W, false, true>), g, t, 0, st, a);
  } else {
    hipLaunchKernelGGL((norm_chain_mx_kernel<NC, W, false, false>), g, t, 0, st, a);
  }
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace fl

extern "C" int32_t fl_mx_quantize(const void* x, int32_t x_is_f32, int64_t x_stride, int64_t rows, int32_t k,
                                  int32_t bits, uint8_t* codes, uint8_t* scales, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(x && codes && scales, "fl_mx_quantize: null pointer");
  FL_REQUIRE(bits == 4 || bits == 8, "fl_mx_quantize: bits must be 4 or 8");
  FL_REQUIRE(rows >= 0 && k > 0 && k <= FL_MX_MAX_K && x_stride >= 0, "fl_mx_quantize: bad sizes");
  FL_REQUIRE(aligned(x, x_is_f32 ? 4 : 2), "fl_mx_quantize: x is not aligned to its elements");
  FL_REQUIRE(aligned(codes, 16), "fl_mx_quantize: codes must be 16-byte aligned");
  if (rows == 0) return FL_OK;
  QuantArgs a{};
  a.x = x;
  a.x_stride = x_stride;
  a.k = k;
  a.per_row = static_cast<int>(mx_padded(k) / 8);
  FL_REQUIRE(rows <= INT64_MAX / 2 / a.per_row, "fl_mx_quantize: too many rows");
  a.pieces = rows * a.per_row;
  a.codes = codes;
  a.scales = scales;
  const int64_t blocks = (a.pieces + kThreads - 1) / kThreads;
  FL_REQUIRE(blocks <= 0xFFFFFFFFll / kThreads, "fl_mx_quantize: grid too large");
  const dim3 g(static_cast<unsigned>(blocks)), t(kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (bits == 4) {
    if (x_is_f32)
      hipLaunchKernelGGL((mx_quantize_kernel<4, true>), g, t, 0, st, a);
    else
      hipLaunchKernelGGL((mx_quantize_kernel<4, false>), g, t, 0, st, a);
  } else {
    if (x_is_f32)
      hipLaunchKernelGGL((mx_quantize_kernel<8, true>), g, t, 0, st, a);
    else
      hipLaunchKernelGGL((mx_quantize_kernel<8, false>), g, t, 0, st, a);
  }
  FL_LAUNCH_CHECK("fl_mx_quantize");
  return FL_OK;
}

extern "C" int32_t fl_mx_swiglu(const uint16_t* gate, const uint16_t* up, int64_t row_stride, int64_t rows, int32_t k,
                                uint8_t* codes, uint8_t* scales, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(gate && up && codes && scales, "fl_mx_swiglu: null pointer");
  FL_REQUIRE(rows >= 0 && k > 0 && k <= FL_MX_MAX_K && row_stride >= k, "fl_mx_swiglu: bad sizes");
  FL_REQUIRE(aligned(gate, 2) && aligned(up, 2), "fl_mx_swiglu: gate or up is not aligned to its elements");
  FL_REQUIRE(aligned(codes, 16), "fl_mx_swiglu: codes must be 16-byte aligned");
  if (rows == 0) return FL_OK;
  SwigluMxArgs a{};
  a.gate.x = gate;
  a.gate.x_stride = row_stride;
  a.gate.k = k;
  a.gate.per_row = static_cast<int>(mx_padded(k) / 8);
  FL_REQUIRE(rows <= INT64_MAX / 2 / a.gate.per_row, "fl_mx_swiglu: too many rows");
  a.gate.pieces = rows * a.gate.per_row;
  a.gate.codes = codes;
  a.gate.scales = scales;
  a.up = up;
  const int64_t blocks = (a.gate.pieces + kThreads - 1) / kThreads;
  FL_REQUIRE(blocks <= 0xFFFFFFFFll / kThreads, "fl_mx_swiglu: grid too large");
  hipLaunchKernelGGL(mx_swiglu_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, static_cast<hipStream_t>(stream), a);
  FL_LAUNCH_CHECK("fl_mx_swiglu");
  return FL_OK;
}

extern "C" int32_t fl_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int32_t k, int32_t bits,
                                    uint16_t* out, int64_t out_stride, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(codes && scales && out, "fl_mx_dequantize: null pointer");
  FL_REQUIRE(bits == 4 || bits == 8, "fl_mx_dequantize: bits must be 4 or 8");
  FL_REQUIRE(rows >= 0 && k > 0 && k <= FL_MX_MAX_K && out_stride >= k, "fl_mx_dequantize: bad sizes");
  FL_REQUIRE(aligned(codes, 16), "fl_mx_dequantize: codes must be 16-byte aligned");
  FL_REQUIRE(aligned(out, 2), "fl_mx_dequantize: out is not aligned to its elements");
  if (rows == 0) return FL_OK;
  DequantArgs a{};
  a.codes = codes;
  a.scales = scales;
  a.out = out;
  a.out_stride = out_stride;
  a.k = k;
  a.per_row = static_cast<int>(mx_padded(k) / 8);
  FL_REQUIRE(rows <= INT64_MAX / 2 / a.per_row, "fl_mx_dequantize: too many rows");
  a.pieces = rows * a.per_row;
  const int64_t blocks = (a.pieces + kThreads - 1) / kThreads;
  FL_REQUIRE(blocks <= 0xFFFFFFFFll / kThreads, "fl_mx_dequantize: grid too large");
  const dim3 g(static_cast<unsigned>(blocks)), t(kThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (bits == 4)
    hipLaunchKernelGGL(mx_dequantize_kernel<4>, g, t, 0, st, a);
  else
    hipLaunchKernelGGL(mx_dequantize_kernel<8>, g, t, 0, st, a);
  FL_LAUNCH_CHECK("fl_mx_dequantize");
  return FL_OK;
}

extern "C" int32_t fl_norm_chain_mx(int32_t m, int32_t d, double eps, const uint16_t* x, const uint16_t* r,
                                    const uint16_t* w_a, const uint16_t* w_f, const uint16_t* w_b, uint16_t* h_out,
                                    uint8_t* z_codes, uint8_t* z_scales, int64_t stride, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(m >= 0 && d > 0 && d % 8 == 0 && d <= 8192 && stride >= d && stride % 8 == 0,
             "fl_norm_chain_mx: d must be a multiple of 8 up to 8192 and the row stride a multiple of 8");
  FL_REQUIRE(r != nullptr, "fl_norm_chain_mx: null residual/input");
  FL_REQUIRE(w_b == nullptr || (z_codes && z_scales), "fl_norm_chain_mx: z needs its outputs");
  FL_REQUIRE(w_b || h_out, "fl_norm_chain_mx: nothing to write");
  FL_REQUIRE(x == nullptr || w_a != nullptr, "fl_norm_chain_mx: x needs its norm weight");
  for (const void* p : {static_cast<const void*>(x), static_cast<const void*>(r), static_cast<const void*>(w_a),
                        static_cast<const void*>(w_f), static_cast<const void*>(w_b),
                        static_cast<const void*>(h_out), static_cast<const void*>(z_codes)})
    FL_REQUIRE(aligned(p, 16), "fl_norm_chain_mx: every tensor must be 16-byte aligned");
  if (m == 0) return FL_OK;
  const int per_row = static_cast<int>(mx_padded(d) / 8);
  const NormMxArgs a{m, stride, d, per_row, eps, x, r, w_a, w_f, w_b, h_out, z_codes, z_scales};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (per_row <= 64)
    launch_norm<1, 1>(a, st);
  else if (per_row <= 128)
    launch_norm<2, 1>(a, st);
  else if (per_row <= 256)
    launch_norm<2, 2>(a, st);
  else if (per_row <= 512)
    launch_norm<2, 4>(a, st);
  else
    launch_norm<2, 8>(a, st);
  FL_LAUNCH_CHECK("fl_norm_chain_mx");
  return FL_OK;
}
