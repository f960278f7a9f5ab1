// y[m, n] = sum_k X[m, k] W[n, k] for rows X of 8 bits and weights W of 4 bits, both microscaled.
//
// bf16 results: v_mfma_scale_f32_16x16x128_f8f6f4 takes the codes as they are.  W is its first operand
// (lane l: row l % 16, block g = l / 16 of 32 codes), X its second (row l % 16, bytes 16 g .. +15 and
// 64 + 16 g .. +15 of the row's 128), and lane group g gives the scales of block g of both.  Results: a
// lane holds four neighbouring n of row m = l % 16.  Of every eight neighbouring products the instruction
// drops what lies under 2^-13 of the largest of them (groups of eight and steps add up in fp32): less than
// 7 * 2^-13 of the sum of the products' magnitudes.  Against the result that has no bound: where far
// products cancel, what they leave may be dropped whole.  Rows of normal values whose channels are
// e^N(0, s^2) apart, normal weights, K 128 to 8192, the part that is dropped in relative norm (and at most of
// the magnitudes): s = 0 2^-18 (2^-16), s = 1 2^-16 (2^-15), s = 2 and 3 2^-14 (2^-12), where the rounding
// to bf16 is 2^-9.2; 0.1, 0.6 and 2 in a hundred results lose more than 2^-9 of themselves.  The
// instruction is taken for its rate all the same, four times that of exact products: an f32 result has
// those, for a caller to round.
// f32 results: every value is exact in bf16 (but for rows' values under 2^-126, which become multiples of
// 2^-133, and 2^128, to which finite values next to f32's largest are rounded: an infinity), so the operands are widened in registers and v_mfma_f32_16x16x32_bf16 sums exact products in
// fp32 (a quarter of the rate).
//
// A workgroup's tile is BN rows of W by BM rows of X, K in steps of 128 through LDS.  The operands go from
// memory to LDS without passing registers, two steps ahead, in three buffers (one barrier a step);
// 16-byte pieces of a row are stored at a place that depends on the row, so that the lanes of a read
// meet all banks.  Scales come four steps at a time (a row's 16 bytes).  Rows past the matrix read
// as zeros.  The largest tile takes the LDS of a CU: its eight waves alternate between reading and
// multiplying, and it goes on to further tiles, whose first steps are on their way while it stores.
//
// What bounds it: with operands in registers the instruction reaches 3500-3750 TFLOP/s on random codes (4700
// on zeros, by its power).  8192^3 takes 355-396 us (2780-3100 TFLOP/s; in parts, on a build at 359: 306 without the transfers, 311 without the LDS
// reads, 273 without the products, and 278 with nothing but the products and barriers): the reading and
// the multiplying turns are about equally long.  8192 x 2048 -> 5632 80-90 us (2100-2380; 704 tiles in three
// rounds of 256, matrix cores busy 47-49% of the time), 8192 x 5632 -> 2048 67-75.  The bf16 library product
// of the three: 777-816, 174-185, 132-137 us.
#include <algorithm>

#include "lds_load.h"
#include "mx_common.h"

namespace fl {
namespace {

typedef int mx_i32x8_t __attribute__((ext_vector_type(8)));
typedef int mx_i32x4_t __attribute__((ext_vector_type(4)));
typedef float mx_f32x4_t __attribute__((ext_vector_type(4)));
typedef __bf16 mx_bf16x8_t __attribute__((ext_vector_type(8)));

struct MmArgs {
  const uint8_t* x;
  const uint8_t* xs;
  const uint8_t* w;
  const uint8_t* ws;
  void* y;
  int64_t m, y_stride;
  int n;
  int steps;  // of 128 k
  int tiles_n, tiles_m;
};

// A lane's 16 + 32 bytes of one step and their scales (low bytes) into the sums.
template <bool EXACT>
__device__ __forceinline__ mx_f32x4_t mx_step(const uint4& w, uint32_t ws, const uint4& x0, const uint4& x1, uint32_t xs,
                                              mx_f32x4_t c) {
  if constexpr (EXACT) {
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
    const uint2 p[4] = {make_uint2(x0.x, x0.y), make_uint2(x0.z, x0.w), make_uint2(x1.x, x1.y), make_uint2(x1.z, x1.w)};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mx_bf16x8_t, mx_decode4(q[j], mx_scale(ws & 255u))),
                                                  __builtin_bit_cast(mx_bf16x8_t, mx_decode8(p[j], mx_scale(xs & 255u))), c, 0, 0, 0);
    return c;
  } else {
    const mx_i32x8_t a = {static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w), 0, 0, 0, 0};
    const mx_i32x8_t b = {static_cast<int>(x0.x), static_cast<int>(x0.y), static_cast<int>(x0.z), static_cast<int>(x0.w),
                          static_cast<int>(x1.x), static_cast<int>(x1.y), static_cast<int>(x1.z), static_cast<int>(x1.w)};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 0, 0, static_cast<int>(ws), 0, static_cast<int>(xs));
  }
}
// 16-byte pieces of an X row's step that lane group g takes (the bf16 product wants block g's own 32)
template <bool EXACT>
__device__ __forceinline__ int x_piece(int g, int half) {
  return EXACT ? 2 * g + half : g + 4 * half;
}

// Outputs of row m from n on, 16 bytes a lane at an element's alignment (rows of any length: global memory
// takes it).  f32: four neighbours.
__device__ __forceinline__ void store4(const MmArgs& a, int64_t m, int n, const mx_f32x4_t& v) {
  if (m >= a.m || n >= a.n) return;
  float* y = static_cast<float*>(a.y) + m * a.y_stride + n;
  if (n + 4 <= a.n) {
    reinterpret_cast<Bytes16*>(y)->v = __builtin_bit_cast(u32x4_t, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) y[i] = v[i];
  }
}

// bf16, of two groups of 16 n side by side (v, u): the odd rows of 16 lanes change their v for the u of the even
// ones, so that a lane holds eight neighbours of one group and the four lanes of an m 32.
__device__ __forceinline__ void store8(const MmArgs& a, int64_t m, int n, int g, const mx_f32x4_t& v, const mx_f32x4_t& u) {
  const auto p = __builtin_amdgcn_permlane16_swap(bf16_pair(v[0], v[1]), bf16_pair(u[0], u[1]), false, false);
  const auto q = __builtin_amdgcn_permlane16_swap(bf16_pair(v[2], v[3]), bf16_pair(u[2], u[3]), false, false);
  const u32x4_t w = {p[0], q[0], p[1], q[1]};
  n += 16 * (g & 1) + 8 * (g >> 1);
  if (m >= a.m || n >= a.n) return;
  uint16_t* y = static_cast<uint16_t*>(a.y) + m * a.y_stride + n;
  if (n + 8 <= a.n) {
    reinterpret_cast<Bytes16*>(y)->v = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < a.n) y[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
  }
}

// ---------------------------------------------------------------------------------
// Byte g of each of four dwords (pick: g, 4 + g), the first lowest.
__device__ __forceinline__ uint32_t lane_scales(const uint4& q, uint32_t pick) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(q.w, q.z, pick), __builtin_amdgcn_perm(q.y, q.x, pick), 0x05040100u);
}

// A piece of a W row (four of 16 bytes) lies at its number xor this, one of an X row (eight) at its number xor
// (row / 2) % 8.  A 16-byte LDS read serves 16 lanes at a time, of rows 0-3 and 12-15 of one k group and 4-11
// of the next: their pieces then cover all 64 banks (with (row / 4) % 4 here, two of a bank).
__device__ __forceinline__ int w_turn(int row) { return (4 - (row >> 2)) & 3; }

template <int BN, int BM, int WN, int WM, int KS>
struct TileGeom {
  static constexpr int kWaves = WN * WM;  // of one of the KS groups that divide K
  static constexpr int kThreads = KS * kWaves * kWave;
  static constexpr int kFN = BN / WN / 16, kFM = BM / WM / 16;  // 16-row groups of a wave
  static constexpr int kWBytes = BN * 64, kXBytes = BM * 128;   // of a step
  static constexpr int kBuffer = kWBytes + kXBytes;
  static constexpr int kSRows = (BN + BM + 16 * kWaves - 1) / (16 * kWaves) * (16 * kWaves);
  static constexpr int kScales = kSRows * 16;                   // of four steps
  static constexpr int kGroup = 3 * kBuffer + 2 * kScales;      // LDS of a group
  static constexpr int kLds = KS * kGroup;
  // wave-wide transfers a wave makes
  static constexpr int kWLoads = kWBytes / 1024 / kWaves, kXLoads = kXBytes / 1024 / kWaves;
  static constexpr int kSLoads = kScales / 256 / kWaves;
  static_assert(kWLoads * 1024 * kWaves == kWBytes && kXLoads * 1024 * kWaves == kXBytes && BN % 16 == 0);
  static_assert(kLds <= 160 * 1024);
  // the groups' sums meet in the LDS of the steps
  static_assert(KS == 1 || (KS - 1) * kWaves * kFN * kFM * kWave * 16 <= kLds);
};

// XCD-aware order: workgroups go to the 8 XCDs in turn, so XCD d takes the d-th stretch of the tiles; a
// stretch walks groups of 8 tile rows of X.  One tile of 256 x 256 for each of an XCD's 32 CUs then takes 8
// panels of X and 4 of W: they stay in its 4 MB L2 up to K of about 1500, and past that X is read again for
// every such round (8192 x 2048 -> 5632: 4.3 + 1.1 MB, three rounds, 129 MB read for operands of 23).
__device__ __forceinline__ void tile_of(const MmArgs& a, int id, int* tn, int64_t* tm) {
  const int total = a.tiles_n * a.tiles_m;
  const int d = id & 7, per = total >> 3, more = total & 7;
  const int t = d * per + min(d, more) + (id >> 3);
  const int group = 8 * a.tiles_n, g = t / group, in = t - g * group;
  const int rows = min(8, a.tiles_m - 8 * g);
  *tn = in / rows;
  *tm = 8 * g + in - *tn * rows;
}

template <int BN, int BM, int WN, int WM, int KS, bool F32, bool TURNS>
__global__ __launch_bounds__(KS* WN* WM* kWave) void mx_matmul_tile_kernel(MmArgs a) {
  using G = TileGeom<BN, BM, WN, WM, KS>;
  static_assert(KS == 1 || !TURNS);
  __shared__ __attribute__((aligned(1024))) uint8_t lds_all[G::kLds];
  const int lane = threadIdx.x & 63;
  const int all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = KS == 1 ? all_waves : all_waves % G::kWaves, part = KS == 1 ? 0 : all_waves / G::kWaves;
  uint8_t* const lds = lds_all + part * G::kGroup;
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)lds_all)) + part * G::kGroup;
  const int i = lane & 15, g = lane >> 4;
  const int wn = wave % WN, wm = wave / WN;
  const int64_t blocks = static_cast<int64_t>(a.steps) * 4;  // of a row
  // this workgroup's tiles: blockIdx.x, + gridDim.x, ... (TURNS; else the one); their steps are counted through
  const int tiles =
      TURNS ? (a.tiles_n * a.tiles_m - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) : 1;
  // this group's steps: all, or the part-th stretch of them
  const int per = (a.steps + KS - 1) / KS, first_step = KS == 1 ? 0 : part * per;
  const int total = KS == 1 ? tiles * a.steps : max(0, min(per, a.steps - first_step));
  // what this lane moves: piece p of the tile's step lies at LDS 16 p
  uint32_t wv[G::kWLoads], xv[G::kXLoads], sv[G::kSLoads];
#pragma unroll
  for (int j = 0; j < G::kWLoads; ++j) {
    const int p = (wave * G::kWLoads + j) * 64 + lane, row = p / 4, c = (p & 3) ^ w_turn(row);
    wv[j] = static_cast<uint32_t>(row) * static_cast<uint32_t>(blocks) * 16u + 16u * c;
  }
#pragma unroll
  for (int j = 0; j < G::kXLoads; ++j) {
    const int p = (wave * G::kXLoads + j) * 64 + lane, row = p / 8, c = (p & 7) ^ ((row >> 1) & 7);
    xv[j] = static_cast<uint32_t>(row) * static_cast<uint32_t>(blocks) * 32u + 16u * c;
  }
#pragma unroll
  for (int j = 0; j < G::kSLoads; ++j) {
    const int p = (wave * G::kSLoads + j) * 64 + lane, row = p / 4;
    sv[j] = static_cast<uint32_t>(row < BN ? row : row - BN) * static_cast<uint32_t>(blocks) + 4u * (p & 3);
    if (row >= BN + BM) sv[j] = 0x80000000u;  // (past every buffer)
  }
  // the next step to request: tile, step in it, buffer, buffer of its scales
  mx_i32x4_t wr{}, xr{}, wsr{}, xsr{};
  int rtile = blockIdx.x, rs = 0, rbuf = 0, rscale = 1;
  const auto request = [&]() __attribute__((always_inline)) {
    if (rs == 0) {
      int tn;
      int64_t tm;
      tile_of(a, rtile, &tn, &tm);
      const int64_t n0 = static_cast<int64_t>(tn) * BN, m0 = tm * BM;
      wr = raw_buffer(a.w + n0 * blocks * 16, (a.n - n0) * blocks * 16);
      xr = raw_buffer(a.x + m0 * blocks * 32, (a.m - m0) * blocks * 32);
      wsr = raw_buffer(a.ws + n0 * blocks, (a.n - n0) * blocks);
      xsr = raw_buffer(a.xs + m0 * blocks, (a.m - m0) * blocks);
    }
    if ((rs & 3) == 0) {
      rscale ^= 1;
      const uint32_t at = lds0 + 3 * G::kBuffer + rscale * G::kScales;
      const uint32_t off = 4u * (first_step + rs);  // (in the lane's offset: past the last row's end it is past the buffer's)
#pragma unroll
      for (int j = 0; j < G::kSLoads; ++j) {
        const int first = (wave * G::kSLoads + j) * 16;  // (16 rows a transfer: all of W or all of X)
        if (first < BN)
          to_lds<4>(wsr, sv[j] + off, 0, at + 256u * (wave * G::kSLoads + j));
        else
          to_lds<4>(xsr, sv[j] + off, 0, at + 256u * (wave * G::kSLoads + j));
      }
    }
    const uint32_t at = lds0 + rbuf * G::kBuffer;
#pragma unroll
    for (int j = 0; j < G::kWLoads; ++j) to_lds<16>(wr, wv[j], 64u * (first_step + rs), at + 1024u * (wave * G::kWLoads + j));
#pragma unroll
    for (int j = 0; j < G::kXLoads; ++j)
      to_lds<16>(xr, xv[j], 128u * (first_step + rs), at + G::kWBytes + 1024u * (wave * G::kXLoads + j));
    rbuf = rbuf == 2 ? 0 : rbuf + 1;
    if (++rs == a.steps) {
      rs = 0;
      rtile += gridDim.x;
    }
  };

  mx_f32x4_t acc[G::kFN][G::kFM];
  const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < G::kFN; ++n)
#pragma unroll
      for (int m = 0; m < G::kFM; ++m) acc[n][m] = mx_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  };
  const int wrow = wn * (BN / WN) + i, xrow = wm * (BM / WM) + i;
  const uint8_t* wl = lds + wrow * 64 + 16 * (g ^ w_turn(i));
  const uint8_t* xl0 = lds + G::kWBytes + xrow * 128 + 16 * (x_piece<F32>(g, 0) ^ ((i >> 1) & 7));
  const uint8_t* xl1 = lds + G::kWBytes + xrow * 128 + 16 * (x_piece<F32>(g, 1) ^ ((i >> 1) & 7));
  const uint32_t pick = static_cast<uint32_t>(g) | static_cast<uint32_t>(4 + g) << 8;

  uint4 w[G::kFN], x0[G::kFM], x1[G::kFM];
  uint32_t ws[G::kFN], xs[G::kFM];
  // the step in hand: tile, step in it, buffer, buffer of its scales
  int ctile = blockIdx.x, cs = 0, cbuf = 0, cscale = 1;
  const auto read_step = [&]() __attribute__((always_inline)) {
    const uint32_t at = cbuf * G::kBuffer;
    cbuf = cbuf == 2 ? 0 : cbuf + 1;
#pragma unroll
    for (int n = 0; n < G::kFN; ++n) w[n] = *reinterpret_cast<const uint4*>(wl + at + n * 1024);
#pragma unroll
    for (int m = 0; m < G::kFM; ++m) {
      x0[m] = *reinterpret_cast<const uint4*>(xl0 + at + m * 2048);
      x1[m] = *reinterpret_cast<const uint4*>(xl1 + at + m * 2048);
    }
    // scales: this lane's bytes of four steps at once, the step's own in the low byte
    if ((cs & 3) == 0) {
      cscale ^= 1;
      const uint8_t* sl = lds + 3 * G::kBuffer + cscale * G::kScales;
#pragma unroll
      for (int n = 0; n < G::kFN; ++n) ws[n] = lane_scales(*reinterpret_cast<const uint4*>(sl + (wrow + 16 * n) * 16), pick);
#pragma unroll
      for (int m = 0; m < G::kFM; ++m) xs[m] = lane_scales(*reinterpret_cast<const uint4*>(sl + (BN + xrow + 16 * m) * 16), pick);
    } else {
#pragma unroll
      for (int n = 0; n < G::kFN; ++n) ws[n] >>= 8;
#pragma unroll
      for (int m = 0; m < G::kFM; ++m) xs[m] >>= 8;
    }
  };
  const auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < G::kFM; ++m)
#pragma unroll
      for (int n = 0; n < G::kFN; ++n) acc[n][m] = mx_step<F32>(w[n], ws[n], x0[m], x1[m], xs[m], acc[n][m]);
  };
  constexpr int kStep = G::kWLoads + G::kXLoads;  // transfers of a step, its scales aside (they are made first)
  // this wave's transfers of step s have landed (those of step s + 1, if made, may be under way)
  const auto landed = [&](int s) __attribute__((always_inline)) {
    if (s + 1 < total)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kStep) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  const auto barrier = [&]() __attribute__((always_inline)) {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
  };

  // after a tile's last step: its results, while the next tile's first steps are on their way
  const auto finish = [&]() __attribute__((always_inline)) {
    int tn;
    int64_t tm;
    tile_of(a, ctile, &tn, &tm);
    ctile += gridDim.x;
#pragma unroll
    for (int m = 0; m < G::kFM; ++m)
#pragma unroll
      for (int n = 0; n < G::kFN; n += 2) {
        const int64_t row = tm * BM + xrow + 16 * m;
        const int col = tn * BN + wn * (BN / WN) + 16 * n;
        if constexpr (F32) {
          store4(a, row, col + 4 * g, acc[n][m]);
          store4(a, row, col + 16 + 4 * g, acc[n + 1][m]);
        } else {
          store8(a, row, col, g, acc[n][m], acc[n + 1][m]);
        }
      }
  };

  clear();
  if (KS == 1 || total > 0) request();
  if (total > 1) request();
  if constexpr (TURNS) {
    // The waves of a SIMD take turns: four waves read a step from LDS while the other four multiply the one
    // that they hold, a barrier between the turns.  Waves 0..3 read step s in turn 2 s, waves 4..7 in turn
    // 2 s + 1.  Step s + 1 has landed for every wave before the barrier that ends turn 2 s + 1, and the
    // buffer that step s + 2 fills was last read in turn 2 s - 1, before a barrier that follows that read.
    const bool second = wave >= G::kWaves / 2;
    landed(0);
    barrier();
    if (second) barrier();
    for (int s = 0; s < total; ++s) {
      if (s + 2 < total) request();
      read_step();
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (second && s + 1 < total) landed(s + 1);
      barrier();
      multiply();
      if (!second && s + 1 < total) landed(s + 1);
      if (++cs == a.steps) {
        cs = 0;
        finish();
        clear();
      }
      barrier();
    }
    if (!second) barrier();
  } else {
    for (int s = 0; s < (KS == 1 ? total : per); ++s) {
      // step s has landed for every wave, and no wave reads step s - 1 any more, whose buffer the next
      // request fills
      landed(s);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      barrier();
      if (s + 2 < total) request();
      if (KS == 1 || s < total) {
        read_step();
        multiply();
      }
      ++cs;
    }
    if constexpr (KS > 1) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      barrier();
      mx_f32x4_t* sums = reinterpret_cast<mx_f32x4_t*>(lds_all);
      const auto at = [&](int p, int n, int m) { return (((p - 1) * G::kWaves + wave) * G::kFN * G::kFM + n * G::kFM + m) * kWave + lane; };
      if (part > 0) {
#pragma unroll
        for (int n = 0; n < G::kFN; ++n)
#pragma unroll
          for (int m = 0; m < G::kFM; ++m) sums[at(part, n, m)] = acc[n][m];
      }
      __syncthreads();
      if (part > 0) return;
#pragma unroll
      for (int p = 1; p < KS; ++p)
#pragma unroll
        for (int n = 0; n < G::kFN; ++n)
#pragma unroll
          for (int m = 0; m < G::kFM; ++m) acc[n][m] += sums[at(p, n, m)];
    }
    finish();
  }
}

template <int BN, int BM, int WN, int WM, int KS, bool F32, bool TURNS>
void launch_tiles(MmArgs a, hipStream_t st) {
  a.tiles_n = (a.n + BN - 1) / BN;
  a.tiles_m = static_cast<int>((a.m + BM - 1) / BM);
  // A workgroup takes further tiles where all CUs are in use (one workgroup each), but for tiles of a single
  // step: a buffer of scales is filled again for the stretch after the next, whose first step is requested two
  // steps ahead, so the stretch that it held has to start three steps before that one (the later waves read
  // a step a turn after the earlier ones).  Stretches of 1, 1, ... steps break that; 4, 1, 4, 1 do not.  us with
  // one tile a workgroup and with further ones, 8192 x 5632 by k 640: 45, 38; 1152: 57, 49; 2176: 85, 78.
  const int tiles = a.tiles_n * a.tiles_m, grid = TURNS && a.steps > 1 ? std::min(tiles, 256) : tiles;
  hipLaunchKernelGGL((mx_matmul_tile_kernel<BN, BM, WN, WM, KS, F32, TURNS>), dim3(grid), dim3(KS * WN * WM * kWave), 0, st, a);
}

// The larger the tile, the less LDS traffic a product needs; the more workgroups, the more CUs work, and where
// a CU has few of them KS groups of waves divide K, so that its steps do not follow one another.  Measured, us,
// bf16 results, m x n x k (tile of n by m, groups):
//   8192 x 5632 x 2048: 256 x 256 80.5, 128 x 128 129; 8192^3: 367, 656
//   820 x 5632 x 2048: 128 x 128 18.6, 64 x 64 18.9
//   up to 64 rows, of which larger tiles would be half empty (64 x 64, 128 x 128, two groups of 64 x 64): 40 x 49152
//   x 2048 12.0, 17.1, 14.1; 64 13.3, 17.8, 15.0; 100 19.5, 19.2, 23.7; f32 results of 64 20.1, 32.0, 21.4, of 100
//   32.5, 33.3, 39.1; 64 x 131072 42.6, 41.9 (256 x 256: 50.6)
//   820 x 2048 x 2048: 64 x 64 in two groups 9.7, one 9.8; 512 x 2048 x 2048: 7.4, 8.5; 32 x 32 in four 10.2
//   128 x 2048 x 2048: 32 x 32 in four groups 5.0, 64 x 64 in one, two, four 8.1, 7.0, 7.1
//   256 x 2048 x 2048: 6.4, 64 x 64 in two 7.1; 128 x 5632 x 2048: 8.7, 7.2
//   32 x 49152 x 2048: 64 x 32 11.2, 64 x 64 12.6, 32 x 32 in four groups 15.2
//   around 256 tiles of 256 x 256 (these, then 128 x 128), k 2048: 96 of them 27.5, 19.0; 176 28.1, 29.0; 192 28.3,
//   29.2; 240 29.6, 34.0; 256 30.1, 34.7; 288 48.2, 43.1; 352 49.3, 48.6.  k 5632: 128 56.7, 45.0; 192 58.8,
//   69.1; 256 64.8, 86.2
// f32 results by m, n 49152, k 2048 (bf16 ones of the same rows): 16 14.8 (10.2), 64 20.1 (13.3), 512 94.6 (50.1),
// 2048 372 (165), 8192 1460 (644; 1130 TFLOP/s of the 1400 that a bf16 library product reaches).
template <bool F32>
void launch_matmul(const MmArgs& a, hipStream_t st) {
  const auto tiles = [&](int64_t bn, int64_t bm) { return ((a.n + bn - 1) / bn) * ((a.m + bm - 1) / bm); };
  if (tiles(32, 32) <= 512) return launch_tiles<32, 32, 1, 2, 4, F32, false>(a, st);
  if (a.m <= 32) return launch_tiles<64, 32, 2, 2, 1, F32, false>(a, st);
  if (tiles(64, 64) <= 512) return launch_tiles<64, 64, 2, 2, 2, F32, false>(a, st);
  if (a.m <= 64) return launch_tiles<64, 64, 2, 2, 1, F32, false>(a, st);
  if constexpr (!F32)
    if (tiles(256, 256) >= 256) return launch_tiles<256, 256, 2, 4, 1, F32, true>(a, st);
  if (tiles(128, 128) >= 256) return launch_tiles<128, 128, 2, 2, 1, F32, false>(a, st);
  launch_tiles<64, 64, 2, 2, 1, F32, false>(a, st);
}

}  // namespace
}  // namespace fl

extern "C" int32_t fl_mx_matmul(const uint8_t* x_codes, const uint8_t* x_scales, int64_t m, int32_t k,
                                const uint8_t* w_codes, const uint8_t* w_scales, int32_t n, void* y, int32_t y_is_f32,
                                int64_t y_stride, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(x_codes && x_scales && w_codes && w_scales && y, "fl_mx_matmul: null pointer");
  FL_REQUIRE(m >= 0 && k > 0 && k <= FL_MX_MAX_K && n > 0 && y_stride >= n, "fl_mx_matmul: bad sizes");
  FL_REQUIRE(reinterpret_cast<uintptr_t>(x_codes) % 16 == 0 && reinterpret_cast<uintptr_t>(w_codes) % 16 == 0,
             "fl_mx_matmul: codes must be 16-byte aligned");
  FL_REQUIRE(reinterpret_cast<uintptr_t>(x_scales) % 4 == 0 && reinterpret_cast<uintptr_t>(w_scales) % 4 == 0,
             "fl_mx_matmul: scales must be 4-byte aligned");
  FL_REQUIRE(reinterpret_cast<uintptr_t>(y) % (y_is_f32 ? 4 : 2) == 0, "fl_mx_matmul: y is not aligned to its elements");
  // (a grid counts tiles of 64 x 64 in 32 bits, of at most 2^32 threads)
  FL_REQUIRE(m <= 0x7FFFFFFF && ((m + 63) / 64) * ((static_cast<int64_t>(n) + 63) / 64) <= 0xFFFFFF && n <= 0x7FFFFFF,
             "fl_mx_matmul: too many outputs");
  if (m == 0) return FL_OK;
  const MmArgs a{x_codes, x_scales, w_codes, w_scales, y, m, y_stride, n, static_cast<int>(mx_padded(k) / kMxPad), 0, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (y_is_f32)
    launch_matmul<true>(a, st);
  else
    launch_matmul<false>(a, st);
  FL_LAUNCH_CHECK("fl_mx_matmul");
  return FL_OK;
}
