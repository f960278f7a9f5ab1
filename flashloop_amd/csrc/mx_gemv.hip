// Decode-step products with 4-bit microscaled weights: y[m, n] = sum_k x[m, k] W[n, k] for 1..8 rows
// of x in bf16 -- fl_gemv_bf16 with a quarter of its weight bytes, the same epilogues, and the norm
// chain of the input rows in the prologue where there is one.
//
// Bytes: N K (1/2 + 1/32) for the weights, next to which x and y are nothing.  A weight is exact in
// bf16 (two bits of fraction and an exponent), so the codes become bf16 in registers, two an
// instruction with their scale, and v_mfma_f32_16x16x32_bf16 takes them against unrounded bf16 rows.
//
// As in gemv_mfma_kernel a tile is T rows of W (8, or 4 for one row of x) and the instruction's other
// rows and columns hold further k of the same rows; the diagonal T x T blocks of the product add up to
// the tile.  A lane's 16-byte load is one block of 32 values, four products' worth, so the lanes of a
// W row read 128 (T = 8) or 256 bytes in a row, and a workgroup's step is 2048 k.
#include "decode_common.h"
#include "mx_common.h"

namespace fl {
namespace {

struct MxGemvArgs {
  const void* x;  // [M, K] bf16, or f32 (rounded to bf16 on load)
  int64_t x_stride;
  int x_f32;
  int M, K, N;
  uint32_t blocks;  // stored blocks of a row
  const uint8_t* codes[3];  // plain / add / f32: [0]; SwiGLU: gate, up; RoPE: q, k, v
  const uint8_t* scales[3];
  void* y[3];
  int64_t y_stride;
  const uint16_t* addend;
  int64_t addend_stride;
  const uint16_t* cos;  // [M, head_dim]
  const uint16_t* sin;
  int head_dim;
};

template <int MT>
struct MxGeom {
  static constexpr int kWaves = MT == 1 ? 4 : 8;
  static constexpr int kThreads = kWaves * kWave;
  static constexpr int kTile = MT == 1 ? 4 : 8;    // rows of W (and of x) per tile
  static constexpr int kSlices = 16 / kTile;       // groups of 4 blocks side by side in one product
  static constexpr int kParts = kWaves * kSlices;  // partial tiles
};
constexpr int kMxStep = 2048;      // k of one step of a workgroup
constexpr int kMxChainMaxK = 4096;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer

template <int EPI>
constexpr bool kPairs = EPI == kEpiSwiGlu || EPI == kEpiRope;

// Groups of T rows (pair epilogues: of T pairs) that a unit's NT tiles hold.
template <int EPI, int NT>
constexpr int kGroups = kPairs<EPI> ? NT / 2 : NT;

template <int EPI, int MT, int NT>
__host__ __device__ __forceinline__ int mx_units(int n) {
  constexpr int rows = kGroups<EPI, NT> * MxGeom<MT>::kTile;
  return ((EPI == kEpiRope ? n / 2 : n) + rows - 1) / rows;
}

// Where the rows of a unit's tiles lie: a buffer of codes and one of scales from the unit's first row
// on, and this lane's row in them.  Rows past the matrix repeat its last (not stored).
template <int NT>
struct MxRows {
  BufRes codes[NT], scales[NT];
  uint32_t row[NT];
};

template <int EPI, int MT, int NT>
__device__ __forceinline__ void mx_unit_rows(const MxGemvArgs& a, int u, MxRows<NT>& r) {
  constexpr int kTile = MxGeom<MT>::kTile;
  const int i = threadIdx.x & (kTile - 1);
  const auto buffer = [&](int t, int mat, int first) {
    const int64_t left = a.N - first, bytes = left * a.blocks * 16;
    const uint8_t* c = mat == 0 ? a.codes[0] : (mat == 1 ? a.codes[1] : a.codes[2]);
    const uint8_t* s = mat == 0 ? a.scales[0] : (mat == 1 ? a.scales[1] : a.scales[2]);
    r.codes[t] = buf_res(c + static_cast<int64_t>(first) * a.blocks * 16,
                         static_cast<uint32_t>(bytes < 0x7FFFFFFF ? bytes : 0x7FFFFFFF));
    r.scales[t] = buf_res(s + static_cast<int64_t>(first) * a.blocks,
                          static_cast<uint32_t>(left * a.blocks < 0x7FFFFFFF ? left * a.blocks : 0x7FFFFFFF));
  };
  if constexpr (EPI == kEpiRope) {
    const int per = mx_units<EPI, MT, NT>(a.N), half = a.head_dim / 2;
    const int mat = u / per, p0 = (u - mat * per) * (NT / 2) * kTile;
    const int first = (p0 / half) * a.head_dim + p0 % half;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int p = min(p0 + (t / 2) * kTile + i, a.N / 2 - 1);
      buffer(t, mat, first);
      r.row[t] = static_cast<uint32_t>((p / half) * a.head_dim + p % half + (t & 1) * half - first);
    }
  } else {
    const int first = u * kGroups<EPI, NT> * kTile;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int g = kPairs<EPI> ? t / 2 : t;
      buffer(t, kPairs<EPI> ? t & 1 : 0, first);
      r.row[t] = static_cast<uint32_t>(min(g * kTile + i, a.N - 1 - first));
    }
  }
}

// The chain of the input rows as norm_chain_mx_kernel defines it, in fp32: h = r + norm_a(x) through
// norm_f where there is one, rounded to bf16 once, and z = norm_b(h) rounded once.  (norm_chain_kernel
// rounds each norm and the sum, as the modules do.)  One row: the workgroup's threads hold its chunks.
template <int NC>
__device__ __forceinline__ void mx_chain(const NormArgs& c, bool write_h, const ChainIn<NC>& in, uint4 (&z)[NC], BlockSum& bs) {
  const float d = static_cast<float>(c.D);
  float h[NC][8];
  float ss = 0.0f;
  const auto add = [&](float v) { ss = fmaf(v, v, ss); };
  if (c.x != nullptr)
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float f[8];
      unpack_bf16x8(in.xr[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) add(f[e]);
    }
  const float ia = c.x != nullptr ? rsqrtf(bs(ss) / d + c.eps) : 0.0f;
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float f[8], w[8];
    unpack_bf16x8(in.rr[i], h[i]);
    unpack_bf16x8(in.xr[i], f);
    unpack_bf16x8(in.wa[i], w);
    if (c.x != nullptr)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = fmaf(w[e], f[e] * ia, h[i][e]);
#pragma unroll
    for (int e = 0; e < 8; ++e) add(h[i][e]);
  }
  if (c.wf != nullptr) {
    const float fi = rsqrtf(bs(ss) / d + c.eps);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float w[8];
      unpack_bf16x8(in.wf[i], w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = w[e] * (h[i][e] * fi);
    }
  }
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    z[i] = pack_bf16x8(h[i]);
    unpack_bf16x8(z[i], h[i]);
    const int q = static_cast<int>(threadIdx.x) + i * kNormThreads;
    if (write_h && c.h_out != nullptr && q < c.D / 8) reinterpret_cast<uint4*>(c.h_out)[q] = z[i];
#pragma unroll
    for (int e = 0; e < 8; ++e) add(h[i][e]);
  }
  if (c.wb == nullptr) return;
  const float ib = rsqrtf(bs(ss) / d + c.eps);
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float w[8];
    unpack_bf16x8(in.wb[i], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[i][e] = w[e] * (h[i][e] * ib);
    z[i] = pack_bf16x8(h[i]);
  }
}

// 1 / rms of a wave's row from its four partial sums (those of mx_chain's four waves, added in its order)
__device__ __forceinline__ float mx_wave_inv(float (&ss)[4], int D, float eps) {
#pragma unroll
  for (int i = 0; i < 4; ++i) ss[i] = wave_sum(ss[i]);
  const float inv = rsqrtf((((ss[0] + ss[1]) + ss[2]) + ss[3]) / static_cast<float>(D) + eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) ss[i] = 0.0f;
  return inv;
}

// The same by one wave (lane l: chunks l + 64 j); z (or h without n_b) in in.r.
template <int CH>
__device__ __forceinline__ void mx_wave_chain(const NormArgs& c, int64_t base, bool write_h, WaveChainIn<CH>& in) {
  float ss[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const auto add = [&](int j, const float* f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) ss[j & 3] = fmaf(f[e], f[e], ss[j & 3]);
  };
  float ia = 0.0f;
  if (c.x != nullptr) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float f[8];
      unpack_bf16x8(in.x[j], f);
      add(j, f);
    }
    ia = mx_wave_inv(ss, c.D, c.eps);
  }
  const auto sum_of = [&](int j, float* h) __attribute__((always_inline)) {
    unpack_bf16x8(in.r[j], h);
    if (c.x == nullptr) return;
    float f[8], w[8];
    unpack_bf16x8(in.x[j], f);
    unpack_bf16x8(in.wa[j], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = fmaf(w[e], f[e] * ia, h[e]);
  };
  float fi = 1.0f;
  if (c.wf != nullptr) {
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float h[8];
      sum_of(j, h);
      add(j, h);
    }
    fi = mx_wave_inv(ss, c.D, c.eps);
  }
  const BufRes wf = buf_res(c.wf, c.wf ? static_cast<uint32_t>(c.D) * 2u : 0u);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    float h[8];
    sum_of(j, h);
    if (c.wf != nullptr) {  // the last chain of a loop only: loaded here, so that the others keep the registers
      float w[8];
      unpack_bf16x8(buf_load16(wf, 16u * (threadIdx.x & 63u) + 1024u * j), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = w[e] * (h[e] * fi);
    }
    in.r[j] = pack_bf16x8(h);
    const int q = static_cast<int>(threadIdx.x & 63u) + 64 * j;
    if (write_h && c.h_out != nullptr && q < c.D / 8) reinterpret_cast<uint4*>(c.h_out + base)[q] = in.r[j];
    unpack_bf16x8(in.r[j], h);
    add(j, h);
  }
  if (c.wb == nullptr) return;
  const float ib = mx_wave_inv(ss, c.D, c.eps);
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    float h[8], w[8];
    unpack_bf16x8(in.r[j], h);
    unpack_bf16x8(in.wb[j], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = w[e] * (h[e] * ib);
    in.r[j] = pack_bf16x8(h);
  }
}

// This lane's block in step 0: wave, k-slice, quarter of the product.
template <int MT>
__device__ __forceinline__ uint32_t mx_lane_block() {
  using G = MxGeom<MT>;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  return static_cast<uint32_t>(4 * (wave * G::kSlices + (lane & 15) / G::kTile) + (lane >> 4));
}

template <int NT, int CS>
struct MxWeights {
  uint4 w[NT][CS];
  uint32_t s[NT][CS];
};

template <int MT, int NT, int CS>
__device__ __forceinline__ void mx_load_weights(const MxRows<NT>& r, uint32_t row_blocks, uint32_t blocks, uint32_t b0,
                                                MxWeights<NT, CS>& w) {
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const uint32_t b = b0 + s * (kMxStep / kMxBlock);
    const bool in = b < blocks;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w.w[t][s] = buf_load16(r.codes[t], in ? (r.row[t] * row_blocks + b) * 16u : kOutside);
      w.s[t][s] = __builtin_amdgcn_raw_buffer_load_b8(r.scales[t], static_cast<int>(in ? r.row[t] * row_blocks + b : kOutside), 0, 0);
    }
  }
}

// This lane's x of a step: the 32 values of its block in row lane % 8 (zero past K and past M).
template <int MT, int CS>
__device__ __forceinline__ void mx_load_x(const MxGemvArgs& a, BufRes xr, uint32_t b0, uint4 (&x)[CS][4]) {
  const uint32_t m = MT == 1 ? 0u : (threadIdx.x & 7u);
  const uint32_t es = a.x_f32 ? 4u : 2u;
  const uint32_t row = m * static_cast<uint32_t>(a.x_stride) * es;
  const bool live = static_cast<int>(m) < a.M;
#pragma unroll
  for (int s = 0; s < CS; ++s) {
    const uint32_t k0 = (b0 + s * (kMxStep / kMxBlock)) * kMxBlock;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t k = k0 + 8u * j;
      const uint32_t o = live && k < static_cast<uint32_t>(a.K) ? row + k * es : kOutside;
      if (a.x_f32) {
        const uint4 lo = buf_load16(xr, o), hi = buf_load16(xr, o + 16u);
        const float f[8] = {__uint_as_float(lo.x), __uint_as_float(lo.y), __uint_as_float(lo.z), __uint_as_float(lo.w),
                            __uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w)};
        x[s][j] = pack_bf16x8(f);
      } else {
        x[s][j] = buf_load16(xr, o);
      }
    }
  }
}

// Output (m, i-th row of the tile or pair g) of unit u from its sums; one rounding.
template <int EPI, int MT, int NT>
__device__ __forceinline__ void mx_store(const MxGemvArgs& a, int u, int g, int m, int i, float v, float v2) {
  constexpr int kTile = MxGeom<MT>::kTile;
  if constexpr (EPI == kEpiRope) {  // rotate_half(x)[c] = -x[c + half], [c + half] = x[c]
    const int per = mx_units<EPI, MT, NT>(a.N), half = a.head_dim / 2;
    const int mat = u / per, p = ((u - mat * per) * (NT / 2) + g) * kTile + i;
    if (p >= a.N / 2) return;
    const int c = p % half;
    uint16_t* y = static_cast<uint16_t*>(mat == 0 ? a.y[0] : (mat == 1 ? a.y[1] : a.y[2])) +
                  static_cast<int64_t>(m) * a.y_stride + (p / half) * a.head_dim + c;
    if (mat < 2) {
      const uint16_t* cs = a.cos + static_cast<int64_t>(m) * a.head_dim + c;
      const uint16_t* sn = a.sin + static_cast<int64_t>(m) * a.head_dim + c;
      const float lo = v * bf16_to_f32(cs[0]) - v2 * bf16_to_f32(sn[0]);
      v2 = v2 * bf16_to_f32(cs[half]) + v * bf16_to_f32(sn[half]);
      v = lo;
    }
    y[0] = f32_to_bf16_rne(v);
    y[half] = f32_to_bf16_rne(v2);
  } else {
    const int n = (u * kGroups<EPI, NT> + g) * kTile + i;
    if (n >= a.N) return;
    const int64_t o = static_cast<int64_t>(m) * a.y_stride + n;
    if constexpr (EPI == kEpiF32)
      static_cast<float*>(a.y[0])[o] = v;
    else if constexpr (EPI == kEpiAdd)
      static_cast<uint16_t*>(a.y[0])[o] = f32_to_bf16_rne(v + bf16_to_f32(a.addend[static_cast<int64_t>(m) * a.addend_stride + n]));
    else if constexpr (EPI == kEpiSwiGlu)
      static_cast<uint16_t*>(a.y[0])[o] = f32_to_bf16_rne(v / (1.0f + expf(-v)) * v2);
    else
      static_cast<uint16_t*>(a.y[0])[o] = f32_to_bf16_rne(v);
  }
}

// CS: steps of 2048 k whose weights are in registers together; K past CS of them goes round again
// (LOOP).  MT: rows of x (1, or up to 8).  NT: tiles of a unit.  DEPTH: units whose weights are in flight (1: a
// workgroup a unit; 2: a workgroup takes several, and the next one's weights are requested before the
// products of the one in hand).
template <int EPI, int MT, int CS, int NT, bool CHAIN, bool LOOP, int DEPTH>
__global__ __launch_bounds__(MxGeom<MT>::kThreads, 2) void mx_gemv_kernel(MxGemvArgs a, NormArgs c, int units) {
  using G = MxGeom<MT>;
  static_assert(!LOOP || DEPTH == 1);
  constexpr int kCap = CS * kMxStep;
  constexpr int kRow = kCap + 8;  // x row in LDS, elements
  __shared__ uint16_t xs[CHAIN ? MT * kRow : 8];
  __shared__ float red[DEPTH][G::kParts][NT][MT][G::kTile];
  __shared__ float nred[2][kNormWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t b0 = mx_lane_block<MT>();
  MxRows<NT> rows;
  MxWeights<NT, CS> w[DEPTH];
  int u = blockIdx.x;
  const int step = gridDim.x;
  const auto load = [&](int unit, int d) __attribute__((always_inline)) {
    // (past the last unit nothing is read)
    const uint32_t blocks = DEPTH == 1 || unit < units ? a.blocks : 0u;
    mx_unit_rows<EPI, MT, NT>(a, DEPTH == 1 ? unit : min(unit, units - 1), rows);
    mx_load_weights<MT, NT, CS>(rows, a.blocks, blocks, b0, w[d]);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto load_first = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(u + d * step, d);
  };
  uint4 x[CHAIN ? 1 : CS][4];
  BufRes xr;
  if constexpr (CHAIN && MT == 1) {
    static_assert(G::kThreads == kNormThreads, "one GEMV thread per chain thread");
    constexpr int NC = kCap / (kNormThreads * 8);
    ChainIn<NC> in;
    uint4 z[NC];
    BlockSum bs{nred, 0};
    chain_load<NC>(c, 0, in);
    __builtin_amdgcn_sched_barrier(0);  // the chain's inputs return before the weights
    load_first();
    mx_chain<NC>(c, blockIdx.x == 0, in, z, bs);
#pragma unroll
    for (int i = 0; i < NC; ++i)
      *reinterpret_cast<uint4*>(&xs[8 * (tid + i * kNormThreads)]) = z[i];
    lds_barrier();
  } else if constexpr (CHAIN) {
    constexpr int CH = kCap / 512;
    WaveChainIn<CH> in;  // wave w: row w
    const int64_t base = static_cast<int64_t>(min(wave, a.M - 1)) * c.stride;
    wave_chain_load<CH>(c, base, in);
    __builtin_amdgcn_sched_barrier(0);
    load_first();
    if (wave < a.M) {
      mx_wave_chain<CH>(c, base, blockIdx.x == 0, in);
#pragma unroll
      for (int j = 0; j < CH; ++j) *reinterpret_cast<uint4*>(&xs[wave * kRow + 8 * (lane + 64 * j)]) = in.r[j];
    } else {  // (columns that no output reads, but not whatever LDS held)
#pragma unroll
      for (int j = 0; j < CH; ++j) *reinterpret_cast<uint4*>(&xs[wave * kRow + 8 * (lane + 64 * j)]) = make_uint4(0, 0, 0, 0);
    }
    lds_barrier();
  } else {
    xr = buf_res(a.x, (static_cast<uint32_t>(a.M - 1) * static_cast<uint32_t>(a.x_stride) + a.K) * (a.x_f32 ? 4u : 2u));
    mx_load_x<MT, CS>(a, xr, b0, x);
    load_first();
  }

  const uint16_t* xl = &xs[CHAIN ? (MT == 1 ? 0 : (lane & 7)) * kRow + b0 * kMxBlock : 0];
  const auto multiply = [&](int d, f32x4_t(&acc)[NT]) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < CS; ++s) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bf16x8_t xv;
        if constexpr (CHAIN)
          xv = *reinterpret_cast<const bf16x8_t*>(xl + s * kMxStep + 8 * j);
        else
          xv = __builtin_bit_cast(bf16x8_t, x[s][j]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint4 q = w[d].w[t][s];
          const uint32_t code = j == 0 ? q.x : (j == 1 ? q.y : (j == 2 ? q.z : q.w));
          const uint4 wv = mx_decode4(code, mx_scale(w[d].s[t][s]));
          acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, wv), xv, acc[t], 0, 0, 0);
        }
      }
    }
  };
  const auto compute = [&](int d, int unit) __attribute__((always_inline)) {
    f32x4_t acc[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    multiply(d, acc);
    if constexpr (LOOP) {
      for (uint32_t at = b0 + CS * (kMxStep / kMxBlock); at - b0 < a.blocks; at += CS * (kMxStep / kMxBlock)) {  // (uniform)
        mx_load_x<MT, CS>(a, xr, at, x);
        mx_load_weights<MT, NT, CS>(rows, a.blocks, a.blocks, at, w[0]);
        multiply(0, acc);
      }
    }
    // lane l holds rows 4 (l / 16) ..+3 of column l % 16: the diagonal blocks are kept
    const int row = 4 * (lane >> 4), col = lane & 15;
    if (row / G::kTile == col / G::kTile && col % G::kTile < MT)
#pragma unroll
      for (int t = 0; t < NT; ++t)
        *reinterpret_cast<f32x4_t*>(&red[d][wave * G::kSlices + row / G::kTile][t][col % G::kTile][row % G::kTile]) = acc[t];
    lds_barrier();
    constexpr int kOuts = kGroups<EPI, NT> * MT * G::kTile;
    static_assert(kOuts <= G::kThreads, "one thread an output");
    const int i = tid % G::kTile, m = tid / G::kTile % MT, g = tid / (G::kTile * MT);
    if (tid < kOuts && m < a.M) {
      const int t0 = kPairs<EPI> ? 2 * g : g, t1 = kPairs<EPI> ? t0 + 1 : t0;
      float v = 0.0f, v2 = 0.0f;
#pragma unroll
      for (int p = 0; p < G::kParts; ++p) v += red[d][p][t0][m][i];
      if constexpr (kPairs<EPI>)
#pragma unroll
        for (int p = 0; p < G::kParts; ++p) v2 += red[d][p][t1][m][i];
      mx_store<EPI, MT, NT>(a, unit, g, m, i, v, v2);
    }
  };
  // (a buffer of partial sums is written again after the next unit's barrier)
  for (;; u += DEPTH * step)
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      compute(d, u + d * step);
      if (DEPTH == 1 || u + (d + 1) * step >= units) return;
      load(u + (d + DEPTH) * step, d);
    }
}

template <int EPI, int MT, int CS, int NT, bool CHAIN, bool LOOP, int DEPTH>
void mx_launch_form(const MxGemvArgs& a, const NormArgs& c, hipStream_t st, int workgroups) {
  const int units = mx_units<EPI, MT, NT>(a.N) * (EPI == kEpiRope ? 3 : 1);
  int grid = units;
  if (DEPTH > 1) {  // at most `workgroups`, each with the same number of units
    const int rounds = (units + workgroups - 1) / workgroups;
    grid = (units + rounds - 1) / rounds;
  }
  hipLaunchKernelGGL((mx_gemv_kernel<EPI, MT, CS, NT, CHAIN, LOOP, DEPTH>), dim3(grid), dim3(MxGeom<MT>::kThreads), 0, st, a, c,
                     units);
}

template <int EPI, int MT, int NT, bool CHAIN>
void mx_launch_k(const MxGemvArgs& a, const NormArgs& c, hipStream_t st) {
  if (a.K <= kMxStep) return mx_launch_form<EPI, MT, 1, NT, CHAIN, false, 1>(a, c, st, 0);
  if (CHAIN || a.K <= 2 * kMxStep) return mx_launch_form<EPI, MT, 2, NT, CHAIN, false, 1>(a, c, st, 0);
  if constexpr (!CHAIN) {
    if (a.K <= 3 * kMxStep) return mx_launch_form<EPI, MT, 3, NT, false, false, 1>(a, c, st, 0);
    if (a.K <= 4 * kMxStep) return mx_launch_form<EPI, MT, 4, NT, false, false, 1>(a, c, st, 0);
    mx_launch_form<EPI, MT, 4, NT, false, true, 1>(a, c, st, 0);
  }
}

// Every workgroup reads x, as many bytes as 4 (bf16, one row) or 32 (8 rows) of its W rows, so a unit has as
// many tiles as leave the CUs enough of them: 512 units, of 2 to 8 rows and one matrix 256.  Measured, us, one
// tile (pair) a unit, two, four: one row, K x N 2048 x 8192 5.2, 4.6, 4.6; 8192 x 8192 12.9, 10.7, 11.3; 2048 x
// 4096 3.7, 3.7, 3.8; SwiGLU 2048 x 5632 6.3, 5.4; q/k/v with RoPE 5.0, 5.2.  Eight rows, 2048 x 8192 7.9, 6.0,
// 5.4; 8192 x 8192 22.5, 16.1, 13.0; 5632 x 2048 6.2, 6.8, 8.4; SwiGLU 11264 wide 12.3, 9.8.
//
// A workgroup takes several units where its prologue would cost more than their weights -- eight chained
// rows, ~600 instructions each, run once a CU: SwiGLU 13.2 -> 8.0, q/k/v 9.8 -> 7.4, lm_head 49152 26.7
// -> 15.5 -- and in a head-sized matrix (lm_head 49152: one row 12.1 -> 11.6, eight 16.7 -> 13.7; 16384
// x 2048 loses, 6.1 -> 6.9 and 7.5 -> 7.8).  Around N 32768, where heads begin, a unit a workgroup and several, on
// weights that no cache holds, K 2048: one row 28672 8.5, 9.3; 32768 9.5, 9.6; 36864 10.9, 10.5; two rows
// 28672 9.9, 10.3; 36864 12.0, 11.9; 49152 15.5, 13.7; eight 28672 12.8, 11.0; 36864 15.3, 13.1.  K 4096, one row:
// 28672 15.3, 16.2; 32768 17.5, 16.5; 36864 19.9, 19.3.
template <int EPI, bool CHAIN>
void mx_launch(const MxGemvArgs& a, const NormArgs& c, hipStream_t st) {
  constexpr int kMats = EPI == kEpiRope ? 3 : 1;
  constexpr int kOne = kPairs<EPI> ? 2 : 1;  // tiles of the smallest unit
  const bool head = !kPairs<EPI> && a.N >= 32768;
  if (a.M == 1) {
    if constexpr (!kPairs<EPI>) {
      if (head && a.K <= kMxStep) return mx_launch_form<EPI, 1, 1, 2, CHAIN, false, 2>(a, c, st, 1024);
      if (head && a.K <= 2 * kMxStep) return mx_launch_form<EPI, 1, 2, 2, CHAIN, false, 2>(a, c, st, 1024);
    }
    if (kMats * mx_units<EPI, 1, 4>(a.N) >= 512) return mx_launch_k<EPI, 1, 4, CHAIN>(a, c, st);
    if (kMats * mx_units<EPI, 1, 2>(a.N) >= 512) return mx_launch_k<EPI, 1, 2, CHAIN>(a, c, st);
    return mx_launch_k<EPI, 1, kOne, CHAIN>(a, c, st);
  }
  if constexpr (CHAIN) {
    if constexpr (!kPairs<EPI>) {
      if (a.K <= kMxStep && head) return mx_launch_form<EPI, 8, 1, 4, true, false, 2>(a, c, st, 256);
      if (a.K <= kMxStep && a.N >= 8192) return mx_launch_form<EPI, 8, 1, 2, true, false, 2>(a, c, st, 256);
      if (head) return mx_launch_form<EPI, 8, 2, 2, true, false, 2>(a, c, st, 256);
    }
    if (a.K <= kMxStep) return mx_launch_form<EPI, 8, 1, kOne, true, false, 2>(a, c, st, 256);
    mx_launch_form<EPI, 8, 2, kOne, true, false, 2>(a, c, st, 256);
  } else {
    if constexpr (!kPairs<EPI>) {
      if (head && a.K <= kMxStep) return mx_launch_form<EPI, 8, 1, 2, false, false, 2>(a, c, st, 512);
      if (head && a.K <= 2 * kMxStep) return mx_launch_form<EPI, 8, 2, 2, false, false, 2>(a, c, st, 512);
    }
    const int least = kPairs<EPI> ? 512 : 256;
    if (kMats * mx_units<EPI, 8, 4>(a.N) >= least) return mx_launch_k<EPI, 8, 4, false>(a, c, st);
    if (kMats * mx_units<EPI, 8, 2>(a.N) >= least) return mx_launch_k<EPI, 8, 2, false>(a, c, st);
    mx_launch_k<EPI, 8, kOne, false>(a, c, st);
  }
}

template <bool CHAIN>
void mx_launch_epi(int epilogue, const MxGemvArgs& a, const NormArgs& c, hipStream_t st) {
  switch (epilogue) {
    case kEpiPlain: mx_launch<kEpiPlain, CHAIN>(a, c, st); break;
    case kEpiF32: mx_launch<kEpiF32, CHAIN>(a, c, st); break;
    case kEpiAdd: mx_launch<kEpiAdd, CHAIN>(a, c, st); break;
    case kEpiSwiGlu: mx_launch<kEpiSwiGlu, CHAIN>(a, c, st); break;
    default: mx_launch<kEpiRope, CHAIN>(a, c, st); break;
  }
}

// Rows of `cols` elements, `stride` apart, at p and at q share no memory: one lies behind the other, or both are
// columns of one wider matrix.
bool apart(const void* p, int64_t p_stride, int64_t p_cols, int p_size, const void* q, int64_t q_stride, int64_t q_cols, int q_size,
           int rows) {
  const int64_t a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(p)), b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(q));
  if (a == 0 || b == 0 || a + ((rows - 1) * p_stride + p_cols) * p_size <= b || b + ((rows - 1) * q_stride + q_cols) * q_size <= a)
    return true;
  const int64_t step = p_stride * p_size;
  if (step == 0 || step != q_stride * q_size) return false;
  const int64_t at = ((b - a) % step + step) % step;  // q's columns from p's first
  return p_cols * p_size <= at && at + q_cols * q_size <= step;
}

int32_t make_mx_args(MxGemvArgs& a, const void* x, int32_t x_is_f32, int64_t x_stride, int32_t m, int32_t k,
                     const uint8_t* const* codes, const uint8_t* const* scales, int32_t n, int32_t epilogue,
                     void* const* outputs, int64_t out_stride, const uint16_t* addend, int64_t addend_stride,
                     const uint16_t* rope_cos, const uint16_t* rope_sin, int32_t head_dim, const char* who) {
  const std::string w(who);
  FL_REQUIRE(x && codes && scales && outputs, w + ": null x/codes/scales/outputs");
  FL_REQUIRE(m >= 1 && m <= kMaxM, w + ": rows of x must be 1..8");
  // (a grid has at most 2^32 threads, 48 for each of N)
  FL_REQUIRE(k > 0 && k % 8 == 0 && k <= FL_MX_MAX_K && n > 0 && n <= (1 << 26),
             w + ": K must be a multiple of 8 (up to 2^20) and N positive (up to 2^26)");
  FL_REQUIRE(x_stride >= k && x_stride <= 0x7FFFFFFF / (4 * kMaxM) && out_stride >= n, w + ": bad row strides");
  FL_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && (x_stride * (x_is_f32 ? 4 : 2)) % 16 == 0,
             w + ": x rows must be 16-byte aligned");
  FL_REQUIRE(epilogue >= kEpiPlain && epilogue <= kEpiRope, w + ": unknown epilogue");
  const int nmat = epilogue == kEpiRope ? 3 : (epilogue == kEpiSwiGlu ? 2 : 1);
  for (int i = 0; i < nmat; ++i) {
    FL_REQUIRE(codes[i] != nullptr && scales[i] != nullptr && reinterpret_cast<uintptr_t>(codes[i]) % 16 == 0,
               w + ": codes must be non-null and 16-byte aligned, scales non-null");
    a.codes[i] = codes[i];
    a.scales[i] = scales[i];
  }
  for (int i = 0; i < (epilogue == kEpiRope ? 3 : 1); ++i) {
    FL_REQUIRE(outputs[i] != nullptr, w + ": null output");
    a.y[i] = outputs[i];
  }
  if (epilogue == kEpiAdd) FL_REQUIRE(addend != nullptr && addend_stride >= n, w + ": bad addend");
  a.blocks = static_cast<uint32_t>(mx_padded(k) / kMxBlock);
  if (epilogue == kEpiRope) {
    FL_REQUIRE(rope_cos && rope_sin && head_dim >= 8 && head_dim % 8 == 0 && n % head_dim == 0,
               w + ": rope needs cos/sin tables and N a multiple of head_dim (multiple of 8)");
    // (a unit's rows lie within one buffer of 2^31 bytes)
    FL_REQUIRE((static_cast<int64_t>(head_dim) + 64) * a.blocks * 16 < 0x7FFFFFFF, w + ": head too wide for this K");
  }
  for (int i = 0; i < (epilogue == kEpiRope ? 3 : 1); ++i)
    FL_REQUIRE(apart(outputs[i], out_stride, n, epilogue == kEpiF32 ? 4 : 2, x, x_stride, k, x_is_f32 ? 4 : 2, m),
               w + ": an output lies on x, which every workgroup reads");
  // (the addend's own place is fine: the thread that writes a value has read it)
  if (epilogue == kEpiAdd)
    FL_REQUIRE((outputs[0] == addend && out_stride == addend_stride) || apart(outputs[0], out_stride, n, 2, addend, addend_stride, n, 2, m),
               w + ": the output lies on other values of the addend");
  if (epilogue == kEpiRope)
    for (int i = 0; i < 3; ++i)
      FL_REQUIRE(apart(outputs[i], out_stride, n, 2, rope_cos, head_dim, head_dim, 2, m) &&
                     apart(outputs[i], out_stride, n, 2, rope_sin, head_dim, head_dim, 2, m),
                 w + ": an output lies on a rope table, which every head reads");
  a.x = x;
  a.x_f32 = x_is_f32 ? 1 : 0;
  a.x_stride = x_stride;
  a.M = m;
  a.K = k;
  a.N = n;
  a.y_stride = out_stride;
  a.addend = addend;
  a.addend_stride = addend_stride;
  a.cos = rope_cos;
  a.sin = rope_sin;
  a.head_dim = head_dim;
  return FL_OK;
}

}  // namespace
}  // namespace fl

extern "C" int32_t fl_mx_gemv(const void* x, int32_t x_is_f32, int64_t x_stride, int32_t m, int32_t k,
                              const uint8_t* const* codes, const uint8_t* const* scales, int32_t n, int32_t epilogue,
                              void* const* outputs, int64_t out_stride, const uint16_t* addend, int64_t addend_stride,
                              const uint16_t* rope_cos, const uint16_t* rope_sin, int32_t head_dim, void* stream) {
  using namespace fl;
  clear_error();
  MxGemvArgs a{};
  const int32_t rc = make_mx_args(a, x, x_is_f32, x_stride, m, k, codes, scales, n, epilogue, outputs, out_stride, addend,
                                  addend_stride, rope_cos, rope_sin, head_dim, "fl_mx_gemv");
  if (rc != FL_OK) return rc;
  mx_launch_epi<false>(epilogue, a, NormArgs{}, static_cast<hipStream_t>(stream));
  FL_LAUNCH_CHECK("fl_mx_gemv");
  return FL_OK;
}

extern "C" int32_t fl_mx_gemv_chain(int32_t m, int32_t k, float eps, const uint16_t* x, const uint16_t* r,
                                    const uint16_t* w_a, const uint16_t* w_f, const uint16_t* w_b, uint16_t* h_out,
                                    int64_t stride, const uint8_t* const* codes, const uint8_t* const* scales, int32_t n,
                                    int32_t epilogue, void* const* outputs, int64_t out_stride, const uint16_t* addend,
                                    int64_t addend_stride, const uint16_t* rope_cos, const uint16_t* rope_sin,
                                    int32_t head_dim, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(r != nullptr, "fl_mx_gemv_chain: null residual/input");
  FL_REQUIRE(k <= kMxChainMaxK && stride >= k && stride % 8 == 0,
             "fl_mx_gemv_chain: K must be at most 4096 and the chain row stride a multiple of 8 >= K");
  FL_REQUIRE(x == nullptr || w_a != nullptr, "fl_mx_gemv_chain: x needs its norm weight");
  for (const void* p : {static_cast<const void*>(x), static_cast<const void*>(r), static_cast<const void*>(w_a),
                        static_cast<const void*>(w_f), static_cast<const void*>(w_b), static_cast<const void*>(h_out)})
    FL_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "fl_mx_gemv_chain: every chain tensor must be 16-byte aligned");
  MxGemvArgs a{};
  // the GEMV's x is the chain output: its checks run on the residual row layout
  const int32_t rc = make_mx_args(a, r, 0, stride, m, k, codes, scales, n, epilogue, outputs, out_stride, addend,
                                  addend_stride, rope_cos, rope_sin, head_dim, "fl_mx_gemv_chain");
  if (rc != FL_OK) return rc;
  FL_REQUIRE(apart(h_out, stride, k, 2, r, stride, k, 2, m) && apart(h_out, stride, k, 2, x, stride, k, 2, m),
             "fl_mx_gemv_chain: h_out lies on r or x, which every workgroup reads");
  for (int i = 0; i < (epilogue == kEpiRope ? 3 : 1); ++i)
    FL_REQUIRE(apart(outputs[i], out_stride, n, epilogue == kEpiF32 ? 4 : 2, x, stride, k, 2, m),
               "fl_mx_gemv_chain: an output lies on x, which every workgroup reads");
  const NormArgs c{k, eps, x, r, w_a, w_f, w_b, h_out, nullptr, stride};
  mx_launch_epi<true>(epilogue, a, c, static_cast<hipStream_t>(stream));
  FL_LAUNCH_CHECK("fl_mx_gemv_chain");
  return FL_OK;
}
