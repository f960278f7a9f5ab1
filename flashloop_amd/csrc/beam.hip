// Beam search's selection: of every sequence's beams k and tokens t the `count` largest
//   total[k, t] = score[k] + x[k, t] - log(sum_t' exp(x[k, t'])),
// ties to the lower beam, then the lower token.
//
// One pass over the logits: a workgroup takes a part of a beam's row, 48 values a thread in registers, and
// gives the part's largest values in order and its sum of exponentials.  Of the 64 columns of threads (a lane of
// every wave) `count` have a maximum of at least the count-th largest of the columns' maxima, so only values that
// reach it can be among the largest: 18 of 12288 normal values for 16.  They are gathered in LDS and placed by
// counting.  Rows in which more values reach it than LDS holds (equal ones, masked ones) are inserted one by one
// into sorted lists, an entry a lane.  A second launch joins the parts of a sequence's beams, one list a lane.
// 256 rows of 49152 f32 values (50 MB), 16 results of each eight: 21.9 + 6.6 us (bf16: as long; 512 rows of bf16 45).  The
// bytes are 10 us of it, the exponentials in 64 bits 6, what follows a workgroup's last value 4 (what to reach 0.7, gathering
// 1.5, placing 1.2 in four barriers).  One sequence of four beams: 7.5 + 4.5 us, latencies; the join compares the lists'
// heads once a result, 0.2 us each (gathering what reaches the count-th largest head and counting places: 20 us slower, as
// the lists of a beam that leads hold most of their entries past it).
//
// The sums and totals are in 64 bits: totals of different beams decide the order among nearly equal
// candidates, and 32 bits would leave it to the order of the sum.  Within a beam the logits decide.
#include <algorithm>

#include "fl_common.h"

namespace fl {
namespace {

constexpr int kBeamThreads = 256;
constexpr int kBeamWaves = kBeamThreads / kWave;
constexpr int kPer = 16;                              // values of a thread in a chunk
constexpr int kChunks = 3;                            // chunks of a step
constexpr int kBeamChunk = kBeamThreads * kPer;       // values of a workgroup's chunk
constexpr int kBeamStep = kBeamChunk * kChunks;       // and step
constexpr int kMaxCount = kWave;                      // one list entry a lane
constexpr int kGathered = 128;                        // values of a wave that are placed by counting
constexpr int kLists = kWave;                         // lists of a sequence (beams * parts), one a lane

struct Entry {
  float value;
  int index;
};

struct PartHead {
  double sum;   // of exp(x - shift); NaN where the part holds a NaN or +inf
  float shift;  // a value of the part, at most 600 under its largest; -inf: the part holds nothing else
  int unused;
};

struct BeamArgs {
  const void* logits;  // [seqs * beams, vocab], row_stride apart
  int64_t row_stride;
  const float* scores;  // [seqs, beams]
  int seqs, beams, vocab, count, parts, part_len;
  PartHead* heads;  // [rows, parts]
  Entry* lists;     // [rows, parts, count]
  float* out_scores;
  int32_t* out_beams;
  int64_t* out_tokens;
};

// exp(t), t <= 600, to 2e-12 of it: t log2(e) = k + f, |f| <= 1/2, and the polynomial through 2^f at the nine Chebyshev
// points of [-1/2, 1/2] (1.1e-12; the series takes a degree more and a step more to its argument).
__device__ __forceinline__ double exp64(double t) {
  t = fmax(t, -800.0) * 1.4426950408889634;
  const double k = rint(t), f = t - k;
  double p = 1.325497460306718e-06;
  p = fma(p, f, 1.531007807039615e-05);
  p = fma(p, f, 0.00015403457039410448);
  p = fma(p, f, 0.0013333450573018062);
  p = fma(p, f, 0.009618129157656703);
  p = fma(p, f, 0.055504109412010456);
  p = fma(p, f, 0.24022650695821055);
  p = fma(p, f, 0.6931471805459343);
  p = fma(p, f, 1.0);  // (as exp(0) should be)
  return ldexp(p, static_cast<int>(k));
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}

// exp(shift - top): what sums with one shift are worth with another
__device__ __forceinline__ double scale_to(float shift, float top) {
  return shift == top ? 1.0 : (shift == -INFINITY ? 0.0 : exp64(static_cast<double>(shift) - top));
}

// a comes before b
__device__ __forceinline__ bool before(float av, int ai, float bv, int bi) { return av > bv || (av == bv && ai < bi); }

// x[kPer] <- values at index `from` .. of the row, four neighbouring ones a lane and load.  WHOLE: all of the chunk lie before
// `end`; else those past it are -inf.
template <bool F32, bool ALIGNED, bool WHOLE>
__device__ __forceinline__ void load_values(const BeamArgs& a, int64_t row, int from, int end, float* x) {
  const float* const wide = static_cast<const float*>(a.logits) + row * a.row_stride;
  const uint16_t* const half = static_cast<const uint16_t*>(a.logits) + row * a.row_stride;
#pragma unroll
  for (int j = 0; j < kPer / 4; ++j) {
    const int at = from + j * 4 * kWave;
    if (ALIGNED && WHOLE && F32) {
      const float4 v = *reinterpret_cast<const float4*>(wide + at);
      x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
    } else if (ALIGNED && WHOLE) {
      const uint2 v = *reinterpret_cast<const uint2*>(half + at);
      x[4 * j] = bf16lo_to_f32(v.x), x[4 * j + 1] = bf16hi_to_f32(v.x);
      x[4 * j + 2] = bf16lo_to_f32(v.y), x[4 * j + 3] = bf16hi_to_f32(v.y);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int one = WHOLE ? at + i : min(at + i, end - 1);
        const float v = F32 ? wide[one] : bf16_to_f32(half[one]);
        x[4 * j + i] = WHOLE || at + i < end ? v : -INFINITY;
      }
    }
  }
}

template <bool F32, bool ALIGNED>
__global__ __launch_bounds__(kBeamThreads) void beam_part_kernel(BeamArgs a) {
  __shared__ Entry gathered[kBeamWaves][kGathered], earlier[kMaxCount];  // this step's; the largest of those before
  __shared__ Entry best[kMaxCount];
  __shared__ float column[kBeamWaves][kWave];
  __shared__ PartHead heads[kBeamWaves];
  __shared__ int found[kBeamWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.parts;
  const int part = static_cast<int>(blockIdx.x - row * a.parts);
  const int begin = part * a.part_len, end = min(begin + a.part_len, a.vocab);

  float shift = -INFINITY;  // (wave-uniform)
  double sum = 0.0;         // of this lane's exp(x - shift)
  bool bad = false;
  int held = 0;  // entries of `best`
  // a wave's values of a chunk are neighbours: 1024 of them
  const int mine = begin + wave * (kWave * kPer) + 4 * lane;
  for (int base = begin; base < end; base += kBeamStep) {
    const int from = mine + (base - begin);
    float x[kChunks][kPer], mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (base + (c + 1) * kBeamChunk <= end) {
        load_values<F32, ALIGNED, true>(a, row, from + c * kBeamChunk, end, x[c]);
      } else if (base + c * kBeamChunk < end) {
        load_values<F32, ALIGNED, false>(a, row, from + c * kBeamChunk, end, x[c]);
      } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) x[c][e] = -INFINITY;
      }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (base + c * kBeamChunk >= end) continue;
      float top = x[c][0];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        bad = bad || !(x[c][e] < INFINITY);
        top = fmaxf(top, x[c][e]);
      }
      mx = fmaxf(mx, top);
      top = wave_max(top);
      if (top > shift && (shift == -INFINITY || top - shift > 600.0f)) {
        sum *= shift == -INFINITY ? 0.0 : exp64(static_cast<double>(shift) - top);
        shift = top;
      }
      if (shift > -INFINITY) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) sum += exp64(static_cast<double>(x[c][e]) - shift);
      }
    }
    column[wave][lane] = mx;
    __syncthreads();
    // what a value has to reach: the count-th largest of the columns' maxima
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) mx = fmaxf(mx, column[w][lane]);
    int above = 0;
#pragma unroll
    for (int j = 0; j < kWave; ++j) above += row_lane(mx, j) > mx ? 1 : 0;
    float reach = -wave_max(above < a.count ? -mx : -INFINITY);
    if (held == a.count) reach = fmaxf(reach, best[a.count - 1].value);
    int mine_found = 0;  // (wave-uniform)
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      if (base + c * kBeamChunk >= end) continue;
#pragma unroll
      for (int g = 0; g < kPer / 4; ++g) {  // (few groups of four values hold one that reaches it)
        const float most = fmaxf(fmaxf(x[c][4 * g], x[c][4 * g + 1]), fmaxf(x[c][4 * g + 2], x[c][4 * g + 3]));
        if (__builtin_amdgcn_ballot_w64(most >= reach) == 0ull) continue;
#pragma unroll
        for (int e = 4 * g; e < 4 * g + 4; ++e) {
          const int index = from + c * kBeamChunk + g * 4 * kWave + (e & 3);
          const bool in = x[c][e] >= reach && index < end;
          const unsigned long long who = __builtin_amdgcn_ballot_w64(in);
          const int at = mine_found + __builtin_popcountll(who & ((1ull << lane) - 1));
          if (in && at < kGathered) gathered[wave][at] = Entry{x[c][e], index};
          mine_found += __builtin_popcountll(who);
        }
      }
    }
    if (lane == 0) found[wave] = mine_found;
    if (tid < held) earlier[tid] = best[tid];
    __syncthreads();
    int count[kBeamWaves], total = held, most = 0;
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) {
      count[w] = __builtin_amdgcn_readfirstlane(found[w]);
      most = max(most, count[w]);
    }
    if (most > kGathered) {  // a sorted list a wave, entry `lane`, largest first
      __syncthreads();       // (every wave has read the counts)
      float lv = -INFINITY, last_v = -INFINITY;
      int li = 0x7FFFFFFF, last_i = 0x7FFFFFFF;  // last: entry count - 1
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
          const int index = from + c * kBeamChunk + (e >> 2) * 4 * kWave + (e & 3);
          const float v = x[c][e];
          unsigned long long in = __builtin_amdgcn_ballot_w64(v >= reach && index < end && before(v, index, last_v, last_i));
          while (in != 0ull) {
            const int l = __builtin_ctzll(in);
            in &= in - 1;
            const float cv = row_lane(v, l);
            const int ci = __builtin_amdgcn_readlane(index, l);
            if (!before(cv, ci, last_v, last_i)) continue;
            const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before(lv, li, cv, ci)));
            const float uv = __shfl_up(lv, 1, kWave);
            const int ui = __shfl_up(li, 1, kWave);
            lv = lane < at ? lv : (lane == at ? cv : uv);
            li = lane < at ? li : (lane == at ? ci : ui);
            last_v = row_lane(lv, a.count - 1);
            last_i = __builtin_amdgcn_readlane(li, a.count - 1);
          }
        }
      }
      // (entries that no value took come last: their index is no value's)
      gathered[wave][lane] = Entry{lv, li < 0x7FFFFFFF ? li : 0x7FFFFF00 + tid};
#pragma unroll
      for (int w = 0; w < kBeamWaves; ++w) count[w] = kWave;
      __syncthreads();
    }
    // an entry's place is the number of entries before it
#pragma unroll
    for (int w = 0; w < kBeamWaves; ++w) total += count[w];
    if (total <= kWave) {  // an entry a lane (what LDS would give one after the other comes from the lanes: 2.4 -> 0.5 us)
      if (wave == 0) {
        Entry one = earlier[min(lane, kMaxCount - 1)];
        int at = lane - held;
#pragma unroll
        for (int w = 0; w < kBeamWaves; ++w) {
          if (at >= 0 && at < count[w]) one = gathered[w][at];
          at -= count[w];
        }
        int place = 0;
#pragma unroll 4
        for (int l = 0; l < total; ++l)
          place += before(row_lane(one.value, l), __builtin_amdgcn_readlane(one.index, l), one.value, one.index) ? 1 : 0;
        if (lane < total && place < a.count) best[place] = one;
      }
    } else {
      const auto put = [&](Entry one) __attribute__((always_inline)) {
        int place = 0;
#pragma unroll 4
        for (int l = 0; l < held; ++l) place += before(earlier[l].value, earlier[l].index, one.value, one.index) ? 1 : 0;
#pragma unroll
        for (int w = 0; w < kBeamWaves; ++w)
#pragma unroll 4
          for (int l = 0; l < count[w]; ++l) place += before(gathered[w][l].value, gathered[w][l].index, one.value, one.index) ? 1 : 0;
        if (place < a.count) best[place] = one;
      };
      if (tid < held) put(earlier[tid]);
#pragma unroll
      for (int w = 0; w < kBeamWaves; ++w)
        if (w == wave)
          for (int l = lane; l < count[w]; l += kWave) put(gathered[w][l]);
    }
    held = min(a.count, total);
    __syncthreads();
  }

  const int64_t out = row * a.parts + part;
  if (tid < held) a.lists[out * a.count + tid] = best[tid];
  sum = wave_sum64(sum);
  if (__builtin_amdgcn_ballot_w64(bad) != 0ull) sum = NAN;
  if (lane == 0) heads[wave] = PartHead{sum, shift, 0};
  __syncthreads();
  if (tid == 0) {
    float t = heads[0].shift;
    for (int w = 1; w < kBeamWaves; ++w) t = fmaxf(t, heads[w].shift);
    double s = 0.0;
    for (int w = 0; w < kBeamWaves; ++w) s += heads[w].sum * scale_to(heads[w].shift, t);
    a.heads[out] = PartHead{s, t, 0};
  }
}

// order-preserving image of a double
__device__ __forceinline__ unsigned long long image(double v) {
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) { return max(v, static_cast<unsigned>(dpp_i<CTRL>(static_cast<int>(v)))); }
__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
  v = dpp_max<kDppXor1>(v);
  v = dpp_max<kDppXor2>(v);
  v = dpp_max<kDppHalfMirror>(v);
  v = dpp_max<kDppMirror>(v);
  const auto row = [&](int l) __attribute__((always_inline)) { return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), l)); };
  return max(max(row(0), row(16)), max(row(32), row(48)));
}
// lanes with the largest key; none where all are 0
__device__ __forceinline__ unsigned long long lanes_of_max(unsigned long long key) {
  const unsigned hi = static_cast<unsigned>(key >> 32), lo = static_cast<unsigned>(key);
  const unsigned top = wave_max_u32(hi);
  const bool first = hi == top && key != 0ull;
  const unsigned long long who = __builtin_amdgcn_ballot_w64(first);
  if ((who & (who - 1)) == 0ull) return who;
  const unsigned rest = first ? lo : 0u, most = wave_max_u32(rest);  // (by all lanes)
  return __builtin_amdgcn_ballot_w64(first && rest == most);
}

// One sequence: list `lane` is part lane % parts of beam lane / parts, so equal candidates go to the lower lane.
__global__ __launch_bounds__(kBeamThreads) void beam_join_kernel(BeamArgs a) {
  __shared__ Entry lists[kLists * kMaxCount];
  const int tid = threadIdx.x, lane = tid & 63, seq = blockIdx.x;
  const int used = a.beams * a.parts;
  const int64_t first = static_cast<int64_t>(seq) * used;
  const int beam = lane / a.parts, part = lane - beam * a.parts;  // (parts: a power of two)
  const bool any = beam < a.beams;
  const PartHead head = any ? a.heads[first + lane] : PartHead{0.0, -INFINITY, 0};
  const float score = any ? a.scores[seq * a.beams + beam] : 0.0f;
  for (int i = tid; i < used * a.count; i += kBeamThreads) lists[i] = a.lists[first * a.count + i];
  __syncthreads();
  if (tid >= kWave) return;
  // the beam's shift: score - logsumexp; -inf where it has no distribution or no finite score
  double shift = -INFINITY;
  float top = head.shift;
  for (int off = 1; off < a.parts; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
  double s = head.sum * scale_to(head.shift, top);
  for (int off = 1; off < a.parts; off <<= 1) s += __shfl_xor(s, off, kWave);
  if (any && top > -INFINITY && s == s && fabsf(score) < INFINITY) shift = static_cast<double>(score) - (top + log(s));
  const bool dead = shift == -INFINITY;
  const int left = min(a.part_len, a.vocab - part * a.part_len);  // values of the part
  const int held = beam < a.beams ? (dead && part > 0 ? 0 : min(a.count, dead ? a.vocab : left)) : 0;
  int at = 0, token = 0;
  float value = 0.0f;
  unsigned long long key = 0ull;  // of the list's next candidate; 0: none is left
  double total = 0.0;
  Entry ahead = lists[lane * a.count];  // the entry that comes next (read while others win)
  const auto look = [&]() __attribute__((always_inline)) {
    token = dead ? at : ahead.index;  // (equal totals: the tokens in order)
    value = dead ? 0.0f : ahead.value;
    total = dead ? -INFINITY : shift + static_cast<double>(ahead.value) + 0.0;  // (-0 becomes 0: they are equal, their images not)
    key = at < held ? image(total) : 0ull;
    ahead = lists[lane * a.count + min(at + 1, a.count - 1)];
  };
  look();
  for (int n = 0; n < a.count; ++n) {
    const unsigned long long who = lanes_of_max(key);
    if (who == 0ull) break;
    int winner = __builtin_ctzll(who);
    // totals of one beam may be equal in 64 bits where its logits are not: the logits decide
    for (unsigned long long rest = who & (who - 1); rest != 0ull; rest &= rest - 1) {
      const int l = __builtin_ctzll(rest);
      if (__builtin_amdgcn_readlane(beam, l) != __builtin_amdgcn_readlane(beam, winner)) break;
      if (row_lane(value, l) > row_lane(value, winner)) winner = l;
    }
    if (lane == winner) {
      const int64_t out = static_cast<int64_t>(seq) * a.count + n;
      a.out_scores[out] = static_cast<float>(total);
      a.out_beams[out] = beam;
      a.out_tokens[out] = token;
      ++at;
      look();
    }
  }
}

// Parts of a row: one step each, more where the rows are too few for the chip, and no more lists a sequence than
// lanes (then a part takes several steps).
int beam_parts(int64_t rows, int beams, int64_t vocab) {
  const int64_t least = (vocab + kBeamStep - 1) / kBeamStep, fill = (1024 + rows - 1) / rows;
  const int64_t parts = std::min<int64_t>(std::max(least, std::min<int64_t>(fill, (vocab + 1023) / 1024)), kLists / beams);
  int p = 1;  // (a power of two: a beam's parts are joined by exchanges)
  while (2 * p <= parts) p *= 2;
  return p;
}

}  // namespace
}  // namespace fl

extern "C" size_t fl_beam_select_workspace(int32_t seqs, int32_t beams, int64_t vocab, int32_t count) {
  using namespace fl;
  if (seqs <= 0 || beams <= 0 || beams > kLists || vocab <= 0 || count <= 0 || count > kMaxCount) return 0;
  const int64_t rows = static_cast<int64_t>(seqs) * beams;
  return static_cast<size_t>(rows * beam_parts(rows, beams, vocab)) * (sizeof(PartHead) + count * sizeof(Entry));
}

extern "C" int32_t fl_beam_select(const void* logits, int32_t logits_is_f32, int64_t row_stride, const float* scores, int32_t seqs,
                                  int32_t beams, int64_t vocab, int32_t count, float* out_scores, int32_t* out_beams,
                                  int64_t* out_tokens, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(logits && scores && out_scores && out_beams && out_tokens, "fl_beam_select: null pointer");
  FL_REQUIRE(seqs >= 0 && beams > 0 && beams <= kLists, "fl_beam_select: 1 to 64 beams");
  FL_REQUIRE(vocab > 0 && vocab <= (1 << 30), "fl_beam_select: 1 to 2^30 tokens");
  FL_REQUIRE(count > 0 && count <= kMaxCount && count <= beams * vocab, "fl_beam_select: 1 to 64 candidates, no more than there are");
  FL_REQUIRE(row_stride >= vocab, "fl_beam_select: rows must not overlap");
  FL_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (logits_is_f32 ? 4 : 2) == 0, "fl_beam_select: logits must be aligned");
  if (seqs == 0) return FL_OK;
  const int64_t rows = static_cast<int64_t>(seqs) * beams;
  FL_REQUIRE(rows <= 0x7FFFFFFF / kLists / kBeamThreads, "fl_beam_select: too many rows");
  FL_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 &&
                 workspace_bytes >= fl_beam_select_workspace(seqs, beams, vocab, count),
             "fl_beam_select: workspace too small or not 16-byte aligned");
  const int parts = beam_parts(rows, beams, vocab);
  // whole steps of 4 values a part, so that aligned rows give aligned parts
  const int part_len = static_cast<int>((vocab + 4 * parts - 1) / (4 * parts) * 4);
  PartHead* heads = static_cast<PartHead*>(workspace);
  const BeamArgs a{logits, row_stride, scores, seqs, beams, static_cast<int>(vocab), count, parts, part_len, heads,
                   reinterpret_cast<Entry*>(heads + rows * parts), out_scores, out_beams, out_tokens};
  const bool aligned = reinterpret_cast<uintptr_t>(logits) % (logits_is_f32 ? 16 : 8) == 0 && row_stride % 4 == 0;
  const dim3 grid(static_cast<unsigned>(rows * parts)), block(kBeamThreads);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (logits_is_f32) {
    if (aligned)
      hipLaunchKernelGGL((beam_part_kernel<true, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((beam_part_kernel<true, false>), grid, block, 0, st, a);
  } else {
    if (aligned)
      hipLaunchKernelGGL((beam_part_kernel<false, true>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((beam_part_kernel<false, false>), grid, block, 0, st, a);
  }
  FL_LAUNCH_CHECK("fl_beam_select");
  hipLaunchKernelGGL(beam_join_kernel, dim3(static_cast<unsigned>(seqs)), block, 0, st, a);
  FL_LAUNCH_CHECK("fl_beam_select(join)");
  return FL_OK;
}
