// Attention of new tokens over K/V pages: softmax(q K^T) V of a ragged batch whose keys and values lie in
// pages [pages, KV heads, page, 128] named by a table.  The rows of a sequence are its last tokens, a row
// sees the keys up to its own position; the query heads of a group share one KV head, so a group's rows
// (token i, head g of the group: row i * group + g) are the queries of that head's keys.
//
//  * chunk_kernel: chunks of new tokens.  A workgroup has 256 queries in eight waves, one workgroup a CU; S^T and O^T on
//    v_mfma_f32_32x32x16_bf16, 64 keys a step, K and V through a ring of four tiles in LDS that transfers without registers
//    fill.  A long prompt (8192 tokens, 16 heads) 285-290 us: 950-970 TFLOP/s of the causal half.  On the same transfers with no
//    arithmetic between the products it runs at 1550 TFLOP/s of those it has (the card's power sets that rate); the rest are the
//    exponentials, the roundings to bf16 and the moves of the softmax's reference in the products' shadow, one behind the other in
//    a wave.
//  * step_kernel: few queries a sequence (one decode step).  A wave owns steps of 32 keys and up to 16
//    queries on v_mfma_f32_16x16x32_bf16: K goes from memory into the first product's operand, V through a
//    part of LDS of the wave's own, the next step's loads in flight, no barrier until the waves' join.  Bound by bytes: 32
//    sequences of up to 8192 tokens, 16 heads, 185 us, 5.6 TB/s.  One sequence of 2048 tokens takes 7 us, five memory latencies.
//  * join_kernel and join_slices_kernel join the parts where a launch divides keys.
//
// A key that a row does not see has no part in its result, whatever its K and V rows hold: scores are
// replaced, V rows past a sequence's end are zeroed, and where some row of a tile does not see a key, the
// key's infinite and NaN values are zeroed too and added for the rows that see it afterwards.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "attn_common.h"
#include "lds_load.h"

namespace fl {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kChunkWaves = 8;           // waves of a workgroup of chunk_kernel
constexpr int kChunkThreads = kChunkWaves * kWave;
constexpr int kChunkRows = 32 * kChunkWaves;  // its queries
constexpr int kStepKeys = 32;            // keys of a wave's step in step_kernel
constexpr int kStepRows = 16;            // its queries
constexpr int kMaxRanges = kWave;        // parts of an item's keys: step_kernel's join has one a lane
// Workgroups that a call aims at
constexpr int kStepAim = 1024;
constexpr int kChunkAim = 256;          // (one a CU: its LDS is theirs)
// least steps of a range in step_kernel, one a wave; and up to which a sequence alone is one range (512 tokens 14 us in four,
// 10.5 in one)
constexpr int kStepLeast = kWaves, kStepWhole = 16;

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// Arrays that a launch only reads, at wave-uniform indexes: as constant memory their loads are scalar ones, which
// leave the vector loads in flight alone (read as ordinary memory, each page number waited for all of them).
typedef const __attribute__((address_space(4))) int32_t* uniform_ints;
__device__ __forceinline__ uniform_ints uniform(const int32_t* p) {
  return reinterpret_cast<uniform_ints>(reinterpret_cast<uintptr_t>(p));
}

struct PagedArgs {
  const uint16_t* q;  // rows [n, heads * 128], q_row apart
  int64_t q_row;
  const uint16_t* k;  // pages [pages, kv, page, 128]
  const uint16_t* v;
  uint16_t* o;           // [n, heads * 128]
  const int32_t* table;  // [seqs, width]
  const int32_t* lens;   // [seqs]
  const int32_t* starts; // [seqs + 1], or null: row s is sequence s's
  int n, seqs, heads, kv, group, width, pages, page_log2;
  float scale;  // scaling * log2(e)
  // Divided keys.  aim: step_kernel's workgroups aimed at, chunk_kernel's slices a KV head; 0: nothing is divided.  And the
  // workspace for their outputs
  int aim, ranges, slots, items;  // ranges of an item at most; ranges' outputs a KV head and divided items that there is room for
  int32_t* divided;       // number of divided items (step_kernel)
  struct Divided* list;   // [items]
  float2* part_ml;        // [kv][slots][rows of an item]: maximum of q.k (kUnseen: no key) and sum
  float* part_o;          // [kv][slots][rows of an item][128]
};

// An item whose keys are divided: queries [item * ROWS, ..) of the rows [first, first + rows), in `ranges` slots.
struct Divided {
  int32_t first, rows, item, ranges, slot;
};

// the maximum of a query that sees no key (kNone: its scores are all -inf)
constexpr float kUnseen = -INFINITY;

// The rows [first, first + rows) of sequence s, within the call's whatever `starts` holds.
__device__ __forceinline__ int2 rows_of(const PagedArgs& a, int s) {
  if (a.starts == nullptr) return make_int2(s, 1);
  const int first = min(max(a.starts[s], 0), a.n);
  return make_int2(first, min(max(a.starts[s + 1], first), a.n) - first);
}

// The same of one sequence of the whole wave.
__device__ __forceinline__ int2 rows_of_one(const PagedArgs& a, int s) {
  if (a.starts == nullptr) return make_int2(s, 1);
  const uniform_ints starts = uniform(a.starts);
  const int first = min(max(starts[s], 0), a.n);
  return make_int2(first, min(max(starts[s + 1], first), a.n) - first);
}

// One sequence's pages of one KV head.
struct Pages {
  uniform_ints table;
  int width, pages, log2, last;  // last: its last key that a table entry can name
  int64_t page_elems, head_elems;
  // Page of the 16 keys from `key` (a multiple of 16, at most `last`) on, as the table has it.
  __device__ __forceinline__ int page(int key) const { return table[key >> log2]; }
  __device__ __forceinline__ bool exists(int id) const { return static_cast<unsigned>(id) < static_cast<unsigned>(pages); }
  // First element of these 16 keys; of page 0 where they have no page.
  __device__ __forceinline__ int64_t at(int id, int key) const {
    return (exists(id) ? id : 0) * page_elems + head_elems + static_cast<int64_t>(key & ((1 << log2) - 1)) * kDim;
  }
};

__device__ __forceinline__ Pages pages_of(const PagedArgs& a, int s, int head, int len) {
  Pages p;
  p.table = uniform(a.table + static_cast<int64_t>(s) * a.width);
  p.width = a.width;
  p.pages = a.pages;
  p.log2 = a.page_log2;
  p.last = static_cast<int>(min(static_cast<int64_t>(len), static_cast<int64_t>(a.width) << a.page_log2)) - 1;
  p.page_elems = static_cast<int64_t>(a.kv) << (a.page_log2 + 7);
  p.head_elems = static_cast<int64_t>(head) << (a.page_log2 + 7);
  return p;
}

__device__ __forceinline__ int items_of(const PagedArgs& a, int rows, int each) { return (rows * a.group + each - 1) / each; }

// The keys of a sequence that its table row can name.
__device__ __forceinline__ int keys_of(const PagedArgs& a, int len) {
  return static_cast<int>(min(static_cast<int64_t>(max(len, 0)), static_cast<int64_t>(a.width) << a.page_log2));
}

// v of the lane that CTRL names, in the rows of 16 lanes of MASK; elsewhere 0
template <int CTRL, int MASK>
__device__ __forceinline__ int from_lane(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, MASK, 0xF, false); }
template <int CTRL, int MASK>
__device__ __forceinline__ double from_lane(double v) {
  const int64_t u = __double_as_longlong(v);
  const int lo = from_lane<CTRL, MASK>(static_cast<int>(u)), hi = from_lane<CTRL, MASK>(static_cast<int>(u >> 32));
  return __longlong_as_double((static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo));
}
// sum over the lanes up to this one: within rows of 16, then with the rows before
template <class T>
__device__ __forceinline__ T scan_lanes(T v) {
  v += from_lane<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
  v += from_lane<0x112, 0xF>(v);
  v += from_lane<0x114, 0xF>(v);
  v += from_lane<0x118, 0xF>(v);
  v += from_lane<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  return v + from_lane<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// step_kernel's work.  An item is a sequence with up to 16 queries, against its keys in steps; where the items are too few
// for the chip, or too unequal, a sequence's are divided into ranges of about T steps, T such that the call makes about `aim`
// workgroups.  Every workgroup finds this out for itself, sequences in lanes: the lengths are on the device alone.  Since
// a divided item has more than T steps, there are at most 2 aim / kv ranges of divided ones.
struct Work {
  int seq, range, ranges;
  int slot;  // of its first range's output (ranges > 1)
};

// index: this workgroup's number for its KV head.  (Sequences of more than 16 queries -- short
// ones of wide groups, or more rows than max_q says -- are never divided.)
__device__ __forceinline__ bool find_work(const PagedArgs& a, int head, int index, Work& w) {
  const int lane = threadIdx.x & 63;
  const auto look = [&](int s, int& items, int& steps, bool& whole) __attribute__((always_inline)) {
    const int2 rows = s < a.seqs ? rows_of(a, s) : make_int2(0, 0);
    const int keys = s < a.seqs ? keys_of(a, a.lens[s]) : 0;
    items = min(rows.y, 1);
    whole = items_of(a, rows.y, kStepRows) > 1;
    steps = (keys + kStepKeys - 1) / kStepKeys;
  };
  int items, steps;
  bool whole;
  look(lane, items, steps, whole);
  float sum = wave_sum(static_cast<float>(items) * static_cast<float>(steps)), number = wave_sum(static_cast<float>(items));
  for (int base = kWave; base < a.seqs; base += kWave) {
    int its, sts;
    bool all;
    look(base + lane, its, sts, all);
    sum += wave_sum(static_cast<float>(its) * static_cast<float>(sts));
    number += wave_sum(static_cast<float>(its));
  }
  // T: two rounds of the workgroups that the CUs hold, one where it is of no more than 16 steps each (one sequence of 8192 tokens,
  // 16 heads: 25 us in two rounds, 20 in one).  Each sequence's last range is half a one on average: without that some
  // workgroups are left for a round of their own (48 sequences 85 -> 82.5 us, 12 of 8000 76 -> 72).
  const float aim = sum * a.kv <= 8.0f * a.aim ? 0.5f * a.aim : a.aim;
  const int most = max(kStepLeast, static_cast<int>(fminf(ceilf(sum * a.kv / fmaxf(aim - 0.5f * number * a.kv, 0.5f * aim)), 1e9f)));
  w.seq = -1;
  int total = 0, slots = 0, divided = 0;
  for (int base = 0; base < a.seqs; base += kWave) {
    if (base > 0) look(base + lane, items, steps, whole);
    const int ranges = whole ? 1 : min(max(1, (steps + most - 1) / most), a.ranges);
    const int groups = items * ranges, parts = ranges > 1 ? groups : 0, split = ranges > 1 ? items : 0;
    const int to = total + scan_lanes(groups), slots_to = slots + scan_lanes(parts), split_to = divided + scan_lanes(split);
    const unsigned long long past = __builtin_amdgcn_ballot_w64(to > index);
    if (w.seq < 0 && past != 0ull) {
      const int l = __builtin_ctzll(past);
      w.seq = base + l;
      w.ranges = __builtin_amdgcn_readlane(ranges, l);
      w.range = index - (__builtin_amdgcn_readlane(to, l) - w.ranges);
      w.slot = __builtin_amdgcn_readlane(slots_to, l) - w.ranges;
      if (w.ranges > 1 && head == 0 && w.range == 0 && threadIdx.x == 0) {
        const int2 rows = rows_of_one(a, w.seq);
        a.list[__builtin_amdgcn_readlane(split_to, l) - 1] = Divided{rows.x, rows.y, 0, w.ranges, w.slot};
      }
      if (index != 0) return true;
    }
    total = __builtin_amdgcn_readlane(to, kWave - 1);
    slots = __builtin_amdgcn_readlane(slots_to, kWave - 1);
    divided = __builtin_amdgcn_readlane(split_to, kWave - 1);
  }
  if (head == 0 && index == 0 && threadIdx.x == 0) *a.divided = divided;
  return w.seq >= 0;
}

// Rows that belong to no sequence: zeros, by all workgroups.
__device__ __forceinline__ void clear_behind(const PagedArgs& a, int head, int index, int threads) {
  if (a.starts == nullptr) return;
  const int behind = min(max(uniform(a.starts)[a.seqs], 0), a.n), groups = static_cast<int>(gridDim.x) / a.kv, width = a.group * kDim / 8;
  for (int64_t row = static_cast<int64_t>(behind) + index; row < a.n; row += groups)
    for (int c = threadIdx.x; c < width; c += threads)
      *reinterpret_cast<uint4*>(a.o + (row * a.heads + head * a.group) * kDim + 8 * c) = make_uint4(0, 0, 0, 0);
}

// Infinite and NaN values of a chunk of 8 bf16 become zeros; returns whether there were any.
__device__ __forceinline__ bool drop_nonfinite(u32x4_t& w) {
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool lo = (w[i] & 0x7F80u) == 0x7F80u, hi = (w[i] & 0x7F800000u) == 0x7F800000u;
    any = any || lo || hi;
    w[i] &= (lo ? 0u : 0xFFFFu) | (hi ? 0u : 0xFFFF0000u);
  }
  return any;
}
// w * v where v is infinite or NaN, else 0
__device__ __forceinline__ float nonfinite_part(float w, float v) { return fabsf(v) < INFINITY ? 0.0f : w * v; }
__device__ __forceinline__ void add_nonfinite(float w, uint2 v, float& a, float& b, float& c, float& d) {
  a += nonfinite_part(w, bf16lo_to_f32(v.x));
  b += nonfinite_part(w, bf16hi_to_f32(v.x));
  c += nonfinite_part(w, bf16lo_to_f32(v.y));
  d += nonfinite_part(w, bf16hi_to_f32(v.y));
}

__device__ __forceinline__ uint2 pair4(const float* o, float inv) {
  return make_uint2(attn_bf16_pair(o[0] * inv, o[1] * inv), attn_bf16_pair(o[2] * inv, o[3] * inv));
}

// read_v_tr (attn_common.h) of an address that is known to be one in LDS, so that fixed distances are offsets of the read
typedef const __attribute__((address_space(3))) uint16_t* lds_rows;
__device__ __forceinline__ lds_rows as_lds(const uint16_t* p) {
  return reinterpret_cast<lds_rows>(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)));
}
__device__ __forceinline__ bf16x4_t read_tr(lds_rows p) {
  typedef __attribute__((address_space(3))) bf16x4_t lds_t;
  return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_t*)p);
}

// The chunk kernel's LDS: four tiles each of K and V, rows of 256 bytes as 16 pieces of 16.  Piece p of K row r lies at
// p ^ (r % 16): the 32 rows of an operand read meet all banks.  Piece p of V row r at p ^ 4 (r % 4): so do the four rows of a
// transposed read's 16 lanes.
constexpr int kRing = 4;
constexpr int kTileBytes = kKeys * kDim * 2;

// f(0), f(1), .. with constant arguments
template <int... I, class F>
__device__ __forceinline__ void slots(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>{}), ...);
}

// chunk_kernel's work.  An item is up to 256 queries of a sequence against the keys up to its last one.  Where keys are
// divided, a KV head's items lie one after another on a line, each as long as its keys (times `group`) and kApart steps of 64
// more; the line is cut into `aim` equal slices, and a workgroup takes a slice: the end of one item, whole ones, the
// beginning of another.  So the workgroups end at about the same time, however unequal the sequences are.  (20 sequences of
// 1-700 new tokens over up to 3000, 16 heads on 4: 112 us as whole items, 88 in slices; 8 of up to 300 over 6000, 16 heads:
// 170, 98; four of 40 over 9000: 209, 59.)  Else a workgroup takes one item, a sequence's last ones first: they see more
// keys.  Every workgroup finds its work for itself, sequences in lanes: the lengths are on the device alone.
// kApart: beginning a part costs some 10 us, finding it, first latencies and the stores (3, 5, 7, 10 steps: these 20 sequences
// 95, 90, 88, 92 us; 12 of up to 2000 over 8000, 32 heads on 4, 540, 523, 514, 511).
constexpr double kApart = 7.0;
constexpr int kLeastSteps = 7;  // of a slice; a cut moves by less than 2

// One sequence's items on the line.
struct Line {
  int q, items;   // queries, items
  double before;  // of each item: keys before the call's, and kApart
  __device__ __forceinline__ Line(const PagedArgs& a, int rows, int keys) {
    q = rows * a.group;
    items = items_of(a, rows, kChunkRows);
    before = static_cast<double>(max(keys - rows, 0)) * a.group + kApart * kKeys * a.group;
  }
  // where item i begins (i = items: where the last one ends)
  __device__ __forceinline__ double at(int i) const {
#pragma clang fp contract(off)  // (all workgroups get the same, wherever this is inlined)
    const double n = i;
    return n * before + (i < items ? 0.5 * kChunkRows * n * (n + 1) : 0.5 * kChunkRows * n * (n - 1) + q);
  }
};

// The step of the `all` of an item at begins .. ends that a cut falls on: none within two of the item's ends.
__device__ __forceinline__ int cut_at(double cut, double begins, double ends, double apart, double scale, int all) {
#pragma clang fp contract(off)
  const double steps = (cut - begins - apart) * scale;
  return cut >= ends || steps > all - 2 ? all : (steps < 2.0 ? 0 : static_cast<int>(steps));
}

__device__ __forceinline__ double lane_f64(double v, int l) {
  const int64_t u = __double_as_longlong(v);
  const int lo = __builtin_amdgcn_readlane(static_cast<int>(u), l), hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), l);
  return __longlong_as_double((static_cast<int64_t>(hi) << 32) | static_cast<uint32_t>(lo));
}

// Where a wave is on the line.  (In LDS, each wave's its own: no register is held while it works on a part.)
struct Walk {
  double x, begin, end, slice;  // the next item; the workgroup's slice; a slice's length
  double from;                  // where the sequences from `base` on begin
  int base, opens;              // opens: the slice ends in an item that it begins
};

// chunk_kernel's arguments, read again where this stands: held all at once over its loop they leave no scalar register, and
// from where the launch put them they take a microsecond.
__device__ __forceinline__ PagedArgs args_again(const PagedArgs& lds) {
  asm volatile("" ::: "memory");
  constexpr int kWords = sizeof(PagedArgs) / 4;
  int w[kWords];
#pragma unroll
  for (int i = 0; i < kWords; ++i) w[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(&lds)[i]);
  PagedArgs a;
  __builtin_memcpy(&a, w, sizeof(a));
  // (pointers to global memory: the compiler knows it of arguments only)
  const auto global = [](auto*& p) __attribute__((always_inline)) {
    typedef typename std::remove_reference<decltype(*p)>::type value_t;
    p = (value_t*)(__attribute__((address_space(1))) value_t*)p;
  };
  global(a.q), global(a.k), global(a.v), global(a.o), global(a.table), global(a.lens), global(a.starts), global(a.list);
  global(a.part_ml), global(a.part_o);
  return a;
}

__global__ __launch_bounds__(kChunkThreads, 2) void chunk_kernel(PagedArgs first_args) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds_all[2 * kRing * kTileBytes];
  __shared__ unsigned long long odd_keys[4];  // by tile % 4: keys of a tile with infinite or NaN values
  __shared__ int no_page;                     // the first key without a page
  __shared__ Walk walk[kChunkWaves];
  __shared__ PagedArgs args;
  __shared__ int3 line_of[kChunkWaves][kWave];    // a lane's sequence: first row, rows, length
  __shared__ double line_to[kChunkWaves][kWave];  // where the lane's sequence of the 64 from `base` on ends, from `from` on
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = static_cast<int>(blockIdx.x) % first_args.kv, mine_index = static_cast<int>(blockIdx.x) / first_args.kv;

  // the lane's sequence of those from `base` on: into line_of, and where it ends into line_to
  const auto look = [&](const PagedArgs& a, int s, double& to, double& most) __attribute__((always_inline)) {
    const int known = min(s, a.seqs - 1);  // (the loads one beside the other)
    const int given = a.lens[known];
    int2 rows = rows_of(a, known);
    rows.y = s < a.seqs ? rows.y : 0;
    const int len = s < a.seqs ? max(given, 0) : 0;
    const Line line(a, rows.y, keys_of(a, len));
    to = scan_lanes(a.aim > 0 ? (line.items > 0 ? line.at(line.items) : 0.0) : static_cast<double>(line.items));
    most = fmax(most, line.before + line.q);
    line_to[wave][lane] = to;
    line_of[wave][lane] = make_int3(rows.x, rows.y, len);
  };
  {
    const PagedArgs a = first_args;
    double to, most = 0.0, x = mine_index, x_end = mine_index + 1.0, slice = 1.0;
    if (lane == 0) args = a;
    if (a.aim > 0) {
      double total = 0.0;
      for (int base = (a.seqs - 1) / kWave * kWave; base >= 0; base -= kWave) {  // (the first ones last: they stay)
        look(a, base + lane, to, most);
        total += lane_f64(to, kWave - 1);
      }
      // (An item lies in at most 64 slices.  More gain nothing, as the join takes eight parts after another: one sequence with slices
      // of seven steps instead, 32 rows over 100000 tokens, 8 heads on one, 70 -> 77 us, 256 over 40000, one head, 46.7 -> 47.4.  `most` in
      // 32 bits and a little more.)
      const double longest = 1.001 * wave_max(static_cast<float>(most));
      slice = fmax(total / a.aim, fmax(static_cast<double>(kLeastSteps) * kKeys * a.group, longest * (1.0 / (kMaxRanges - 2))));
      x = mine_index < a.aim ? mine_index * slice : 1e300;
      x_end = mine_index + 1 < a.aim ? (mine_index + 1) * slice : 1e300;
    } else {
      look(a, lane, to, most);
    }
    walk[wave] = Walk{x, x, x_end, slice, 0.0, 0, 0};
  }

  while (true) {
    const PagedArgs a = args_again(args);
    int tid = threadIdx.x, index = mine_index;
    asm volatile("" : "+v"(tid), "+s"(index));  // (nor is what depends on it held from part to part)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    double to = line_to[wave][lane];
    int3 of = line_of[wave][lane];
    const double x = walk[wave].x, x_begin = walk[wave].begin, x_end = walk[wave].end, slice = walk[wave].slice;
    if (__builtin_amdgcn_readfirstlane(x >= x_end)) break;
    double from = walk[wave].from;
    int base = __builtin_amdgcn_readfirstlane(walk[wave].base);
    unsigned long long past;
    while ((past = __builtin_amdgcn_ballot_w64(from + to > x)) == 0ull) {
      base += kWave;
      if (base >= a.seqs) break;
      from += lane_f64(to, kWave - 1);
      double unused = 0.0;
      look(a, base + lane, to, unused);
      of = line_of[wave][lane];
      walk[wave].from = from;
      walk[wave].base = base;
    }
    if (past == 0ull) break;
    const int who = __builtin_ctzll(past), seq = base + who;
    const double start = from + (who > 0 ? lane_f64(to, who - 1) : 0.0), stop = from + lane_f64(to, who);
    const int2 rows = make_int2(__builtin_amdgcn_readlane(of.x, who), __builtin_amdgcn_readlane(of.y, who));
    const int len = __builtin_amdgcn_readlane(of.z, who);
    const Pages pages = pages_of(a, seq, head, len);
    const Line line(a, rows.y, pages.last + 1);
    int item = 0;
    double begins = 0.0, ends = 0.0;  // the item's place on the line
    if (a.aim > 0) {
      for (int high = line.items - 1; item < high;) {
        const int mid = item + (high - item + 1) / 2;
        if (__builtin_amdgcn_readfirstlane(start + line.at(mid) <= x))
          item = mid;
        else
          high = mid - 1;
      }
      begins = start + line.at(item);
      ends = item + 1 < line.items ? start + line.at(item + 1) : stop;
    } else {
      item = line.items - 1 - static_cast<int>(x - start);
      ends = x + 1.0;
    }
    item = __builtin_amdgcn_readfirstlane(item);
    walk[wave].x = ends;
    const auto position = [&](int query) __attribute__((always_inline)) { return len - rows.y + min(query, line.q - 1) / a.group; };
    const int low = position(item * kChunkRows), end = min(position((item + 1) * kChunkRows - 1), pages.last);
    const int all = end >= 0 ? end / kKeys + 1 : 0;
    int tiles = all, first = 0, parts = 1;  // this slice's; slices of the item
    if (a.aim > 0) {
      // scale: steps a unit of the line, never less than a step for each 64 keys of it.  An item that sees fewer keys than its
      // length stands for (rows in front of the sequence's first key, a length past the table) would else be spread so thin
      // that a slice in its middle gets no step, and the join would read a part that no workgroup has written.
      const double apart = kApart * kKeys * a.group, scale = fmax(all / (ends - begins - apart), 1.0 / (kKeys * a.group));
      const auto cut = [&](double at) __attribute__((always_inline)) { return cut_at(at, begins, ends, apart, scale, all); };
      first = __builtin_amdgcn_readfirstlane(x_begin <= begins ? 0 : cut(x_begin));
      tiles = __builtin_amdgcn_readfirstlane(cut(x_end));
      if (__builtin_amdgcn_readfirstlane(all > 0 ? first >= tiles : x_begin > begins)) continue;  // (the next or the last slice has it)
      if (first > 0 || tiles < all) parts = 2;
      if (first == 0 && tiles < all) {
        walk[wave].opens = 1;
        if (head == 0 && tid == 0) {
          int last = min(static_cast<int>(ends / slice), a.aim - 1);
          while (last > index && (last * slice >= ends || cut(last * slice) >= all)) --last;
          a.list[index] = Divided{rows.x, rows.y, item, last - index + 1, 2 * index + 1};
        }
      }
    }
    const int part_slot = 2 * index + (first == 0 ? 1 : 0);
    // this lane's query: column lane % 32 of the wave's
    const int pos = position(item * kChunkRows + wave * 32 + (lane & 31));
    const int wmin = position(item * kChunkRows + wave * 32), wmax = position(item * kChunkRows + wave * 32 + 31);
    if (tid < 4) odd_keys[tid] = 0ull;
    if (tid == 0) no_page = 0x7FFFFFFF;
    const int mine = min(tiles, (wmax >> 6) + 1);  // tiles that some query of the wave sees (none: at most `first`)

    f32x16_t o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    // the reference of the running softmax (a score, and it scaled to base 2), this lane's parts of the sum
    float raw = kNone, off = -scaled_max(kNone, a.scale), sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    bool far = false;  // (wave-uniform) some query's reference lies past kFar

    if (first < tiles) {
      bf16x8_t q[8];
      const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_u8*)lds_all));
      constexpr uint32_t kV = kRing * kTileBytes;  // V's tiles lie behind K's

      // Transfers: a wave brings the 8 keys 8 w .. of a tile, which share a page: twice four rows.  Their places for 64
      // tiles lie in the lanes of two registers (a scalar load among a tile's LDS reads would make their waits wait for all).
      uint32_t kv[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) kv[i] = 1024 * i + 256 * (lane >> 4) + 16 * ((lane & 15) ^ (8 * (wave & 1) + 4 * i + (lane >> 4)));
      const uint32_t vv = 256 * (lane >> 4) + 16 * ((lane & 15) ^ (4 * (lane >> 4)));
      const auto block_key = [&](int tile) __attribute__((always_inline)) {
        return min(min(tile, tiles - 1) * kKeys + 8 * (wave & ~1), pages.last & ~15);
      };
      uint32_t at_lo = 0, at_hi = 0;  // bytes from the pool's start
      int at_from = 0, lost = 0x7FFFFFFF;  // lost: the first key of this wave's without a page
      const auto look_up = [&](int tile) __attribute__((always_inline)) {
        at_from = tile;
        const int key = block_key(tile + lane);
        const int id = *(a.table + static_cast<int64_t>(seq) * a.width + (key >> pages.log2));
        __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): it, and q before the first, have arrived here, and no use waits for them
        const uint64_t at = 2 * static_cast<uint64_t>(pages.at(id, key) + 8 * (wave & 1) * kDim);
        at_lo = static_cast<uint32_t>(at);
        at_hi = static_cast<uint32_t>(at >> 32);
        const unsigned long long none = __builtin_amdgcn_ballot_w64(!pages.exists(id));
        if (none != 0ull) lost = min(lost, __builtin_amdgcn_readlane(key, __builtin_ctzll(none)));
      };
      const auto place = [&](int tile) __attribute__((always_inline)) {  // of the wave's keys of a tile
        return (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_hi), tile - at_from))) << 32) |
               static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at_lo), tile - at_from));
      };
      // (past the last tile: of no bytes, so that it moves none, and the number of transfers in flight is the same)
      const auto part_of = [&](const uint16_t* pool, int tile, uint64_t at) __attribute__((always_inline)) {
        const uint64_t u = reinterpret_cast<uintptr_t>(pool) + at;
        return lds_buffer_t{static_cast<int>(u), static_cast<int>(u >> 32), tile < tiles ? 8 * kDim * 2 : 0, 0x00020000};
      };
      const auto ring = [&](int tile) __attribute__((always_inline)) { return static_cast<uint32_t>((tile - first) % kRing) * kTileBytes; };
      const auto bring_k = [&](int tile, uint64_t at) __attribute__((always_inline)) {
        const lds_buffer_t r = part_of(a.k, tile, at);
        const uint32_t to = lds0 + ring(tile) + 2048u * wave;
        to_lds<16>(r, kv[0], 0, to);
        to_lds<16>(r, kv[1], 0, to + 1024u);
      };
      const auto bring_v = [&](int tile, uint64_t at) __attribute__((always_inline)) {
        const lds_buffer_t r = part_of(a.v, tile, at);
        const uint32_t to = lds0 + kV + ring(tile) + 2048u * wave;
        to_lds<16>(r, vv, 0, to);
        to_lds<16>(r, vv, 1024u, to + 1024u);
      };
      // This wave's V rows of a tile, arrived: zeros past the sequence's end, and in the place of infinite and NaN values that
      // some row does not see
      const auto mend = [&](int tile) __attribute__((always_inline)) {
        if (tile >= tiles || tile * kKeys + kKeys - 1 <= low) return;
        uint32_t bits = 0;
        uint8_t* const at = lds_all + kV + ring(tile) + 2048 * wave + 16 * lane;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = tile * kKeys + 8 * wave + 4 * i + (lane >> 4);
          u32x4_t v = *reinterpret_cast<u32x4_t*>(at + 1024 * i);
          bool any = false;
          if (key > pages.last)
            v = u32x4_t{0, 0, 0, 0};
          else if (key > low)
            any = drop_nonfinite(v);
          if (any || key > pages.last) *reinterpret_cast<u32x4_t*>(at + 1024 * i) = v;
          const unsigned long long lanes = __builtin_amdgcn_ballot_w64(any);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((lanes >> (16 * j)) & 0xFFFFull) bits |= 1u << (4 * i + j);
        }
        if (bits != 0 && lane == 0) atomicOr(&odd_keys[tile & 3], static_cast<unsigned long long>(bits) << (8 * wave));
      };

      // Operands: K fragment i is rows lane % 32 of half i % 2 of the tile, channels 16 (i / 2) + 8 h ..; V fragment j rows
      // 16 (j / 4) + 4 h .. (+ 8), channels 32 (j % 4) + ..
      typedef const __attribute__((address_space(3))) uint8_t* lds_at;
      uint32_t kx[8], vx[4];
      const int i16 = lane & 15;
#pragma unroll
      for (int st = 0; st < 8; ++st) kx[st] = lds0 + 256 * (lane & 31) + (16 * (h ^ i16) ^ 32 * st);
#pragma unroll
      for (int d = 0; d < 4; ++d) vx[d] = lds0 + kV + 256 * (4 * h + (i16 >> 2)) + 32 * ((lane >> 4) & 1) + 8 * (i16 & 3) + (64 * (i16 >> 2) ^ 64 * d);
      const auto k_part = [&](uint32_t of, int i) __attribute__((always_inline)) {
        return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>(reinterpret_cast<lds_at>(kx[i >> 1] + of) + 8192 * (i & 1));
      };
      const auto v_part = [&](uint32_t of, int j) __attribute__((always_inline)) {
        const lds_at at = reinterpret_cast<lds_at>(vx[j & 3] + of) + 4096 * (j >> 2);
        const bf16x4_t lo = read_tr((lds_rows)at), hi = read_tr((lds_rows)(at + 2048));
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      };
      const auto scores_part = [&](int i, bf16x8_t k, f32x16_t (&s)[2]) __attribute__((always_inline)) {
        f32x16_t zero;
#pragma unroll
        for (int e = 0; e < 16; ++e) zero[e] = 0.0f;
        s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[i >> 1], i < 2 ? zero : s[i & 1], 0, 0, 0);
      };
      // probabilities 2 k and 2 k + 1 of the tile's 32 a lane: words of the second product's operand
      u32x4_t p[4];
      const auto pair = [&](int k, const f32x16_t (&s)[2]) __attribute__((always_inline)) {
        const int t = k >> 2, e = 8 * (t & 1) + 2 * (k & 3);
        const float p0 = fast_exp2(fmaf(s[t >> 1][e], a.scale, off)), p1 = fast_exp2(fmaf(s[t >> 1][e + 1], a.scale, off));
        p[t][k & 3] = attn_bf16_pair(p0, p1);
        sum[k & 3] = add_pair(p[t][k & 3], sum[k & 3]);
      };
      const auto outputs_part = [&](int j, bf16x8_t v) __attribute__((always_inline)) {
        o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8_t, p[j >> 2]), o[j & 3], 0, 0, 0);
      };
      const auto hide = [&](int tile, f32x16_t (&s)[2]) __attribute__((always_inline)) {
        if (tile * kKeys + kKeys - 1 > wmin) {  // keys past a query's position
          const int lim = pos - tile * kKeys - 4 * h;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (32 * b + 8 * (i >> 2) + (i & 3) > lim) s[b][i] = -INFINITY;
        }
      };
      const auto largest = [&](const f32x16_t (&s)[2]) __attribute__((always_inline)) {
        float m = s[0][0];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 16; ++i) m = fmaxf(m, s[b][i]);
        return m;
      };
      // The reference is the largest score so far, so that the largest probability is 1 and has no rounding: it carries much of a
      // row.  (Moved only where a score passes it by 2^8, most tiles leave the outputs alone, 8192 prompt rows 289 -> 270 us, and the
      // result is off by 2.10e-3 of its norm instead of 1.87e-3, of which its own rounding is 1.65e-3.)
      const auto move_to = [&](float m, f32x16_t (&s)[2]) __attribute__((always_inline)) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
        m = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
        if (__builtin_amdgcn_ballot_w64(m > raw) != 0ull) {
          const float top = fmaxf(raw, m), mn = scaled_max(top, a.scale);
          const float alpha = exp2_between(raw, top, scaled_max(raw, a.scale), mn, a.scale);
          raw = top;
          off = -mn;
          far = __builtin_amdgcn_ballot_w64(fabsf(mn) > kFar && top > kNone) != 0ull;
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] *= alpha;
#pragma unroll
          for (int d = 0; d < 4; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
        }
        if (far) {  // (differences before the scale)
          off = 0.0f;
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] -= raw;
        }
      };
      const auto add_odd = [&](int tile) __attribute__((always_inline)) {
        if (tile * kKeys + kKeys - 1 <= low) return;
        for (unsigned long long odd = odd_keys[tile & 3]; odd != 0ull; odd &= odd - 1) {
          // key j lies in result register 4 (j / 8) + j % 4 of lane half j / 4 % 2
          const int j = __builtin_amdgcn_readfirstlane(__builtin_ctzll(odd)), e = 4 * (j >> 3) + (j & 3);
          const int key = tile * kKeys + j;
          const uint16_t* vp = a.v + pages.at(pages.page(key & ~15), key & ~15) + (key & 15) * kDim + 4 * h;
          float w = 0.0f;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (8 * t + i == e) w = static_cast<float>(__builtin_bit_cast(bf16x8_t, p[t])[i]);
          w = __shfl(w, (lane & 31) + 32 * ((j >> 2) & 1), kWave);
          if (key <= pos) {
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const uint2 v = *reinterpret_cast<const uint2*>(vp + 32 * d + 8 * g);
                float x[4] = {o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
                add_nonfinite(w, v, x[0], x[1], x[2], x[3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) o[d][4 * g + i] = x[i];
                __builtin_amdgcn_sched_barrier(0);  // (a piece at a time: this path must not set the kernel's registers)
              }
          }
        }
      };

      const int token = pos - len + rows.y, out_head = head * a.group + min(item * kChunkRows + wave * 32 + (lane & 31), line.q - 1) - token * a.group;
      const uint16_t* qp = a.q + (rows.x + token) * a.q_row + out_head * kDim + 8 * h;
#pragma unroll
      for (int s = 0; s < 8; ++s) q[s] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * s);
      look_up(first);
      uint64_t at_v = 0;  // place of the tile whose V goes next
      {
        uint64_t at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = place(first + i);
        bring_k(first, at[0]);
        bring_v(first, at[0]);
        bring_k(first + 1, at[1]);
        bring_k(first + 2, at[2]);
        bring_v(first + 1, at[1]);
        bring_k(first + 3, at[3]);
        bring_v(first + 2, at[2]);
        at_v = at[3];
      }
      asm volatile("s_waitcnt vmcnt(12)" ::: "memory");  // K of the first tile
      lds_barrier();
      f32x16_t sa[2], sb[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) scores_part(i, k_part(ring(first), i), sa);
      hide(first, sa);
      move_to(largest(sa), sa);
      asm volatile("s_waitcnt vmcnt(6)" ::: "memory");  // all but V of the second and third, K of the fourth
      lds_barrier();

      // One tile: the next one's scores (matrix slots 0-15) and this one's outputs (16-31), with this one's exponentials and
      // then the next one's maximum spread over the slots, so that the vector unit works in the matrix core's shadow.
      // Fragments are read four slots ahead, the first four of the tile after that before the barrier: K arrives two tiles
      // before its scores, V one before its outputs.  EDGE: some row of the workgroup does not see some key of this tile or
      // the next.  The order is kept by hand: left to it, the compiler computes all exponentials at once.
      bf16x8_t ahead[4];
      const auto flow = [&](int tile, uint32_t v_at, uint32_t k_at, uint32_t k_then, f32x16_t (&now)[2], f32x16_t (&next)[2],
                            auto edge_tag) __attribute__((always_inline)) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        bf16x8_t kf[16], vf[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) kf[i] = ahead[i];
        float m = kNone;
        uint64_t at = 0;
        slots(std::make_integer_sequence<int, 32>{}, [&](auto slot) __attribute__((always_inline)) {
          constexpr int i = decltype(slot)::value;
          if constexpr (i < 12)
            kf[i + 4] = k_part(k_at, i + 4);
          else if constexpr (i < 28)
            vf[i - 12] = v_part(v_at, i - 12);
          else
            ahead[i - 28] = k_part(k_then, i - 28);
          if constexpr (i < 16)
            scores_part(i, kf[i], next);
          else
            outputs_part(i - 16, vf[i - 16]);
          // 16 pairs over the slots 0-25 (operand t is complete well before slot 16 + 4 t)
          constexpr int k = (3 * i + 2) / 5;
          if constexpr (i < 26 && 5 * k / 3 == i) {
            asm volatile("" : "+v"(off));  // (no pair is computed before its slot)
            pair(k, now);
          }
          if constexpr (i == 2) bring_v(tile + 3, at_v);
          if constexpr (i == 4) at = place(tile + 4);
          if constexpr (i == 7) bring_k(tile + 4, at);
          if constexpr (EDGE && i == 18) hide(tile + 1, next);
          if constexpr (i >= 26 || i == 19 || i == 24) {  // 4 scores a time
            constexpr int e = i >= 26 ? 2 + (i - 26) : (i == 19 ? 0 : 1);
#pragma unroll
            for (int x = 0; x < 4; ++x) m = fmaxf(m, next[e >> 2][4 * (e & 3) + x]);
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        at_v = at;
        if (EDGE) add_odd(tile);
        if (tile + 1 < tiles) move_to(m, next);
      };
      const auto arrive = [&](int tile) __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        __builtin_amdgcn_s_barrier();  // (this wave's reads of what the next transfers replace are done: their results were used)
        asm volatile("" ::: "memory");
        if (tile + 8 >= at_from + kWave) look_up(tile + 5);
      };
      int tile = first;
#pragma unroll
      for (int i = 0; i < 4; ++i) ahead[i] = k_part(ring(tile + 1), i);
      // (four tiles at a time: their places in the ring are constants, and the scores change places)
      for (; tile + 4 <= tiles && min(tile + 5, tiles) * kKeys - 1 <= low; tile += 4) {
        constexpr uint32_t kT = kTileBytes;
        flow(tile, 0 * kT, 1 * kT, 2 * kT, sa, sb, std::false_type{});
        arrive(tile);
        flow(tile + 1, 1 * kT, 2 * kT, 3 * kT, sb, sa, std::false_type{});
        arrive(tile + 1);
        flow(tile + 2, 2 * kT, 3 * kT, 0 * kT, sa, sb, std::false_type{});
        arrive(tile + 2);
        flow(tile + 3, 3 * kT, 0 * kT, 1 * kT, sb, sa, std::false_type{});
        arrive(tile + 3);
      }
      // The last tiles, of which some row does not see some key
      mend(tile);
      lds_barrier();
      const auto last = [&](f32x16_t (&now)[2], f32x16_t (&next)[2]) __attribute__((always_inline)) {
        if (tid == 0) odd_keys[(tile + 2) & 3] = 0ull;
        if (tile < mine) {
          flow(tile, ring(tile), ring(tile + 1), ring(tile + 2), now, next, std::true_type{});
        } else {
          bring_v(tile + 3, at_v);
          at_v = place(tile + 4);
          bring_k(tile + 4, at_v);
        }
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        mend(tile + 1);
        lds_barrier();
        if (tile + 8 >= at_from + kWave) look_up(tile + 5);
        ++tile;
      };
      while (tile < tiles) {
        last(sa, sb);
        if (tile < tiles) last(sb, sa);
      }
      if (lost != 0x7FFFFFFF && lane == 0) atomicMin(&no_page, lost);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing is on its way into LDS when the workgroup ends)
      lds_barrier();
    }

    float l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    // NaN: a sequence longer than its table row, a key without a page
    l += swap_half(l) + ((len - 1 > pages.last && pos >= 0) || pos >= no_page ? NAN : 0.0f);
    const PagedArgs e = args_again(args);
    const int r = item * kChunkRows + wave * 32 + (lane & 31), token = pos - len + rows.y;
    const bool valid = r < rows.y * e.group;
    if (parts > 1) {
      const int64_t part = static_cast<int64_t>(head) * e.slots + part_slot;
      float* const op = e.part_o + ((part * kChunkWaves + wave) * 16 * kWave + lane) * 4;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(op + (4 * d + g) * kWave * 4) =
              make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
      if (h == 0) e.part_ml[part * kChunkRows + wave * 32 + lane] = make_float2(pos >= first * kKeys ? raw : kUnseen, l);
    } else if (valid) {
      const float inv = pos >= 0 ? 1.0f / l : 0.0f;
      uint16_t* op = e.o + (static_cast<int64_t>(rows.x + token) * e.heads + head * e.group + r - token * e.group) * kDim + 4 * h;
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float y[4] = {o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
          *reinterpret_cast<uint2*>(op + 32 * d + 8 * g) = pair4(y, inv);
        }
    }
    lds_barrier();  // (no_page and the tiles are the next part's)
  }
  const PagedArgs a = args_again(args);
  if (a.aim > 0 && walk[wave].opens == 0 && head == 0 && tid == 0 && mine_index < a.aim) a.list[mine_index].ranges = 0;
  clear_behind(a, head, mine_index, kChunkThreads);
}

__global__ __launch_bounds__(kThreads, 2) void step_kernel(PagedArgs a) {
  // a wave's V rows of 256 bytes; 32-byte piece d of row r lies at d ^ (r % 8), so that the 16 rows of a transposed
  // read cover all banks without padding
  __shared__ __attribute__((aligned(16))) uint16_t lds[kWaves][kStepKeys * kDim];
  __shared__ float2 wave_ml[kWaves][kStepRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const int head = static_cast<int>(blockIdx.x) % a.kv, index = static_cast<int>(blockIdx.x) / a.kv;
  clear_behind(a, head, index, kThreads);
  Work w{index, 0, 1, 0};
  if (a.aim > 0 ? !find_work(a, head, index, w) : index >= a.seqs) return;
  const int seq = __builtin_amdgcn_readfirstlane(w.seq), ranges = __builtin_amdgcn_readfirstlane(w.ranges);
  const int2 rows = rows_of_one(a, seq);
  const int len = max(uniform(a.lens)[seq], 0);
  const Pages pages = pages_of(a, seq, head, len);

  for (int base = 0; base < rows.y * a.group; base += kStepRows) {
    const int rc = min(base + c, rows.y * a.group - 1);
    const int token = rc / a.group, out_head = head * a.group + rc - token * a.group;
    const int64_t row = rows.x + token;
    const int pos = len - rows.y + token;
    const int low = len - rows.y + base / a.group;
    const int end = min(len - rows.y + min(base + kStepRows - 1, rows.y * a.group - 1) / a.group, pages.last);
    int steps = end >= 0 ? end / kStepKeys + 1 : 0, first = 0;
    if (ranges > 1) {
      const int range = __builtin_amdgcn_readfirstlane(w.range);
      first = static_cast<int>(static_cast<int64_t>(steps) * range / ranges);
      steps = static_cast<int>(static_cast<int64_t>(steps) * (range + 1) / ranges);
    }
    bf16x8_t q[4];
    {
      const uint16_t* qp = a.q + row * a.q_row + out_head * kDim + 8 * g;
#pragma unroll
      for (int st = 0; st < 4; ++st) q[st] = *reinterpret_cast<const bf16x8_t*>(qp + 32 * st);
    }
    f32x4_t o[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) o[d] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float raw = kNone, m = scaled_max(kNone, a.scale), l = 0.0f;
    float poison = len - 1 > pages.last && pos >= 0 ? NAN : 0.0f;
    bool far = false;

    bf16x8_t kr[2][4];
    u32x4_t vr[8];
    int ids[2];
    const auto look_up = [&](int step) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) ids[b] = pages.page(min(step * kStepKeys + 16 * b, pages.last & ~15));
    };
    const auto fetch = [&](int step) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = min(step * kStepKeys + 16 * b, pages.last & ~15);
        if (!pages.exists(ids[b]) && pos >= key) poison = NAN;
        const int64_t at = pages.at(ids[b], key);
        const uint16_t* kp = a.k + at + c * kDim + 8 * g;
        const uint16_t* vp = a.v + at + g * kDim + 8 * c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          kr[b][i] = *reinterpret_cast<const bf16x8_t*>(kp + 32 * i);
          vr[4 * b + i] = *reinterpret_cast<const u32x4_t*>(vp + 4 * i * kDim);
        }
      }
    };
    uint16_t* const vl = lds[wave];
    const int turn = (4 * g + (c >> 2)) & 7;  // of the rows that this lane reads, 4 g + c / 4 and 16 further
    const lds_rows vt = as_lds(vl + (4 * g + (c >> 2)) * kDim + 4 * (c & 3));
    const int begin = __builtin_amdgcn_readfirstlane(first + wave);
    if (begin < steps) {
      look_up(begin);
      fetch(begin);
      look_up(min(begin + kWaves, steps - 1));
    }
    for (int step = begin; step < steps; step += kWaves) {
      f32x4_t s[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        s[b] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < 4; ++st) s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr[b][st], q[st], s[b], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + g;
        *reinterpret_cast<u32x4_t*>(&vl[r * kDim + 8 * (c ^ (2 * (r & 7)))]) = vr[i];
      }
      uint32_t odd = 0;  // keys with infinite or NaN values that some row does not see
      if (step * kStepKeys + kStepKeys - 1 > low) {
        // (rows are mended where they lie: mended before they are written, they would all be copied first)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int r = 4 * i + g, key = step * kStepKeys + r;
          u32x4_t v = vr[i];
          bool any = false;
          if (key > pages.last) {
            v = u32x4_t{0, 0, 0, 0};
          } else if (key > low) {
            any = drop_nonfinite(v);
          }
          if (any || key > pages.last) *reinterpret_cast<u32x4_t*>(&vl[r * kDim + 8 * (c ^ (2 * (r & 7)))]) = v;
          const unsigned long long lanes = __builtin_amdgcn_ballot_w64(any);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((lanes >> (16 * j)) & 0xFFFFull) odd |= 1u << (4 * i + j);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (step * kStepKeys + 16 * b + 4 * g + i > pos) s[b][i] = -INFINITY;
      }
      if (step + kWaves < steps) {
        fetch(step + kWaves);
        look_up(min(step + 2 * kWaves, steps - 1));
      }
      __builtin_amdgcn_sched_barrier(0);  // the loads leave before the softmax, however many registers that takes
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
      mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
      if (__builtin_amdgcn_ballot_w64(mx > raw) != 0ull) {
        const float top = fmaxf(raw, mx), mn = scaled_max(top, a.scale);
        const float alpha = exp2_between(raw, top, m, mn, a.scale);
        raw = top;
        m = mn;
        l *= alpha;
        far = __builtin_amdgcn_ballot_w64(fabsf(m) > kFar && raw > kNone) != 0ull;
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d][i] *= alpha;
      }
      float off = -m;
      if (far) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[b][i] -= raw;
        off = 0.0f;
      }
      // the second product's k index 8 g + 4 b + i is key 16 b + 4 g + i: the scores stay in their lanes
      u32x4_t w;
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = fast_exp2(fmaf(s[b][2 * i], a.scale, off)), p1 = fast_exp2(fmaf(s[b][2 * i + 1], a.scale, off));
          w[2 * b + i] = attn_bf16_pair(p0, p1);
          sum[b] = add_pair(w[2 * b + i], sum[b]);
        }
      l += sum[0] + sum[1];
      const bf16x8_t p = __builtin_bit_cast(bf16x8_t, w);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const lds_rows piece = vt + 16 * (d ^ turn);
        const bf16x4_t lo = read_tr(piece), hi = read_tr(piece + 16 * kDim);
        const bf16x8_t va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, p, o[d], 0, 0, 0);
      }
      __builtin_amdgcn_wave_barrier();
      for (odd = __builtin_amdgcn_readfirstlane(odd); odd != 0; odd &= odd - 1) {
        const int j = __builtin_ctz(odd), e = 4 * (j >> 4) + (j & 3);  // register e of lane group j / 4 % 4
        float pw = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i == e) pw = static_cast<float>(p[i]);
        pw = __shfl(pw, c + 16 * ((j >> 2) & 3), kWave);
        const int key = step * kStepKeys + j;
        if (key <= pos) {
          const uint16_t* vp = a.v + pages.at(pages.page(key & ~15), key & ~15) + (key & 15) * kDim + 4 * g;
#pragma unroll
          for (int d = 0; d < 8; ++d) {  // (a piece at a time: this path must not set the kernel's registers)
            const uint2 v = *reinterpret_cast<const uint2*>(vp + 16 * d);
            float e[4] = {o[d][0], o[d][1], o[d][2], o[d][3]};
            add_nonfinite(pw, v, e[0], e[1], e[2], e[3]);
            o[d] = f32x4_t{e[0], e[1], e[2], e[3]};
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }

    // the waves' join: their outputs through LDS (each wave over its own V rows)
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    l += poison;
    const bool seen = begin < steps && pos >= begin * kStepKeys;
    if (g == 0) wave_ml[wave][c] = make_float2(seen || l != l ? raw : kUnseen, l);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    float* const wo = reinterpret_cast<float*>(vl);
    static_assert(kStepRows * kDim * sizeof(float) <= kStepKeys * kDim * sizeof(uint16_t), "a wave's outputs fit its V rows");
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4_t*>(&wo[c * kDim + 4 * ((4 * d + g) ^ c)]) = o[d];  // (16-byte piece p at p ^ c)
    lds_barrier();
    const int jr = tid >> 4, ch = 8 * (tid & 15);
    if (base + jr < rows.y * a.group) {
      float top = kUnseen;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_ml[w][jr].x);
      const float st = scaled_max(top, a.scale);
      float sum = 0.0f, acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float2 ml = wave_ml[w][jr];
        if (ml.x == kUnseen) continue;
        const float f = exp2_between(ml.x, top, scaled_max(ml.x, a.scale), st, a.scale);
        sum = fmaf(f, ml.y, sum);
        const float* src = reinterpret_cast<const float*>(lds[w]) + jr * kDim;
        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(src + 4 * (ch / 4 ^ jr)), hi = *reinterpret_cast<const f32x4_t*>(src + 4 * ((ch / 4 + 1) ^ jr));
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = fmaf(f, i < 4 ? lo[i & 3] : hi[i & 3], acc[i]);
      }
      const int tok = (base + jr) / a.group, oh = head * a.group + base + jr - tok * a.group;
      const int64_t orow = static_cast<int64_t>(rows.x + tok) * a.heads + oh;
      if (ranges > 1) {
        const int64_t part = (static_cast<int64_t>(head) * a.slots + w.slot + w.range) * kStepRows + jr;
        float* op = a.part_o + part * kDim + ch;
        if (top != kUnseen) {
          *reinterpret_cast<float4*>(op) = make_float4(acc[0], acc[1], acc[2], acc[3]);
          *reinterpret_cast<float4*>(op + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
        }
        if (ch == 0) a.part_ml[part] = make_float2(top, sum);
      } else {
        const float inv = top != kUnseen ? 1.0f / sum : 0.0f;
        const uint2 x = pair4(acc, inv), y = pair4(acc + 4, inv);
        *reinterpret_cast<uint4*>(a.o + orow * kDim + ch) = make_uint4(x.x, x.y, y.x, y.y);
      }
    }
    lds_barrier();  // (the next rows' V goes where these outputs lie)
  }
}

// Joins the key ranges of step_kernel's divided items: a wave takes a row of one KV head, 2 channels a lane.  Range r's maximum and sum come to lane r in one load, and the ranges' rows are loaded eight at a time, so that a
// join costs two or three memory latencies (one load after another: 13 us for one row of 16 ranges).
__global__ __launch_bounds__(kThreads) void join_kernel(PagedArgs a) {
  const int head = static_cast<int>(blockIdx.x) % a.kv, nth = static_cast<int>(blockIdx.x) / a.kv;
  if (nth >= *a.divided) return;
  const Divided d = a.list[nth];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t slot = static_cast<int64_t>(head) * a.slots + d.slot;
  const int r = static_cast<int>(blockIdx.y) * kWaves + wave;
  if (r >= d.rows * a.group) return;
  const int token = r / a.group;
  const int64_t out = (static_cast<int64_t>(d.first + token) * a.heads + head * a.group + r - token * a.group) * kDim + 2 * lane;
  const float2 ml = lane < d.ranges ? a.part_ml[(slot + lane) * kStepRows + r] : make_float2(kUnseen, 0.0f);
  const float* const part = a.part_o + (slot * kStepRows + r) * kDim + 2 * lane;
  const float top = wave_max(ml.x);
  const bool seen = ml.x != kUnseen;
  const float w = seen ? exp2_between(ml.x, top, scaled_max(ml.x, a.scale), scaled_max(top, a.scale), a.scale) : 0.0f;
  const float l = wave_sum(seen ? w * ml.y : (ml.y != ml.y ? ml.y : 0.0f));
  const unsigned long long parts = __builtin_amdgcn_ballot_w64(seen);
  float o0 = 0.0f, o1 = 0.0f;
  for (int base = 0; base < d.ranges; base += 8) {
    float2 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      v[k] = (parts >> (base + k)) & 1 ? *reinterpret_cast<const float2*>(part + static_cast<int64_t>(base + k) * kStepRows * kDim)
                                       : make_float2(0.0f, 0.0f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = row_lane(w, base + k);
      o0 = fmaf(f, v[k].x, o0);
      o1 = fmaf(f, v[k].y, o1);
    }
  }
  const float inv = top != kUnseen || l != l ? 1.0f / l : 0.0f;
  *reinterpret_cast<uint32_t*>(a.o + out) = attn_bf16_pair(o0 * inv, o1 * inv);
}

// Joins chunk_kernel's parts of the item that a slice opens: its slots are 2 i + 1, 2 (i + 1), 2 (i + 2) ..  A wave takes the
// 32 queries of a wave of that kernel and 16 channels, in its registers' order, so that all loads are of whole kilobytes; eight
// parts' at a time, under a running maximum.
__global__ __launch_bounds__(kThreads) void join_slices_kernel(PagedArgs a) {
  const int head = static_cast<int>(blockIdx.x) % a.kv, index = static_cast<int>(blockIdx.x) / a.kv;
  const Divided item = a.list[index];
  const int lane = threadIdx.x & 63, h = lane >> 5, block = blockIdx.y >> 1;
  const int piece = (blockIdx.y & 1) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // of 16 channels
  const int r = item.item * kChunkRows + 32 * block + (lane & 31);
  if (item.item * kChunkRows + 32 * block >= item.rows * a.group || item.ranges == 0) return;
  constexpr int kAhead = 8;
  float top = kUnseen, l = 0.0f, bad = 0.0f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.0f;
  for (int base = 0; base < item.ranges; base += kAhead) {
    float2 ml[kAhead];
    f32x4_t v[kAhead][2];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      ml[k] = make_float2(kUnseen, 0.0f);
      v[k][0] = v[k][1] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
      const int range = base + k;
      if (range >= item.ranges) continue;
      const int64_t part = static_cast<int64_t>(head) * a.slots + item.slot + (range > 0 ? 2 * range - 1 : 0);
      ml[k] = a.part_ml[part * kChunkRows + 32 * block + (lane & 31)];
      const float* const p = a.part_o + (((part * kChunkWaves + block) * 16 + 2 * piece) * kWave + lane) * 4;
#pragma unroll
      for (int g = 0; g < 2; ++g) v[k][g] = *reinterpret_cast<const f32x4_t*>(p + g * kWave * 4);
    }
    float most = top;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) most = fmaxf(most, ml[k].x);
    const float sm = scaled_max(most, a.scale);
    const float keep = top == kUnseen ? 0.0f : exp2_between(top, most, scaled_max(top, a.scale), sm, a.scale);
    l *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= keep;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const bool seen = ml[k].x != kUnseen;
      if (!seen && ml[k].y != ml[k].y) bad = ml[k].y;
      const float w = seen ? exp2_between(ml[k].x, most, scaled_max(ml[k].x, a.scale), sm, a.scale) : 0.0f;
      l = seen ? fmaf(w, ml[k].y, l) : l;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = seen ? fmaf(w, v[k][i >> 2][i & 3], o[i]) : o[i];
    }
    top = most;
  }
  if (r >= item.rows * a.group) return;
  l += bad;
  const float inv = top != kUnseen || l != l ? 1.0f / l : 0.0f;
  const int token = r / a.group;
  uint16_t* const out = a.o + (static_cast<int64_t>(item.first + token) * a.heads + head * a.group + r - token * a.group) * kDim + 16 * piece + 4 * h;
#pragma unroll
  for (int g = 0; g < 2; ++g) *reinterpret_cast<uint2*>(out + 8 * g) = pair4(o + 4 * g, inv);
}

// How a call is launched: which kernel, and the room for divided items.
struct Launch {
  bool step;
  int aim, ranges, slots, items;
  int64_t groups;  // workgroups a KV head, at most
  size_t list_at, ml_at, o_at, bytes;
};

// (max_q: 1 without q_starts)
Launch plan(int64_t n, int64_t seqs, int kv, int group, int64_t max_q, int64_t max_kv) {
  Launch p{};
  // Up to 16 queries of a KV head are one pass over its keys in step_kernel.  More would be several there, by one workgroup for
  // which the keys are not divided (32 heads on one KV head, a token over 8192, 32768 tokens: 147, 558 us there and 26.8, 38 in
  // chunk_kernel; of 32 sequences of 4096 78 and 37), so they go there only as single tokens over keys that are one range anyway
  // (a token over 512: 15.5 there, 19.7 in chunk_kernel, of 1024 sequences 80 and 104, 4096 of 100 93 and 343), in up to four
  // passes (128 heads on one, 64 sequences of 500: 61 there, 29).
  p.step = max_q * group <= kStepRows || (max_q == 1 && group <= 4 * kStepRows && max_kv <= kStepWhole * kStepKeys);
  const int rows = p.step ? kStepRows : kChunkRows, unit = p.step ? kStepKeys : kKeys;
  const int64_t items = p.step ? seqs : (n * group + kChunkRows - 1) / kChunkRows + (seqs > 1 ? seqs : 0);
  const int64_t steps = (max_kv + unit - 1) / unit;
  p.groups = items;
  p.ranges = 1;
  if (p.step) {
    // nothing is divided where the longest sequence is one range, or the sequences alone make as many workgroups as ranges would
    if (steps <= kStepWhole || items * kv >= kStepAim) return p;
    p.aim = kStepAim;
    p.ranges = static_cast<int>(std::min<int64_t>(kMaxRanges, (steps + kStepLeast - 1) / kStepLeast));
    p.slots = static_cast<int>(std::min<int64_t>(2 * (p.aim / kv) + 8, items * p.ranges));
    p.items = static_cast<int>(std::min<int64_t>(p.aim / kv + 8, items));
    p.groups += p.slots;
  } else {
    // One sequence's items are divided where they are fewer than the CUs.  Several sequences' always, as their lengths are not
    // known here: whole items would be 5% faster where there are many of about one length (12 sequences of up to 2000 tokens
    // over 8000, 8 query heads a KV head, 4 of these: 487 and 514 us), and as long as the longest where one is long.
    const int64_t slices = std::min<int64_t>(kChunkAim / kv, (items * (steps + static_cast<int>(kApart)) + kLeastSteps - 1) / kLeastSteps);
    if (slices < 2 || steps <= kLeastSteps || (seqs == 1 && items * kv >= kChunkAim)) return p;
    p.aim = p.items = static_cast<int>(slices);
    p.groups = p.aim;
    p.slots = 2 * p.aim;
  }
  p.list_at = 16;
  p.ml_at = (p.list_at + p.items * sizeof(Divided) + 15) / 16 * 16;
  p.o_at = p.ml_at + static_cast<size_t>(kv) * p.slots * rows * sizeof(float2);
  p.bytes = p.o_at + static_cast<size_t>(kv) * p.slots * rows * kDim * sizeof(float);
  return p;
}

}  // namespace
}  // namespace fl

extern "C" size_t fl_paged_attention_workspace(int32_t rows, int32_t seqs, int32_t heads, int32_t kv_heads, int32_t max_q,
                                               int32_t max_kv) {
  using namespace fl;
  if (rows <= 0 || seqs <= 0 || kv_heads <= 0 || heads < kv_heads || heads % kv_heads || max_q <= 0 || max_kv <= 0) return 0;
  // (with or without q_starts: what both may take)
  const size_t a = plan(rows, seqs, kv_heads, heads / kv_heads, max_q, max_kv).bytes;
  return rows == seqs ? std::max(a, plan(rows, seqs, kv_heads, heads / kv_heads, 1, max_kv).bytes) : a;
}

extern "C" int32_t fl_paged_attention(const uint16_t* q, int64_t q_row_stride, const uint16_t* k_pages, const uint16_t* v_pages,
                                      uint16_t* out, const int32_t* page_table, const int32_t* kv_lens, const int32_t* q_starts,
                                      int32_t rows, int32_t seqs, int32_t heads, int32_t kv_heads, int32_t table_width,
                                      int32_t pages, int32_t page_size, int32_t max_q, int32_t max_kv, float scaling,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(q && k_pages && v_pages && out && page_table && kv_lens, "fl_paged_attention: null pointer");
  FL_REQUIRE(rows >= 0 && seqs >= 0 && table_width > 0 && pages > 0, "fl_paged_attention: bad sizes");
  FL_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "fl_paged_attention: heads must be a multiple of the KV heads");
  FL_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
             "fl_paged_attention: the page size must be a power of two from 16 to 1024");
  FL_REQUIRE(q_row_stride >= static_cast<int64_t>(heads) * kDim && q_row_stride % 8 == 0, "fl_paged_attention: bad row stride");
  FL_REQUIRE(q_starts != nullptr || rows == seqs, "fl_paged_attention: one row a sequence without q_starts");
  FL_REQUIRE(max_q > 0 && max_kv > 0, "fl_paged_attention: max_q and max_kv must be positive");
  FL_REQUIRE(scaling > 0.0f && std::isfinite(scaling * kLog2e), "fl_paged_attention: scaling must be positive and finite");
  FL_REQUIRE(static_cast<int64_t>(table_width) * page_size <= 0x7FFFFFFF - 4096, "fl_paged_attention: a sequence's pages hold too many tokens");
  const int group = heads / kv_heads;
  FL_REQUIRE(static_cast<int64_t>(rows) * group <= 0x7FFFFFFF - 4096, "fl_paged_attention: too many rows");
  for (const void* p : {static_cast<const void*>(q), static_cast<const void*>(k_pages), static_cast<const void*>(v_pages),
                        static_cast<const void*>(out)})
    FL_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "fl_paged_attention: every tensor must be 16-byte aligned");
  if (rows == 0) return FL_OK;
  FL_REQUIRE(seqs > 0, "fl_paged_attention: rows without a sequence");
  // (in q's place is fine: who writes a row's head has read it, or runs after all who do)
  const int64_t cols = static_cast<int64_t>(heads) * kDim, pool = static_cast<int64_t>(pages) * kv_heads * page_size * kDim;
  FL_REQUIRE((out == q && q_row_stride == cols) || apart(out, cols, cols, 2, q, q_row_stride, cols, 2, rows),
             "fl_paged_attention: out lies on other values of q");
  for (const uint16_t* p : {k_pages, v_pages})
    FL_REQUIRE(apart(out, rows * cols, rows * cols, 2, p, pool, pool, 2, 1), "fl_paged_attention: out lies on the pages");
  Launch p = plan(rows, seqs, kv_heads, group, q_starts ? max_q : 1, max_kv);
  if (workspace == nullptr || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 || workspace_bytes < p.bytes) {
    p = plan(rows, seqs, kv_heads, group, q_starts ? max_q : 1, 1);  // (no room for divided items: none is)
  }
  FL_REQUIRE(p.groups * kv_heads <= 0x7FFFFFFF / kChunkThreads, "fl_paged_attention: grid too large");
  uint8_t* const ws = static_cast<uint8_t*>(workspace);
  const PagedArgs a{q, q_row_stride, k_pages, v_pages, out, page_table, kv_lens, q_starts, rows, seqs, heads, kv_heads, group,
                    table_width, pages, __builtin_ctz(static_cast<unsigned>(page_size)), scaling * kLog2e,
                    p.aim, p.ranges, p.slots, p.items, reinterpret_cast<int32_t*>(ws), reinterpret_cast<Divided*>(ws + p.list_at),
                    reinterpret_cast<float2*>(ws + p.ml_at), reinterpret_cast<float*>(ws + p.o_at)};
  const dim3 grid(static_cast<unsigned>(p.groups * kv_heads));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p.step)
    hipLaunchKernelGGL(step_kernel, grid, dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL(chunk_kernel, grid, dim3(kChunkThreads), 0, st, a);
  FL_LAUNCH_CHECK("fl_paged_attention");
  if (p.aim == 0) return FL_OK;
  const unsigned items = static_cast<unsigned>(p.items * kv_heads);
  if (p.step)
    hipLaunchKernelGGL(join_kernel, dim3(items, kStepRows / kWaves), dim3(kThreads), 0, st, a);
  else
    hipLaunchKernelGGL(join_slices_kernel, dim3(items, 2 * kChunkWaves), dim3(kThreads), 0, st, a);
  FL_LAUNCH_CHECK("fl_paged_attention(join)");
  return FL_OK;
}
