// Tokens into K/V pages, and the pages of beams that take over each other's state.
//
//  * fl_paged_append -- rotary embedding of q and k rows and the placement of k and v in pages
//    [pages, KV heads, page, 128] at the positions that the sequences' lengths imply.
//  * fl_paged_reorder -- new page tables for the beams of each sequence, and copies of the filled rows of
//    a page that several children of one beam go on filling.
//
// Both move bytes: 16 of them a lane and access.  3014 rows of 16 + 2 x 16 heads, 50 MB, 10 us (5.0 TB/s, what a copy reaches;
// eight rows 3.3 us, a launch and two dependent reads); pages of 8 sequences in 8 beams, 503 MB, 88-94 us (5.4 TB/s: a parent's
// page that several children copy is read from memory once).
#include <algorithm>

#include "fl_common.h"

namespace fl {
namespace {

struct AppendArgs {
  const uint16_t* src[3];  // q [n, heads * 128], k, v [n, kv * 128]
  int64_t src_row[3];
  uint16_t* q_out;  // row stride q_out_row (may be q in place)
  int64_t q_out_row;
  uint16_t* pages[2];  // k, v
  const void* cos;     // [positions, 128] bf16 or f32; null: no rotation, q is left alone
  const void* sin;
  const int32_t* table;   // [seqs, width]
  const int32_t* lens;    // [seqs], the call's rows among them
  const int32_t* starts;  // [seqs + 1], or null: row s is sequence s's
  int n, seqs, heads, kv, width, page_count, page_log2, positions, units;
};

template <bool F32>
__device__ __forceinline__ void load_table(const void* t, int64_t at, float* f) {
  if (F32) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(t) + at);
    const float4 a = p[0], b = p[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(t) + at), f);
  }
}

// A wave takes one row and eight of its heads (q's, then k's, then v's): a lane 8 channels and their
// rotary partners, 64 further on.  The row's sequence is found by a vote over 64 sequences at a time.  The products and
// their sum are fp32, rounded to bf16 once.
template <bool F32>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= static_cast<int64_t>(a.n) * a.units) return;
  const int row = static_cast<int>(item / a.units), unit = static_cast<int>(item - static_cast<int64_t>(row) * a.units);
  int seq = row, pos = 0;
  if (a.starts == nullptr) {
    pos = a.lens[row] - 1;
  } else {
    seq = 0;  // sequences that end at or before the row
    for (int base = 0; base < a.seqs; base += kWave) {
      const int s = base + lane;
      const int ends = __builtin_popcountll(__builtin_amdgcn_ballot_w64(s < a.seqs && a.starts[s + 1] <= row));
      seq += ends;
      if (ends < kWave) break;
    }
    if (seq < a.seqs) pos = a.lens[seq] - (a.starts[seq + 1] - row);
  }
  const int which_head = unit * 8 + (lane >> 3), c = (lane & 7) * 8;
  if (which_head >= a.heads + 2 * a.kv) return;
  const int which = which_head < a.heads ? 0 : (which_head < a.heads + a.kv ? 1 : 2);
  const int head = which_head - (which == 0 ? 0 : (which == 1 ? a.heads : a.heads + a.kv));
  if (which == 0 && a.cos == nullptr) return;
  const uint16_t* src = (which == 0 ? a.src[0] + row * a.src_row[0] : (which == 1 ? a.src[1] + row * a.src_row[1] : a.src[2] + row * a.src_row[2])) +
                        head * kDim + c;
  uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + 64);
  const bool mine = seq < a.seqs;  // (rows behind the last sequence: q as it is)
  const int slot = mine && pos >= 0 && (pos >> a.page_log2) < a.width ? a.table[static_cast<int64_t>(seq) * a.width + (pos >> a.page_log2)] : -1;
  const bool placed = static_cast<unsigned>(slot) < static_cast<unsigned>(a.page_count) && (a.cos == nullptr || pos < a.positions);
  if (which < 2 && a.cos != nullptr && placed) {
    float x[8], y[8], cs[8], sn[8], u[8];
    unpack_bf16x8(lo, x);
    unpack_bf16x8(hi, y);
    const int64_t at = static_cast<int64_t>(pos) * kDim + c;
    load_table<F32>(a.cos, at, cs);
    load_table<F32>(a.sin, at, sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = fmaf(x[e], cs[e], -y[e] * sn[e]);
    lo = pack_bf16x8(u);
    load_table<F32>(a.cos, at + 64, cs);
    load_table<F32>(a.sin, at + 64, sn);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = fmaf(y[e], cs[e], x[e] * sn[e]);
    hi = pack_bf16x8(u);
  }
  uint16_t* dst;
  if (which == 0) {
    if (mine && !placed) lo = hi = make_uint4(0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u, 0x7FC07FC0u);
    dst = a.q_out + row * a.q_out_row + head * kDim + c;
  } else {
    if (!placed) return;
    dst = (which == 1 ? a.pages[0] : a.pages[1]) +
          ((((static_cast<int64_t>(slot) * a.kv + head) << a.page_log2) + (pos & ((1 << a.page_log2) - 1))) << 7) + c;
  }
  *reinterpret_cast<uint4*>(dst) = lo;
  *reinterpret_cast<uint4*>(dst + 64) = hi;
}

struct ReorderArgs {
  uint16_t* pages[2];  // k, v [layers, page_count, kv, page, 128]
  const int32_t* table;  // [seqs * beams, width]
  int32_t* table_out;
  const int32_t* lens;     // [seqs * beams]
  const int32_t* parents;  // [seqs, beams]
  int seqs, beams, layers, width, page_count, kv, page_log2;
};

constexpr int kMaxBeams = 64;

// blockIdx.y: a beam; its table row, and the filled rows of its last page where an earlier child of the same
// parent has the parent's page: the children without one take the pages of beams that have no child, in order.
// blockIdx.x: layer, and K or V; blockIdx.z: a share of its 16-byte pieces.
__global__ __launch_bounds__(256) void reorder_kernel(ReorderArgs a) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int seq = blockIdx.y / a.beams, beam = blockIdx.y - seq * a.beams;
  const int32_t* const old = a.table + static_cast<int64_t>(seq) * a.beams * a.width;
  const int len = max(a.lens[seq * a.beams], 0);
  const int tail = len >> a.page_log2, filled = len & ((1 << a.page_log2) - 1);
  // the plan, by every wave: beams in lanes
  int parent = lane < a.beams ? a.parents[seq * a.beams + lane] : -1;
  if (parent < 0 || parent >= a.beams) parent = -1;
  unsigned long long kept = 0ull, further = 0ull;  // beams with a child; children that need a page
  for (int i = 0; i < a.beams; ++i) {
    const int p = __builtin_amdgcn_readlane(parent, i);
    if (p < 0) continue;
    if ((kept >> p) & 1)
      further |= 1ull << i;
    else
      kept |= 1ull << p;
  }
  const int from = __builtin_amdgcn_readlane(parent, beam);
  int take = from;  // the beam whose last page this one goes on filling
  if (from >= 0 && ((further >> beam) & 1)) {
    const int nth = __builtin_popcountll(further & ((1ull << beam) - 1));
    unsigned long long open = ~kept;
    for (int i = 0; i < nth; ++i) open &= open - 1;
    take = __builtin_ctzll(open);
  }
  if (blockIdx.x == 0 && blockIdx.z == 0) {
    int32_t* const out = a.table_out + (static_cast<int64_t>(seq) * a.beams + beam) * a.width;
    for (int j = tid; j < a.width; j += 256) {
      const int whose = from < 0 ? -1 : (j < tail ? from : (j == tail && filled ? take : beam));
      out[j] = whose < 0 ? -1 : old[static_cast<int64_t>(whose) * a.width + j];
    }
  }
  if (filled == 0 || tail >= a.width || take == from) return;
  const int src_page = old[static_cast<int64_t>(from) * a.width + tail], dst_page = old[static_cast<int64_t>(take) * a.width + tail];
  if (static_cast<unsigned>(src_page) >= static_cast<unsigned>(a.page_count) ||
      static_cast<unsigned>(dst_page) >= static_cast<unsigned>(a.page_count) || src_page == dst_page)
    return;
  const int64_t layer = blockIdx.x >> 1;
  uint16_t* const base = blockIdx.x & 1 ? a.pages[1] : a.pages[0];
  const int64_t page_elems = static_cast<int64_t>(a.kv) << (a.page_log2 + 7);
  const uint16_t* const src = base + (layer * a.page_count + src_page) * page_elems;
  uint16_t* const dst = base + (layer * a.page_count + dst_page) * page_elems;
  const int per_head = filled * (kDim / 8);
  for (int i = blockIdx.z * 256 + tid; i < per_head * a.kv; i += 256 * gridDim.z) {
    const int head = i / per_head;
    const int64_t at = (static_cast<int64_t>(head) << (a.page_log2 + 7)) + (i - head * per_head) * 8;
    *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(src + at);
  }
}

bool paged_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool paged_size(int32_t page_size) { return page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0; }

}  // namespace
}  // namespace fl

extern "C" int32_t fl_paged_append(const uint16_t* q, int64_t q_row_stride, const uint16_t* k, int64_t k_row_stride, const uint16_t* v,
                                   int64_t v_row_stride, uint16_t* q_out, int64_t q_out_row_stride, const void* rope_cos,
                                   const void* rope_sin, int32_t rope_is_f32, int32_t rope_positions, uint16_t* k_pages,
                                   uint16_t* v_pages, const int32_t* page_table, const int32_t* kv_lens, const int32_t* q_starts,
                                   int32_t rows, int32_t seqs, int32_t heads, int32_t kv_heads, int32_t table_width, int32_t pages,
                                   int32_t page_size, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(k && v && k_pages && v_pages && page_table && kv_lens, "fl_paged_append: null pointer");
  FL_REQUIRE((rope_cos == nullptr) == (rope_sin == nullptr), "fl_paged_append: one rope table without the other");
  const bool turn = rope_cos != nullptr;
  FL_REQUIRE(!turn || (q && q_out && rope_positions > 0), "fl_paged_append: null q or empty rope tables");
  FL_REQUIRE(rows >= 0 && seqs >= 0 && table_width > 0 && pages > 0, "fl_paged_append: bad sizes");
  FL_REQUIRE(kv_heads > 0 && heads > 0 && heads <= 65536 && kv_heads <= 65536, "fl_paged_append: bad head counts");
  FL_REQUIRE(paged_size(page_size), "fl_paged_append: the page size must be a power of two from 16 to 1024");
  FL_REQUIRE(q_starts != nullptr || rows == seqs, "fl_paged_append: one row a sequence without q_starts");
  FL_REQUIRE(static_cast<int64_t>(table_width) * page_size <= 0x7FFFFFFF, "fl_paged_append: a sequence's pages hold too many tokens");
  const int64_t kv_cols = static_cast<int64_t>(kv_heads) * kDim, q_cols = static_cast<int64_t>(heads) * kDim;
  FL_REQUIRE(k_row_stride >= kv_cols && v_row_stride >= kv_cols && k_row_stride % 8 == 0 && v_row_stride % 8 == 0,
             "fl_paged_append: bad row strides");
  FL_REQUIRE(!turn || (q_row_stride >= q_cols && q_out_row_stride >= q_cols && q_row_stride % 8 == 0 && q_out_row_stride % 8 == 0),
             "fl_paged_append: bad row strides");
  for (const void* p : {static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(k_pages),
                        static_cast<const void*>(v_pages)})
    FL_REQUIRE(paged_aligned(p), "fl_paged_append: every tensor must be 16-byte aligned");
  FL_REQUIRE(!turn || (paged_aligned(q) && paged_aligned(q_out) && paged_aligned(rope_cos) && paged_aligned(rope_sin)),
             "fl_paged_append: every tensor must be 16-byte aligned");
  if (rows == 0) return FL_OK;
  FL_REQUIRE(seqs > 0, "fl_paged_append: rows without a sequence");
  // (a wave writes its heads of a row while others read theirs)
  const auto outside = [&](const uint16_t* x, int64_t stride, int64_t cols, const void* block, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(x), from = reinterpret_cast<uintptr_t>(block);
    return at + 2 * ((rows - 1) * stride + cols) <= from || from + bytes <= at;
  };
  const int64_t pool = 2 * static_cast<int64_t>(pages) * kv_heads * page_size * kDim;
  for (const uint16_t* p : {k_pages, v_pages})
    FL_REQUIRE(outside(k, k_row_stride, kv_cols, p, pool) && outside(v, v_row_stride, kv_cols, p, pool) &&
                   (!turn || (outside(q, q_row_stride, q_cols, p, pool) && outside(q_out, q_out_row_stride, q_cols, p, pool))),
               "fl_paged_append: rows lie on the pages");
  if (turn) {
    FL_REQUIRE((q_out == q && q_out_row_stride == q_row_stride) || apart(q_out, q_out_row_stride, q_cols, 2, q, q_row_stride, q_cols, 2, rows),
               "fl_paged_append: q_out lies on other values of q");
    FL_REQUIRE(apart(q_out, q_out_row_stride, q_cols, 2, k, k_row_stride, kv_cols, 2, rows) &&
                   apart(q_out, q_out_row_stride, q_cols, 2, v, v_row_stride, kv_cols, 2, rows),
               "fl_paged_append: q_out lies on k or v");
    const int64_t table = static_cast<int64_t>(rope_positions) * kDim * (rope_is_f32 ? 4 : 2);
    FL_REQUIRE(outside(q_out, q_out_row_stride, q_cols, rope_cos, table) && outside(q_out, q_out_row_stride, q_cols, rope_sin, table),
               "fl_paged_append: q_out lies on a rope table");
  }
  const int units = (heads + 2 * kv_heads + 7) / 8;
  const int64_t blocks = (static_cast<int64_t>(rows) * units + 3) / 4;
  FL_REQUIRE(blocks <= 0xFFFFFFFFll / 256, "fl_paged_append: grid too large");
  const AppendArgs a{{q, k, v}, {q_row_stride, k_row_stride, v_row_stride}, q_out, q_out_row_stride, {k_pages, v_pages}, rope_cos,
                     rope_sin, page_table, kv_lens, q_starts, rows, seqs, heads, kv_heads, table_width, pages,
                     __builtin_ctz(static_cast<unsigned>(page_size)), rope_positions, units};
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  if (rope_is_f32)
    hipLaunchKernelGGL(append_kernel<true>, grid, block, 0, static_cast<hipStream_t>(stream), a);
  else
    hipLaunchKernelGGL(append_kernel<false>, grid, block, 0, static_cast<hipStream_t>(stream), a);
  FL_LAUNCH_CHECK("fl_paged_append");
  return FL_OK;
}

extern "C" int32_t fl_paged_reorder(uint16_t* k_pages, uint16_t* v_pages, const int32_t* page_table, int32_t* table_out,
                                    const int32_t* kv_lens, const int32_t* parents, int32_t seqs, int32_t beams, int32_t layers,
                                    int32_t table_width, int32_t pages, int32_t kv_heads, int32_t page_size, void* stream) {
  using namespace fl;
  clear_error();
  FL_REQUIRE(k_pages && v_pages && page_table && table_out && kv_lens && parents, "fl_paged_reorder: null pointer");
  FL_REQUIRE(page_table != table_out, "fl_paged_reorder: the new table must not be the old one");
  FL_REQUIRE(seqs >= 0 && layers > 0 && layers <= 65536 && table_width > 0 && pages > 0 && kv_heads > 0 && kv_heads <= 65536,
             "fl_paged_reorder: bad sizes");
  FL_REQUIRE(beams > 0 && beams <= kMaxBeams, "fl_paged_reorder: 1 to 64 beams");
  FL_REQUIRE(paged_size(page_size), "fl_paged_reorder: the page size must be a power of two from 16 to 1024");
  FL_REQUIRE(paged_aligned(k_pages) && paged_aligned(v_pages), "fl_paged_reorder: pages must be 16-byte aligned");
  FL_REQUIRE(static_cast<int64_t>(kv_heads) * page_size * (kDim / 8) <= 0x7FFFFFFF - 256, "fl_paged_reorder: pages too large");
  FL_REQUIRE(static_cast<int64_t>(seqs) * beams <= 65535, "fl_paged_reorder: too many beams");
  if (seqs == 0) return FL_OK;
  const ReorderArgs a{{k_pages, v_pages}, page_table, table_out, kv_lens, parents, seqs, beams, layers, table_width, pages, kv_heads,
                      __builtin_ctz(static_cast<unsigned>(page_size))};
  // a share of 16 KB and more of a full page, so that few copies fill the chip (two of 32 rows x 16 heads in 16 layers: 9.6 us
  // with one workgroup a page, 5.5 with eight)
  const int64_t page_bytes = static_cast<int64_t>(kv_heads) * page_size * kDim * 2;
  const int shares = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(8, page_bytes / 16384)));
  hipLaunchKernelGGL(reorder_kernel, dim3(2 * layers, seqs * beams, shares), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  FL_LAUNCH_CHECK("fl_paged_reorder");
  return FL_OK;
}
