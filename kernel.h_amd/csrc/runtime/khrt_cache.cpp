// The sequence-cache operators behind the C-ABI (khrt.h, group 8): the checks
// of what the host can see, the launch geometry, and the kernels' parameters.
#include "kernelh/khrt_internal.hpp"
#include "kh_paged.h"
#include "kh_tiles.h"

#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <string>
#include <utility>

namespace {

int bad(const char *op, const std::string &what) { return khrt::fail(KHRT_E_INVALID, std::string(op) + ": " + what); }

// Nothing thrown below leaves a C entry point.
template <class Call>
int guarded(const char *op, Call &&call) {
  try {
    return call();
  } catch (const std::exception &e) {
    try {
      return bad(op, e.what());
    } catch (...) {
      return KHRT_E_INVALID;
    }
  } catch (...) {
    return KHRT_E_INVALID;
  }
}

constexpr int64_t kMaxPageSize = int64_t(1) << 20;
constexpr int64_t kMaxStride = int64_t(1) << 40;   // of tables and weights
constexpr int64_t kMaxSpan = int64_t(1) << 59;     // elements that the strides of q, k, v and out cover
constexpr int64_t kMaxCacheStride = int64_t(1) << 32;  // bytes, exclusive (kh_paged.h)
constexpr int64_t kMaxRows = int64_t(1) << 30;     // tokens x heads
constexpr int64_t kMaxPairs = int64_t(1) << 20;    // sequences x kv heads
constexpr int64_t kCapacity = (int64_t(1) << 31) - (int64_t(1) << 16);  // entries of a sequence

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int element_bytes(int32_t dtype) { return dtype == KHRT_F32 ? 4 : 2; }

bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A stride over `extent` rows: not negative, 16 bytes' worth, and for rows that
// are written (least > 0) no shorter than the row where there is a next one.
bool stride_ok(int64_t stride, int64_t extent, int element, int64_t least) {
  if (extent <= 1) return stride >= 0 && stride <= kMaxSpan;
  return stride >= least && stride <= kMaxSpan / extent && stride % (16 / element) == 0;
}

// Whether rows of `row` elements at i a.stride + j b.stride, i < a.extent,
// j < b.extent, lie apart. One of the extents is below 2^10 wherever this is asked
// of strides that do not nest (pairs of sequence and kv head).
struct Steps {
  int64_t stride, extent;
};

bool nest(Steps inner, Steps outer, int64_t row) {
  if (inner.extent <= 1) return outer.extent <= 1 || outer.stride >= row;
  return inner.stride >= row && (outer.extent <= 1 || outer.stride >= (inner.extent - 1) * inner.stride + row);
}

bool rows_apart(Steps a, Steps b, int64_t row) {
  if (nest(a, b, row) || nest(b, a, row)) return true;
  if (a.extent > b.extent) std::swap(a, b);
  if (a.extent <= 1 || b.stride < row || a.stride < row) return false;
  // Two rows differ by i steps of a and, in the other direction, j of b.
  for (int64_t i = 1; i < a.extent; ++i) {
    const int64_t off = i * a.stride, j = off / b.stride;
    if (j < b.extent && off - j * b.stride < row) return false;
    if (j + 1 < b.extent && (j + 1) * b.stride - off < row) return false;
  }
  return true;
}

// The fields that describe rows, of a cache that may have none.
int check_rows(const char *op, const kh_paged_cache &c) {
  if (c.dtype != KHRT_F32 && c.dtype != KHRT_F16 && c.dtype != KHRT_BF16)
    return bad(op, "dtype must be KHRT_F32, KHRT_F16 or KHRT_BF16 (got " + std::to_string(c.dtype) + ")");
  if (c.head_dim <= 0 || c.head_dim > 256 || c.head_dim % 8 != 0)
    return bad(op, "head_dim must be a multiple of 8 up to 256 (got " + std::to_string(c.head_dim) + ")");
  if (c.kv_heads <= 0 || c.kv_heads > 65535) return bad(op, "kv_heads must be in [1, 65535]");
  return 0;
}

int check_cache(const char *op, const kh_paged_cache &c, bool written) {
  if (int rc = check_rows(op, c)) return rc;
  if (c.k == nullptr || c.v == nullptr) return bad(op, "null cache");
  if (c.pages <= 0 || c.pages > INT32_MAX) return bad(op, "pages must be in [1, 2^31)");
  if (c.page_size <= 0 || c.page_size > kMaxPageSize) return bad(op, "page_size must be in [1, 2^20]");
  const int e = element_bytes(c.dtype);
  const int64_t least = written ? c.head_dim : 0;
  for (const bool is_v : {false, true}) {
    if (!aligned(is_v ? c.v : c.k)) return bad(op, "the cache must be 16-byte aligned");
    for (const int64_t s : {is_v ? c.v_page_stride : c.k_page_stride, is_v ? c.v_slot_stride : c.k_slot_stride,
                            is_v ? c.v_head_stride : c.k_head_stride})
      if (s >= kMaxCacheStride / e) return bad(op, "cache strides must be below 2^32 bytes");
    if (!stride_ok(is_v ? c.v_page_stride : c.k_page_stride, c.pages, e, least) ||
        !stride_ok(is_v ? c.v_slot_stride : c.k_slot_stride, c.page_size, e, least) ||
        !stride_ok(is_v ? c.v_head_stride : c.k_head_stride, c.kv_heads, e, least))
      return bad(op, written ? "cache strides must be multiples of 16 bytes and hold a row"
                             : "cache strides must be multiples of 16 bytes, not negative");
    if (!written) continue;
    // Rows that are written lie apart: whatever the order of pages, slots and heads, each holds the ones inside.
    Steps s[] = {{is_v ? c.v_page_stride : c.k_page_stride, c.pages}, {is_v ? c.v_slot_stride : c.k_slot_stride, c.page_size},
                 {is_v ? c.v_head_stride : c.k_head_stride, c.kv_heads}};
    std::sort(s, s + 3, [](const Steps &a, const Steps &b) { return (a.extent > 1 ? a.stride : 0) < (b.extent > 1 ? b.stride : 0); });
    int64_t inside = c.head_dim;
    for (const Steps &x : s) {
      if (x.extent <= 1) continue;
      if (x.stride < inside) return bad(op, "rows of a cache that is written must not overlap");
      inside += (x.extent - 1) * x.stride;
    }
  }
  return 0;
}

int check_table(const char *op, const kh_page_table &t, const kh_paged_cache &c) {
  if (t.pages == nullptr || t.lens == nullptr) return bad(op, "null page table");
  if (t.seqs <= 0 || t.width <= 0 || t.width > INT32_MAX) return bad(op, "seqs and width must be positive");
  if (t.row_stride < 0 || t.row_stride > kMaxStride) return bad(op, "the table's row stride must not be negative");
  if (t.seqs > kMaxPairs || t.seqs * c.kv_heads > kMaxPairs) return bad(op, "more than 2^20 pairs of sequence and kv head");
  if (t.max_len < 0) return bad(op, "max_len must not be negative");
  return 0;
}

KhCache device_cache(const kh_paged_cache &c) {
  const int e = element_bytes(c.dtype);
  auto bytes = [e](int64_t stride) { return static_cast<uint32_t>(stride * e); };
  return KhCache{static_cast<const char *>(c.k), static_cast<const char *>(c.v), bytes(c.k_page_stride),
                 bytes(c.k_slot_stride), bytes(c.k_head_stride), bytes(c.v_page_stride), bytes(c.v_slot_stride),
                 bytes(c.v_head_stride), static_cast<int32_t>(c.pages), static_cast<int32_t>(c.page_size),
                 static_cast<int32_t>(c.kv_heads), static_cast<int32_t>(c.head_dim),
                 kh_div_by(static_cast<uint32_t>(c.page_size))};
}

int64_t capacity_of(int64_t width, int64_t page_size) { return std::min(width * page_size, kCapacity); }

KhTable device_table(const kh_page_table &t, const kh_paged_cache &c) {
  return KhTable{t.pages, t.lens, t.row_stride, static_cast<int32_t>(t.seqs), static_cast<int32_t>(t.width),
                 static_cast<int32_t>(capacity_of(t.width, c.page_size))};
}

// Rows that follow each other 16 at a time, none longer than their distance,
// and 16 of those distances in 31 bits: pages are walked 16 entries at a time.
bool even_pages(const kh_paged_cache &c) {
  const auto [near, far] = std::minmax(c.k_slot_stride, c.v_slot_stride);
  return c.page_size % 16 == 0 && near >= c.head_dim && far * element_bytes(c.dtype) < 1 << 27;
}

// The longest sequence that a launch is sized for.
int64_t expected_len(const kh_page_table &t, const kh_paged_cache &c) {
  const int64_t all = capacity_of(t.width, c.page_size);
  return t.max_len > 0 ? std::min(t.max_len, all) : all;
}

int check_tokens(const char *op, int64_t tokens, int64_t q_heads, const kh_paged_cache &c) {
  if (tokens <= 0 || q_heads <= 0) return bad(op, "tokens and q_heads must be positive");
  if (tokens > kMaxRows || q_heads > 65535 || tokens * (q_heads + 2 * c.kv_heads) > kMaxRows)
    return bad(op, "more than 2^30 rows");
  return 0;
}

int check_queries(const char *op, const void *q, int64_t q_stride, int64_t tokens, int64_t q_heads, int64_t window,
                  float scale, const kh_paged_cache &c) {
  if (int rc = check_tokens(op, tokens, q_heads, c)) return rc;
  if (q_heads % c.kv_heads != 0) return bad(op, "q_heads must be a multiple of kv_heads");
  if (!aligned(q)) return bad(op, "q must be 16-byte aligned");
  if (!stride_ok(q_stride, tokens, element_bytes(c.dtype), 0)) return bad(op, "q_stride must be a multiple of 16 bytes, not negative");
  if (window < 0 || window > INT32_MAX) return bad(op, "window must be in [0, 2^31)");
  if (!std::isfinite(scale)) return bad(op, "scale must be finite");
  return 0;
}

// Code objects and symbols by element type.
struct Symbol {
  const char *co, *name;
};
#define KH_BY_TYPE(base, suffix)                                                              \
  {                                                                                           \
    {#base "_f32", #base suffix "_f32"}, {#base "_f16", #base suffix "_f16"}, {#base "_bf16", #base suffix "_bf16"} \
  }
const Symbol kRope[3][3] = {KH_BY_TYPE(qk_norm_rope, "_8"), KH_BY_TYPE(qk_norm_rope, "_16"),
                            KH_BY_TYPE(qk_norm_rope, "_32")};
const Symbol kAttention[3][3] = {KH_BY_TYPE(paged_attention, "_64"), KH_BY_TYPE(paged_attention, "_128"),
                                 KH_BY_TYPE(paged_attention, "_256")};
const Symbol kWide[3][3] = {KH_BY_TYPE(paged_attention, "_wide_64"), KH_BY_TYPE(paged_attention, "_wide_128"),
                            KH_BY_TYPE(paged_attention, "_wide_256")};
const Symbol kJoin[3][3] = {KH_BY_TYPE(paged_attention, "_join_64"), KH_BY_TYPE(paged_attention, "_join_128"),
                            KH_BY_TYPE(paged_attention, "_join_256")};
const Symbol kWeights[3][3] = {KH_BY_TYPE(paged_weights, "_64"), KH_BY_TYPE(paged_weights, "_128"),
                               KH_BY_TYPE(paged_weights, "_256")};
const Symbol kWeightsWide[3][3] = {KH_BY_TYPE(paged_weights, "_wide_64"), KH_BY_TYPE(paged_weights, "_wide_128"),
                                   KH_BY_TYPE(paged_weights, "_wide_256")};
const Symbol kChoose = {"paged_evict", "paged_evict_choose"};
const Symbol kMove = {"paged_evict", "paged_evict_move"};

// Which of the kernels' widths holds head_dim: 64, 128 or 256.
int width_of(int64_t head_dim) { return head_dim <= 64 ? 0 : head_dim <= 128 ? 1 : 2; }

template <class Params>
int launch(const Symbol &s, int64_t x, int64_t y, unsigned threads, Params &p, void *stream) {
  void *params[] = {&p};
  return khrt::launch_embedded(s.co, s.name, khrt_dim3{static_cast<unsigned>(x), static_cast<unsigned>(y), 1},
                               khrt_dim3{threads, 1, 1}, stream, params, 1);
}

int check_attention(const char *op, const kh_paged_attention_args &a) {
  if (int rc = check_cache(op, a.cache, false)) return rc;
  if (int rc = check_table(op, a.table, a.cache)) return rc;
  if (!a.q || !a.out || !a.q_starts) return bad(op, "null buffer");
  if (int rc = check_queries(op, a.q, a.q_stride, a.tokens, a.q_heads, a.window, a.scale, a.cache)) return rc;
  if (!aligned(a.out)) return bad(op, "out must be 16-byte aligned");
  if (!stride_ok(a.out_stride, a.tokens, element_bytes(a.cache.dtype), a.q_heads * a.cache.head_dim))
    return bad(op, "out_stride must be a multiple of 16 bytes and hold a token");
  if (a.out == a.q) return bad(op, "out must not be q");
  if (a.max_new < 0) return bad(op, "max_new must not be negative");
  return 0;
}

// log2(e) times the scale, finite as that is: a score of 0 stays one.
float in_powers_of_two(float scale) {
  constexpr float most = std::numeric_limits<float>::max();
  return std::clamp(scale * 1.44269504088896340736f, -most, most);
}

// How a launch of paged_attention spreads over the chip (kh_paged.h).
struct AttentionPlan {
  int64_t groups;              // workgroups of sequences of few rows
  bool whole;                  // their units are not split
  int64_t narrow_rows;         // what few rows are
  int64_t wide_units, splits;  // of sequences of more
  size_t part_bytes, wide_bytes;  // of workspace that their parts take
};

// A sequence of more rows than this goes to the wide form. In 32 bits its 128-row
// tiles cost more where rows are few: MI355X, 58 sequences of 300 to 2000 entries,
// 36 or 64 rows each, heads of 128, fp32 wide 103 / 114 us, narrow 53 / 65; bf16
// wide 28 / 29, narrow 36 / 42.
int64_t narrow_rows_of(int32_t dtype) { return dtype == KHRT_F32 ? 64 : 32; }

// Units of no more blocks than this are not split: a join costs as much as some
// blocks do. MI355X, split and whole: 1 x 300 entries (fp32, one head of 80) 16.1
// us / 12.8, 8 x 300 (bf16, 32 heads on 8 of 128) 17.4 / 11.7, 128 x 10 to 500 51 /
// 41; 1 x 1000 17 / 27, 8 x 1000 17 / 23.
constexpr int64_t kWholeBlocks = 4;

// Entries of a sequence that any of its new tokens sees: with a window nobody
// looks further back than the window and the new tokens.
int64_t seen_len(const kh_paged_attention_args &a) {
  const int64_t len = expected_len(a.table, a.cache);
  return a.window > 0 ? std::min(len, a.window + a.tokens) : len;
}

// A row of a part: fp32, with its maximum and sum.
size_t part_row_bytes(const kh_paged_attention_args &a) { return (2 + static_cast<size_t>(a.cache.head_dim)) * sizeof(float); }

// Workgroups of the narrow form that are on the chip at once.
int64_t most_groups(const kh_paged_attention_args &a) { return (a.cache.head_dim > 128 ? 1 : 2) * KH_GEMM_CUS; }

AttentionPlan attention_plan(const kh_paged_attention_args &a, size_t workspace_bytes) {
  AttentionPlan p{};
  const int64_t group = a.q_heads / a.cache.kv_heads, rows = a.tokens * group;
  const int64_t len = seen_len(a);
  const size_t row_bytes = part_row_bytes(a);

  // Few rows to a sequence, by all the host can know: the narrow form has them
  // all. One sequence: whichever suits its rows. Otherwise both.
  const int64_t few = narrow_rows_of(a.cache.dtype), most_rows = a.cache.dtype == KHRT_F32 ? 1024 : 256;
  const bool narrow_only = kh_narrow_only(a.tokens, a.table.seqs, group, a.max_new, few, most_rows);
  const bool wide_only = !narrow_only && a.table.seqs == 1;
  p.narrow_rows = narrow_only ? INT32_MAX : wide_only ? 0 : few;
  if (!narrow_only) {
    p.wide_units = (rows / KH_WIDE_ROWS + std::min(a.tokens, a.table.seqs)) * a.cache.kv_heads;
    // Two to a CU; parts are worth it while they fill the chip no more than once,
    // and down to 256 entries each. MI355X, bf16, 32 heads on 8 of 128: 1500 tokens
    // of 1500 entries whole 48 us, in two 68; 500 of 8000 in parts for half the
    // chip 112, for all of it 97. Least part 512 against 256 entries: fp32, 2 x 300
    // tokens of 1000 and 16 heads of 64 80 us / 42, bf16 64 of 1500 33 / 23.
    p.splits = std::clamp<int64_t>(2 * KH_GEMM_CUS / p.wide_units, 1, std::max<int64_t>(1, len / 256));
    const size_t all_rows = static_cast<size_t>(a.tokens * a.q_heads);
    p.splits = std::max<int64_t>(1, std::min<int64_t>(p.splits, static_cast<int64_t>(workspace_bytes / (all_rows * row_bytes))));
    p.wide_bytes = p.splits > 1 ? static_cast<size_t>(p.splits) * all_rows * row_bytes : 0;
    workspace_bytes -= p.wide_bytes;
  }
  if (wide_only) return p;

  // At most so many units, of at most so many blocks each.
  const int64_t narrow_most = narrow_only ? rows : std::min(rows, few * a.table.seqs);
  const int64_t units = (narrow_most / KH_TILE_ROWS + std::min(a.tokens, a.table.seqs)) * a.cache.kv_heads;
  const int64_t blocks = ceil_div(len, KH_STRETCH);
  const int64_t most = most_groups(a);
  const size_t per_group = size_t(2) * KH_TILE_ROWS * row_bytes;
  p.groups = std::min<int64_t>(most, std::max(ceil_div(units * blocks, 2), std::min(units, most)));
  p.groups = std::min(p.groups, static_cast<int64_t>(workspace_bytes / per_group));
  // The kernels count blocks in 32 bits, with what lengths beyond the expected
  // ones may add: the whole row of the table.
  const int64_t most_blocks = units * ceil_div(capacity_of(a.table.width, a.cache.page_size), KH_STRETCH);
  p.whole = blocks <= kWholeBlocks || p.groups < std::min(units, most) || p.groups < 2 || most_blocks >= 1 << 30;
  if (p.whole) p.groups = std::min(units, most);
  p.part_bytes = p.whole ? 0 : static_cast<size_t>(p.groups) * per_group;
  return p;
}

// What the plan of no step of at most these tokens, sequences, lengths and window
// takes more than. A single step's own need does not grow with the step: a long
// chunk fills the chip without parts, a short one and single tokens do not. Each
// of the plan's two terms is bounded by one that does grow.
size_t attention_workspace(const kh_paged_attention_args &a) {
  const int64_t group = a.q_heads / a.cache.kv_heads, rows = a.tokens * group, len = seen_len(a);
  const size_t row_bytes = part_row_bytes(a);
  // Narrow: two parts of 16 rows for each workgroup.
  const int64_t blocks = ceil_div(len, KH_STRETCH), most = most_groups(a);
  const int64_t units = (rows / KH_TILE_ROWS + std::min(a.tokens, a.table.seqs)) * a.cache.kv_heads;
  const int64_t groups = blocks <= kWholeBlocks ? 0 : std::min(most, units * blocks);
  // Wide: its splits times its units are at most two to a CU, and its rows fewer
  // than its units times theirs.
  const int64_t splits = len / 256;
  const int64_t wide_rows = splits < 2 || rows <= narrow_rows_of(a.cache.dtype)
                                ? 0 : std::min<int64_t>(2 * KH_GEMM_CUS * KH_WIDE_ROWS, splits * a.tokens * a.q_heads);
  return (static_cast<size_t>(groups < 2 ? 0 : groups) * 2 * KH_TILE_ROWS + static_cast<size_t>(wide_rows)) * row_bytes;
}

}  // namespace

extern "C" {

int kh_qk_norm_rope(const kh_qk_norm_rope_args *args, void *stream) {
  const char *op = "qk_norm_rope";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_qk_norm_rope_args &a = *args;
    const kh_paged_cache &c = a.cache;
    const bool cached = c.k != nullptr;
    if (int rc = cached ? check_cache(op, c, true) : check_rows(op, c)) return rc;
    if (int rc = check_tokens(op, a.tokens, a.q_heads, c)) return rc;
    if (!a.q || !a.k || !a.q_out || (!a.k_out && !cached) || (cached && (!a.v || !a.slots))) return bad(op, "null buffer");
    if (a.rotary_dim < 0 || a.rotary_dim > c.head_dim || a.rotary_dim % 8 != 0)
      return bad(op, "rotary_dim must be a multiple of 8 up to head_dim");
    if (a.rotary_dim > 0 && (!a.inv_freq || !a.positions)) return bad(op, "null inv_freq or positions");
    if (!(a.eps >= 0.0f) || !std::isfinite(a.eps)) return bad(op, "eps must be finite and not negative");
    for (const void *p : {a.q, a.k, cached ? a.v : nullptr, static_cast<const void *>(a.q_out),
                          static_cast<const void *>(a.k_out), a.q_gamma, a.k_gamma})
      if (!aligned(p)) return bad(op, "buffers must be 16-byte aligned");
    if (cached && c.k == c.v) return bad(op, "k and v of the cache must not be the same");
    const int e = element_bytes(c.dtype);
    const int64_t q_row = a.q_heads * c.head_dim, k_row = c.kv_heads * c.head_dim;
    if (!stride_ok(a.q_stride, a.tokens, e, 0) || !stride_ok(a.k_stride, a.tokens, e, 0) ||
        (cached && !stride_ok(a.v_stride, a.tokens, e, 0)))
      return bad(op, "strides must be multiples of 16 bytes, not negative");
    if (!stride_ok(a.q_out_stride, a.tokens, e, q_row) || (a.k_out != nullptr && !stride_ok(a.k_out_stride, a.tokens, e, k_row)))
      return bad(op, "output strides must be multiples of 16 bytes and hold a token");
    if ((a.q_out == a.q && a.q_out_stride != a.q_stride) || (a.k_out == a.k && a.k_out_stride != a.k_stride))
      return bad(op, "in place, input and output strides must be the same");

    const int lanes = c.head_dim <= 64 ? 8 : c.head_dim <= 128 ? 16 : 32;
    // Heads of a token are shared out over waves until the chip has some
    // sixteen of them to a CU.
    const int64_t steps = ceil_div(a.q_heads, 64 / lanes) + 2 * ceil_div(c.kv_heads, 64 / lanes);
    const int64_t parts = std::clamp<int64_t>(ceil_div(16 * KH_GEMM_CUS, a.tokens), 1, steps);
    // A launch has fewer than 2^32 threads: more tokens than this take several.
    constexpr int64_t kMost = int64_t(1) << 25;
    const auto row = [](const void *at, int64_t elements, int size) {
      return at != nullptr ? const_cast<char *>(static_cast<const char *>(at)) + elements * size : nullptr;
    };
    for (int64_t t = 0; t < a.tokens; t += kMost) {
      const int64_t tokens = std::min(kMost, a.tokens - t);
      KhRopeParams p{row(a.q, t * a.q_stride, e), row(a.k, t * a.k_stride, e), cached ? row(a.v, t * a.v_stride, e) : nullptr,
                     row(a.q_out, t * a.q_out_stride, e), row(a.k_out, t * a.k_out_stride, e), a.q_gamma, a.k_gamma, a.inv_freq,
                     a.positions != nullptr ? a.positions + t : nullptr, a.slots != nullptr ? a.slots + t : nullptr, c.k, c.v,
                     a.q_stride, a.k_stride, a.v_stride, a.q_out_stride, a.k_out_stride, c.k_page_stride, c.k_slot_stride,
                     c.k_head_stride, c.v_page_stride, c.v_slot_stride, c.v_head_stride, cached ? c.pages * c.page_size : 0,
                     static_cast<int32_t>(c.page_size), static_cast<int32_t>(tokens), static_cast<int32_t>(a.q_heads),
                     static_cast<int32_t>(c.kv_heads), static_cast<int32_t>(c.head_dim), static_cast<int32_t>(a.rotary_dim),
                     a.interleaved != 0, a.norm != 0, static_cast<int32_t>(parts), a.eps};
      if (int rc = launch(kRope[lanes / 16][c.dtype], ceil_div(tokens * parts, 4), 1, 256, p, stream)) return rc;
    }
    return 0;
  });
}

int kh_paged_attention_workspace(const kh_paged_attention_args *args, size_t *bytes) {
  const char *op = "paged_attention_workspace";
  return guarded(op, [&] {
    if (args == nullptr || bytes == nullptr) return bad(op, "null argument");
    if (int rc = check_attention(op, *args)) return rc;
    *bytes = attention_workspace(*args);
    return 0;
  });
}

int kh_paged_attention(const kh_paged_attention_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  const char *op = "paged_attention";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_paged_attention_args &a = *args;
    if (int rc = check_attention(op, a)) return rc;
    if (!aligned(workspace)) return bad(op, "workspace must be 16-byte aligned");
    const AttentionPlan plan = attention_plan(a, workspace != nullptr ? workspace_bytes : 0);
    const int64_t group = a.q_heads / a.cache.kv_heads, rows = a.tokens * a.q_heads, d = a.cache.head_dim;
    const bool joined = plan.part_bytes + plan.wide_bytes > 0;
    // All rows of parts come first, 16 bytes at a time, then their statistics.
    float *const part_o = static_cast<float *>(workspace), *wide_o = part_o, *part_ml = part_o, *wide_ml = part_o;
    if (joined) {
      wide_o = part_o + (plan.part_bytes > 0 ? plan.groups * 2 * KH_TILE_ROWS * d : 0);
      part_ml = wide_o + (plan.wide_bytes > 0 ? plan.splits * rows * d : 0);
      wide_ml = part_ml + (plan.part_bytes > 0 ? plan.groups * 2 * KH_TILE_ROWS * 2 : 0);
    }
    const int64_t wide_blocks = plan.wide_units * plan.splits;
    const int e = element_bytes(a.cache.dtype);
    const bool even = even_pages(a.cache);
    // Scores are masked before the factor: it is above 0, which a scale of 0 makes up
    // for with queries of 0.
    const float factor = a.scale == 0.0f ? 1.0f : std::fabs(in_powers_of_two(a.scale));
    KhAttentionParams p{device_cache(a.cache), device_table(a.table, a.cache), a.q, a.out, a.lse, a.q_starts, part_o, part_ml,
                        wide_o, wide_ml, a.q_stride, a.out_stride, static_cast<int32_t>(a.tokens),
                        static_cast<int32_t>(a.q_heads), static_cast<int32_t>(group), static_cast<int32_t>(a.window),
                        static_cast<int32_t>(plan.groups), plan.whole, static_cast<int32_t>(plan.narrow_rows),
                        static_cast<int32_t>(wide_blocks), static_cast<int32_t>(std::max<int64_t>(plan.splits, 1)),
                        even, a.scale == 0.0f ? 0u : 0xffffffffu, a.scale < 0.0f ? (e == 4 ? 0x80000000u : 0x80008000u) : 0u,
                        kh_div_by(static_cast<uint32_t>(group)), factor};
    const auto &symbols = wide_blocks > 0 ? kWide : kAttention;
    if (int rc = launch(symbols[width_of(d)][a.cache.dtype], wide_blocks + plan.groups, 1, 256, p, stream)) return rc;
    if (!joined) return 0;
    const int64_t narrow_joins = plan.part_bytes > 0 ? plan.groups : 0;
    const int64_t wide_joins = plan.wide_bytes > 0 ? plan.wide_units * (KH_WIDE_ROWS / KH_TILE_ROWS) : 0;
    return launch(kJoin[width_of(d)][a.cache.dtype], narrow_joins + wide_joins, 1, 256, p, stream);
  });
}

int kh_paged_weights(const kh_paged_weights_args *args, void *stream) {
  const char *op = "paged_weights";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_paged_weights_args &a = *args;
    if (int rc = check_cache(op, a.cache, false)) return rc;
    if (int rc = check_table(op, a.table, a.cache)) return rc;
    if (!a.q || !a.lse || !a.q_starts || !a.weights) return bad(op, "null buffer");
    if (int rc = check_queries(op, a.q, a.q_stride, a.tokens, a.q_heads, a.window, a.scale, a.cache)) return rc;
    if (a.weights_seq_stride < 0 || a.weights_head_stride < 0 || a.weights_seq_stride > kMaxStride ||
        a.weights_head_stride > kMaxStride || (a.cache.kv_heads > 1 && a.weights_head_stride == 0) ||
        (a.table.seqs > 1 && a.weights_seq_stride == 0))
      return bad(op, "strides of weights must be positive");
    if (!rows_apart({a.weights_seq_stride, a.table.seqs}, {a.weights_head_stride, a.cache.kv_heads}, 1))
      return bad(op, "rows of weights must not be the same");
    const int e = element_bytes(a.cache.dtype);
    if (a.q_stride * e >= 1 << 24) return bad(op, "q_stride must be below 2^24 bytes");
    const int64_t group = a.q_heads / a.cache.kv_heads, pairs = a.cache.kv_heads * a.table.seqs;
    // Chunks as long as leaves every CU some four workgroups, up to 1024 entries
    // (eight blocks of a wave); one stretch where sequences may have many rows.
    const int64_t len = expected_len(a.table, a.cache), stretches = ceil_div(len, KH_STRETCH);
    const bool few = a.tokens * group <= 32 * a.table.seqs;
    const int64_t each = few ? std::clamp<int64_t>(pairs * stretches / (4 * KH_GEMM_CUS), 1, 8) : 1;
    const int64_t chunks = std::min(ceil_div(stretches, each), std::max<int64_t>(1, (int64_t(1) << 22) / pairs));
    KhWeightsParams p{device_cache(a.cache), device_table(a.table, a.cache), a.q, a.lse, a.q_starts, a.weights_in, a.weights,
                      a.q_stride, a.weights_seq_stride, a.weights_head_stride, static_cast<int32_t>(a.tokens),
                      static_cast<int32_t>(a.q_heads), static_cast<int32_t>(group), static_cast<int32_t>(a.window),
                      static_cast<int32_t>(each * KH_STRETCH), static_cast<int32_t>(chunks), even_pages(a.cache),
                      32 % group == 0 && a.q_stride >= a.q_heads * a.cache.head_dim, kh_div_by(static_cast<uint32_t>(group)), in_powers_of_two(a.scale)};
    return launch((few ? kWeights : kWeightsWide)[width_of(a.cache.head_dim)][a.cache.dtype], pairs * chunks, 1, 256, p, stream);
  });
}

static int check_evict(const char *op, const kh_paged_evict_args &a) {
  if (int rc = check_cache(op, a.cache, true)) return rc;
  if (int rc = check_table(op, a.table, a.cache)) return rc;
  if (!a.kept_pages || !a.kept_lens || !a.weights_in || !a.weights) return bad(op, "null buffer");
  if (a.budget <= 0 || a.budget > kCapacity || a.budget * a.cache.kv_heads > kMaxRows)
    return bad(op, "budget must be positive, and at most 2^30 rows of a sequence");
  if (a.recent < 0 || a.recent > a.budget) return bad(op, "recent must be in [0, budget]");
  if (a.kept_width <= 0 || a.kept_width > INT32_MAX || a.kept_row_stride < 0 || a.kept_row_stride > kMaxStride ||
      (a.table.seqs > 1 && a.kept_row_stride < a.kept_width))
    return bad(op, "kept_width must be positive and rows of kept_pages not overlap");
  if (a.kept_width * a.cache.page_size < a.budget) return bad(op, "kept_pages must hold budget entries");
  if (a.kept_pages == a.table.pages || a.kept_lens == a.table.lens || a.weights == a.weights_in)
    return bad(op, "what is written must not be what is read");
  const int64_t pairs[][2] = {{a.in_seq_stride, a.table.seqs}, {a.in_head_stride, a.cache.kv_heads},
                              {a.seq_stride, a.table.seqs}, {a.head_stride, a.cache.kv_heads}};
  for (const auto &s : pairs)
    if (s[0] < 0 || s[0] > kMaxStride) return bad(op, "strides of weights must not be negative");
  if ((a.table.seqs > 1 && a.seq_stride < a.budget) || (a.cache.kv_heads > 1 && a.head_stride < a.budget))
    return bad(op, "rows of weights must hold budget entries");
  if (!rows_apart({a.seq_stride, a.table.seqs}, {a.head_stride, a.cache.kv_heads}, a.budget))
    return bad(op, "rows of weights must not overlap");
  return 0;
}

static size_t evict_bytes(const kh_paged_evict_args &a) {
  return static_cast<size_t>(a.table.seqs * a.cache.kv_heads) * static_cast<size_t>(a.budget) * sizeof(int32_t);
}

int kh_paged_evict_workspace(const kh_paged_evict_args *args, size_t *bytes) {
  const char *op = "paged_evict_workspace";
  return guarded(op, [&] {
    if (args == nullptr || bytes == nullptr) return bad(op, "null argument");
    if (int rc = check_evict(op, *args)) return rc;
    *bytes = evict_bytes(*args);
    return 0;
  });
}

int kh_paged_evict(const kh_paged_evict_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  const char *op = "paged_evict";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_paged_evict_args &a = *args;
    if (int rc = check_evict(op, a)) return rc;
    if (workspace == nullptr || workspace_bytes < evict_bytes(a))
      return bad(op, "workspace of " + std::to_string(evict_bytes(a)) + " bytes needed");
    if (!aligned(workspace)) return bad(op, "workspace must be 16-byte aligned");
    const int64_t pairs = a.cache.kv_heads * a.table.seqs, pieces = a.cache.head_dim * element_bytes(a.cache.dtype) / 16;
    int lanes = 1;
    while (lanes < pieces) lanes *= 2;
    const int64_t chunks = std::min(ceil_div(a.budget * a.cache.kv_heads, 4 * 256 / lanes),
                                    std::max<int64_t>(1, (int64_t(1) << 22) / a.table.seqs));
    KhEvictParams p{device_cache(a.cache), device_table(a.table, a.cache), a.kept_pages, a.kept_lens, a.weights_in, a.weights,
                    static_cast<int32_t *>(workspace), a.kept_row_stride, a.in_seq_stride, a.in_head_stride, a.seq_stride,
                    a.head_stride, static_cast<int32_t>(a.kept_width), static_cast<int32_t>(a.budget),
                    static_cast<int32_t>(a.recent), element_bytes(a.cache.dtype), lanes, static_cast<int32_t>(chunks),
                    a.cache.k_head_stride < a.cache.k_slot_stride, kh_div_by(static_cast<uint32_t>(a.cache.kv_heads))};
    if (int rc = launch(kChoose, pairs, 1, 1024, p, stream)) return rc;
    return launch(kMove, a.table.seqs * chunks, 1, 256, p, stream);
  });
}

}  // extern "C"
