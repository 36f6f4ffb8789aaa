// What the operators over paged caches share behind the C-ABI: the checks of what
// the host can see, and the launch geometry of attention.
#pragma once

#include "kernelh/khrt_internal.hpp"
#include "kh_paged.h"
#include "kh_tiles.h"

#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <string>
#include <utility>

namespace khrt::cache {

inline int bad(const char *op, const std::string &what) { return khrt::fail(KHRT_E_INVALID, std::string(op) + ": " + what); }

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

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline int element_bytes(int32_t dtype) { return dtype == KHRT_F32 ? 4 : 2; }

inline bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A stride over `extent` rows: not negative, 16 bytes' worth, and for rows that
// are written (least > 0) no shorter than the row where there is a next one.
inline bool stride_ok(int64_t stride, int64_t extent, int element, int64_t least) {
  if (extent <= 1) return stride >= 0 && stride <= kMaxSpan;
  return stride >= least && stride <= kMaxSpan / extent && stride % (16 / element) == 0;
}

// Whether rows of `row` elements at i a.stride + j b.stride, i < a.extent,
// j < b.extent, lie apart. One of the extents is below 2^10 wherever this is asked
// of strides that do not nest (pairs of sequence and kv head).
struct Steps {
  int64_t stride, extent;
};

inline bool nest(Steps inner, Steps outer, int64_t row) {
  if (inner.extent <= 1) return outer.extent <= 1 || outer.stride >= row;
  return inner.stride >= row && (outer.extent <= 1 || outer.stride >= (inner.extent - 1) * inner.stride + row);
}

inline bool rows_apart(Steps a, Steps b, int64_t row) {
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

// Whether rows of `row` elements over pages, slots and heads lie apart: whatever
// their order, each holds the ones inside.
inline bool nested(Steps pages, Steps slots, Steps heads, int64_t row) {
  Steps s[] = {pages, slots, heads};
  std::sort(s, s + 3, [](const Steps &a, const Steps &b) { return (a.extent > 1 ? a.stride : 0) < (b.extent > 1 ? b.stride : 0); });
  int64_t inside = row;
  for (const Steps &x : s) {
    if (x.extent <= 1) continue;
    if (x.stride < inside) return false;
    inside += (x.extent - 1) * x.stride;
  }
  return true;
}

// The fields that describe rows, of a cache that may have none.
inline int check_rows(const char *op, const kh_paged_cache &c) {
  if (c.dtype != KHRT_F32 && c.dtype != KHRT_F16 && c.dtype != KHRT_BF16)
    return bad(op, "dtype must be KHRT_F32, KHRT_F16 or KHRT_BF16 (got " + std::to_string(c.dtype) + ")");
  if (c.head_dim <= 0 || c.head_dim > 256 || c.head_dim % 8 != 0)
    return bad(op, "head_dim must be a multiple of 8 up to 256 (got " + std::to_string(c.head_dim) + ")");
  if (c.kv_heads <= 0 || c.kv_heads > 65535) return bad(op, "kv_heads must be in [1, 65535]");
  return 0;
}

inline int check_cache(const char *op, const kh_paged_cache &c, bool written) {
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
    if (!nested({is_v ? c.v_page_stride : c.k_page_stride, c.pages}, {is_v ? c.v_slot_stride : c.k_slot_stride, c.page_size},
                {is_v ? c.v_head_stride : c.k_head_stride, c.kv_heads}, c.head_dim))
      return bad(op, "rows of a cache that is written must not overlap");
  }
  return 0;
}

inline int check_table(const char *op, const kh_page_table &t, const kh_paged_cache &c) {
  if (t.pages == nullptr || t.lens == nullptr) return bad(op, "null page table");
  if (t.seqs <= 0 || t.width <= 0 || t.width > INT32_MAX) return bad(op, "seqs and width must be positive");
  if (t.row_stride < 0 || t.row_stride > kMaxStride) return bad(op, "the table's row stride must not be negative");
  if (t.seqs > kMaxPairs || t.seqs * c.kv_heads > kMaxPairs) return bad(op, "more than 2^20 pairs of sequence and kv head");
  if (t.max_len < 0) return bad(op, "max_len must not be negative");
  return 0;
}

inline KhCache device_cache(const kh_paged_cache &c) {
  const int e = element_bytes(c.dtype);
  auto bytes = [e](int64_t stride) { return static_cast<uint32_t>(stride * e); };
  return KhCache{static_cast<const char *>(c.k), static_cast<const char *>(c.v), bytes(c.k_page_stride),
                 bytes(c.k_slot_stride), bytes(c.k_head_stride), bytes(c.v_page_stride), bytes(c.v_slot_stride),
                 bytes(c.v_head_stride), static_cast<int32_t>(c.pages), static_cast<int32_t>(c.page_size),
                 static_cast<int32_t>(c.kv_heads), static_cast<int32_t>(c.head_dim),
                 kh_div_by(static_cast<uint32_t>(c.page_size))};
}

inline int64_t capacity_of(int64_t width, int64_t page_size) { return std::min(width * page_size, kCapacity); }

inline KhTable device_table(const kh_page_table &t, const kh_paged_cache &c) {
  return KhTable{t.pages, t.lens, t.row_stride, static_cast<int32_t>(t.seqs), static_cast<int32_t>(t.width),
                 static_cast<int32_t>(capacity_of(t.width, c.page_size))};
}

// Rows that follow each other 16 at a time, none longer than their distance,
// and 16 of those distances in 31 bits: pages are walked 16 entries at a time.
inline bool even_pages(const kh_paged_cache &c) {
  const auto [near, far] = std::minmax(c.k_slot_stride, c.v_slot_stride);
  return c.page_size % 16 == 0 && near >= c.head_dim && far * element_bytes(c.dtype) < 1 << 27;
}

// The longest sequence that a launch is sized for.
inline int64_t expected_len(const kh_page_table &t, const kh_paged_cache &c) {
  const int64_t all = capacity_of(t.width, c.page_size);
  return t.max_len > 0 ? std::min(t.max_len, all) : all;
}

inline int check_tokens(const char *op, int64_t tokens, int64_t q_heads, const kh_paged_cache &c) {
  if (tokens <= 0 || q_heads <= 0) return bad(op, "tokens and q_heads must be positive");
  if (tokens > kMaxRows || q_heads > 65535 || tokens * (q_heads + 2 * c.kv_heads) > kMaxRows)
    return bad(op, "more than 2^30 rows");
  return 0;
}

inline int check_queries(const char *op, const void *q, int64_t q_stride, int64_t tokens, int64_t q_heads, int64_t window,
                  float scale, const kh_paged_cache &c) {
  if (int rc = check_tokens(op, tokens, q_heads, c)) return rc;
  if (q_heads % c.kv_heads != 0) return bad(op, "q_heads must be a multiple of kv_heads");
  if (!aligned(q)) return bad(op, "q must be 16-byte aligned");
  if (!stride_ok(q_stride, tokens, element_bytes(c.dtype), 0)) return bad(op, "q_stride must be a multiple of 16 bytes, not negative");
  if (window < 0 || window > INT32_MAX) return bad(op, "window must be in [0, 2^31)");
  if (!std::isfinite(scale)) return bad(op, "scale must be finite");
  return 0;
}

// A kernel by its code object and name.
struct Symbol {
  const char *co, *name;
};
// Which of the kernels' widths holds head_dim: 64, 128 or 256.
inline int width_of(int64_t head_dim) { return head_dim <= 64 ? 0 : head_dim <= 128 ? 1 : 2; }

template <class Params>
int launch(const Symbol &s, int64_t x, int64_t y, unsigned threads, Params &p, void *stream) {
  void *params[] = {&p};
  return khrt::launch_embedded(s.co, s.name, khrt_dim3{static_cast<unsigned>(x), static_cast<unsigned>(y), 1},
                               khrt_dim3{threads, 1, 1}, stream, params, 1);
}

inline int check_attention(const char *op, const kh_paged_attention_args &a) {
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
inline float in_powers_of_two(float scale) {
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
inline int64_t narrow_rows_of(int32_t dtype) { return dtype == KHRT_F32 ? 64 : 32; }

// Units of no more blocks than this are not split: a join costs as much as some
// blocks do. MI355X, split and whole: 1 x 300 entries (fp32, one head of 80) 16.1
// us / 12.8, 8 x 300 (bf16, 32 heads on 8 of 128) 17.4 / 11.7, 128 x 10 to 500 51 /
// 41; 1 x 1000 17 / 27, 8 x 1000 17 / 23.
constexpr int64_t kWholeBlocks = 4;

// Entries of a sequence that any of its new tokens sees: with a window nobody
// looks further back than the window and the new tokens.
inline int64_t seen_len(const kh_paged_attention_args &a) {
  const int64_t len = expected_len(a.table, a.cache);
  return a.window > 0 ? std::min(len, a.window + a.tokens) : len;
}

// A row of a part: fp32, with its maximum and sum.
inline size_t part_row_bytes(const kh_paged_attention_args &a) { return (2 + static_cast<size_t>(a.cache.head_dim)) * sizeof(float); }

// Workgroups of the narrow form that are on the chip at once.
inline int64_t most_groups(const kh_paged_attention_args &a) { return (a.cache.head_dim > 128 ? 1 : 2) * KH_GEMM_CUS; }

// How sequences of few rows are worked on: workgroups on the chip at once, kv heads
// that each takes, blocks of units that are not split.
struct NarrowForm {
  int64_t most, together = 1, whole = kWholeBlocks;
};

inline AttentionPlan attention_plan(const kh_paged_attention_args &a, size_t workspace_bytes, const NarrowForm &form) {
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
  const int64_t units = (narrow_most / KH_TILE_ROWS + std::min(a.tokens, a.table.seqs)) * ceil_div(a.cache.kv_heads, form.together);
  const int64_t blocks = ceil_div(len, KH_STRETCH), most = form.most;
  const size_t per_group = static_cast<size_t>(2 * KH_TILE_ROWS * form.together) * row_bytes;
  p.groups = std::min<int64_t>(most, std::max(ceil_div(units * blocks, 2), std::min(units, most)));
  p.groups = std::min(p.groups, static_cast<int64_t>(workspace_bytes / per_group));
  // The kernels count blocks in 32 bits, with what lengths beyond the expected
  // ones may add: the whole row of the table.
  const int64_t most_blocks = units * ceil_div(capacity_of(a.table.width, a.cache.page_size), KH_STRETCH);
  p.whole = blocks <= form.whole || p.groups < std::min(units, most) || p.groups < 2 || most_blocks >= 1 << 30;
  if (p.whole) p.groups = std::min(units, most);
  p.part_bytes = p.whole ? 0 : static_cast<size_t>(p.groups) * per_group;
  return p;
}

// What the plan of no step of at most these tokens, sequences, lengths and window
// takes more than. A single step's own need does not grow with the step: a long
// chunk fills the chip without parts, a short one and single tokens do not. Each
// of the plan's two terms is bounded by one that does grow. form: of the most heads.
inline size_t attention_workspace(const kh_paged_attention_args &a, const NarrowForm &form) {
  const int64_t group = a.q_heads / a.cache.kv_heads, rows = a.tokens * group, len = seen_len(a);
  const size_t row_bytes = part_row_bytes(a);
  // Narrow: two parts of 16 rows of its heads for each workgroup.
  const int64_t blocks = ceil_div(len, KH_STRETCH);
  const int64_t units = (rows / KH_TILE_ROWS + std::min(a.tokens, a.table.seqs)) * (a.cache.kv_heads + form.together - 1);
  const int64_t groups = blocks <= kWholeBlocks ? 0 : std::min(form.most * form.together, units * blocks);
  // Wide: its splits times its units are at most two to a CU, and its rows fewer
  // than its units times theirs.
  const int64_t splits = len / 256;
  const int64_t wide_rows = splits < 2 || rows <= narrow_rows_of(a.cache.dtype)
                                ? 0 : std::min<int64_t>(2 * KH_GEMM_CUS * KH_WIDE_ROWS, splits * a.tokens * a.q_heads);
  return (static_cast<size_t>((groups < 2 ? 0 : groups) * 2 * KH_TILE_ROWS) + static_cast<size_t>(wide_rows)) * row_bytes;
}

}  // namespace khrt::cache
