// The operators over a cache in 8 bits behind the C-ABI (khrt.h, group 9).
#include "kernelh/khrt_cache.hpp"

using namespace khrt::cache;

namespace {

#define KH_BY_TYPE(base, suffix)                                                              \
  {                                                                                           \
    {#base "_f32", #base suffix "_f32"}, {#base "_f16", #base suffix "_f16"}, {#base "_bf16", #base suffix "_bf16"} \
  }
const Symbol kRope[3][3] = {KH_BY_TYPE(rope8, "_8"), KH_BY_TYPE(rope8, "_16"), KH_BY_TYPE(rope8, "_32")};
const Symbol kRead[3] = KH_BY_TYPE(read8, "");
const Symbol kAttention[3][3] = {KH_BY_TYPE(attention8, "_64"), KH_BY_TYPE(attention8, "_128"), KH_BY_TYPE(attention8, "_256")};
constexpr size_t kJoinBytes = sizeof(KhJoin) * 2 * KH_GEMM_CUS;
constexpr unsigned kWaves[3] = {4, 4, 2};  // of a workgroup of kAttention's
const Symbol kOdd[3][3] = {KH_BY_TYPE(attention8, "_odd_64"), KH_BY_TYPE(attention8, "_odd_128"), KH_BY_TYPE(attention8, "_odd_256")};
const Symbol kWide[3][3] = {KH_BY_TYPE(attention8, "_wide_64"), KH_BY_TYPE(attention8, "_wide_128"),
                            KH_BY_TYPE(attention8, "_wide_256")};
const Symbol kJoin[3][3] = {KH_BY_TYPE(attention8, "_join_64"), KH_BY_TYPE(attention8, "_join_128"),
                            KH_BY_TYPE(attention8, "_join_256")};
const Symbol kCombine[3][3] = {KH_BY_TYPE(attention8, "_combine_64"), KH_BY_TYPE(attention8, "_combine_128"),
                               KH_BY_TYPE(attention8, "_combine_256")};

// Rows of `dtype` beside a cache in 8 bits, as the checks of rows take them.
kh_paged_cache rows_of(const kh_paged_cache8 &c, int32_t dtype) {
  kh_paged_cache r{};
  r.pages = c.pages, r.page_size = c.page_size, r.kv_heads = c.kv_heads, r.head_dim = c.head_dim, r.dtype = dtype;
  return r;
}

int check_cache8(const char *op, const kh_paged_cache8 &c, int32_t dtype, bool written) {
  if (int rc = check_rows(op, rows_of(c, dtype))) return rc;
  if (c.head_dim % 16 != 0) return bad(op, "head_dim must be a multiple of 16 (got " + std::to_string(c.head_dim) + ")");
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return bad(op, "null cache");
  if (c.pages <= 0 || c.pages > INT32_MAX) return bad(op, "pages must be in [1, 2^31)");
  if (c.page_size <= 0 || c.page_size > kMaxPageSize) return bad(op, "page_size must be in [1, 2^20]");
  const int64_t least = written ? c.head_dim : 0;
  for (const bool is_v : {false, true}) {
    const Steps pages{is_v ? c.v_page_stride : c.k_page_stride, c.pages}, slots{is_v ? c.v_slot_stride : c.k_slot_stride, c.page_size},
        heads{is_v ? c.v_head_stride : c.k_head_stride, c.kv_heads};
    if (!aligned(is_v ? c.v : c.k)) return bad(op, "the cache must be 16-byte aligned");
    for (const Steps &s : {pages, slots, heads}) {
      if (s.stride >= kMaxCacheStride) return bad(op, "cache strides must be below 2^32 bytes");
      if (!stride_ok(s.stride, s.extent, 1, least))
        return bad(op, written ? "cache strides must be multiples of 16 bytes and hold a row"
                               : "cache strides must be multiples of 16 bytes, not negative");
    }
    if (written && !nested(pages, slots, heads, c.head_dim)) return bad(op, "rows of a cache that is written must not overlap");
  }
  for (const int64_t s : {c.scale_page_stride, c.scale_head_stride})
    if (s < 0 || s >= kMaxCacheStride) return bad(op, "strides of scales must be in [0, 2^32)");
  if (!written) return 0;
  if (!nested({c.scale_page_stride, c.pages}, {1, c.page_size}, {c.scale_head_stride, c.kv_heads}, 1))
    return bad(op, "scales of a cache that is written must not overlap");
  const void *const parts[] = {c.k, c.v, c.k_scale, c.v_scale};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (parts[i] == parts[j]) return bad(op, "k, v and their scales must not be the same");
  return 0;
}

int check_attention8(const char *op, const kh_paged_attention8_args &a) {
  if (int rc = check_cache8(op, a.cache, a.dtype, false)) return rc;
  const kh_paged_cache rows = rows_of(a.cache, a.dtype);
  if (int rc = check_table(op, a.table, rows)) return rc;
  if (!a.q || !a.out || !a.q_starts) return bad(op, "null buffer");
  if (int rc = check_queries(op, a.q, a.q_stride, a.tokens, a.q_heads, a.window, a.scale, rows)) return rc;
  if (!aligned(a.out)) return bad(op, "out must be 16-byte aligned");
  if (!stride_ok(a.out_stride, a.tokens, element_bytes(a.dtype), a.q_heads * a.cache.head_dim))
    return bad(op, "out_stride must be a multiple of 16 bytes and hold a token");
  if (a.out == a.q) return bad(op, "out must not be q");
  if (a.max_new < 0 || a.shared < 0) return bad(op, "max_new and shared must not be negative");
  if (!(a.cap >= 0.0f) || !std::isfinite(a.cap)) return bad(op, "cap must be finite and not negative");
  return 0;
}

// The step as the plan of paged_attention takes it: products are of bf16 numbers.
// behind: entries of every sequence that are not its business.
kh_paged_attention_args as_plain(const kh_paged_attention8_args &a, int64_t behind) {
  kh_paged_attention_args p{};
  p.cache = rows_of(a.cache, KHRT_BF16);
  p.table = a.table;
  p.tokens = a.tokens, p.q_heads = a.q_heads, p.window = a.window, p.max_new = a.max_new;
  p.table.max_len = std::max<int64_t>(1, expected_len(a.table, p.cache) - behind);
  return p;
}

// As even_pages; four scales from a multiple of four slots on are a word; and
// places of scales and page numbers, past a head's first and a row's, fit 32 bits.
bool even_pages8(const kh_paged_attention8_args &a) {
  const kh_paged_cache8 &c = a.cache;
  const auto [near, far] = std::minmax(c.k_slot_stride, c.v_slot_stride);
  const uintptr_t words = reinterpret_cast<uintptr_t>(c.k_scale) | reinterpret_cast<uintptr_t>(c.v_scale) |
                          static_cast<uintptr_t>(c.scale_page_stride) | static_cast<uintptr_t>(c.scale_head_stride);
  return c.page_size % 16 == 0 && near >= c.head_dim && far < 1 << 27 && words % 4 == 0 &&
         c.pages * c.scale_page_stride + c.page_size < int64_t(1) << 32 && a.table.width < 1 << 29;
}

// kv heads that a workgroup reads together at the most: where those of an entry lie
// next to each other, as many as make 256 bytes. Memory is slower by as much as a
// quarter where neighbours of 128 bytes are read at different times: MI355X, 64
// sequences of 513 to 8192 entries, 8 kv heads of 128, one at a time 131 us, two
// 115, four 112 (and longer where parts are joined).
int64_t most_together(const kh_paged_attention8_args &a) {
  const kh_paged_cache8 &c = a.cache;
  if (c.kv_heads == 1 || c.k_head_stride > 256 || c.v_head_stride > 256) return 1;
  return std::min<int64_t>(c.kv_heads, c.head_dim <= 64 ? 4 : c.head_dim <= 128 ? 2 : 1);
}

// Units of up to this many blocks are not split by workgroups of four waves that have
// pages of whole sixteens: shares that end anywhere change units, and a join is
// another launch. MI355X, bf16, 32 heads on 8 of 128, split and whole: 16 x 700
// entries 20.2 us / 15.6, 128 x 10 to 880 45 / 35, 32 x 100 to 880 24.7 / 25.4; of one
// more block, 8 x 1024, 16.5 / 18.0. Workgroups of two waves: 8 x 850, 8 heads of 256,
// 27 / 37.
constexpr int64_t kWholeEven = 7;

// Beside entries that sequences share, whose units take some 25 us, units of up to
// this many blocks are not split: a join is another launch.
constexpr int64_t kWholeShared = 8;

// The kernels' two factors of a cap: scores y (queries times keys) become
// out tanh(y in / (2 log2 e)), in powers of two. in 0: they are not capped.
struct Cap {
  float in, out;
};

// factor: |scale| log2(e). A cap whose factors are past the normal numbers is none: it
// is above 2^127, or above 2^127 times |scale|, and tanh(x) = x - x^3/3 + .. leaves
// a y, or a score, below 2^114 as it is.
Cap cap_of(float cap, float factor) {
  using Float = std::numeric_limits<float>;
  const double in = 2.0 * static_cast<double>(factor) / static_cast<double>(cap), out = static_cast<double>(cap) * 1.44269504088896340736;
  if (!(cap > 0.0f) || in < static_cast<double>(Float::min()) || out > static_cast<double>(Float::max())) return {0.0f, 0.0f};
  return {static_cast<float>(std::min(in, static_cast<double>(Float::max()))), static_cast<float>(out)};
}

// Fewer where there would not be a block of entries for every workgroup.
int64_t heads_together(const kh_paged_attention8_args &a, int64_t behind) {
  const kh_paged_cache8 &c = a.cache;
  const int64_t units = std::min(a.tokens, a.table.seqs) + a.tokens * (a.q_heads / c.kv_heads) / KH_TILE_ROWS;
  const int64_t blocks = ceil_div(seen_len(as_plain(a, behind)), KH_STRETCH);
  int64_t n = most_together(a);
  while (n > 1 && units * ceil_div(c.kv_heads, n) * blocks < 2 * KH_GEMM_CUS) n = (n + 1) / 2;
  return n;
}

// How the entries that sequences share are worked on: not at all (splits 0), or the
// first `entries` of them by units of KH_WIDE_ROWS rows of all tokens, in `splits`
// parts of `each`. Those past the expected length are each sequence's own: what the
// kernels are told is what the parts were cut from.
struct SharedPlan {
  int64_t entries, units, splits, each;
  size_t bytes;
};

constexpr int64_t kSharedLeast = 256;  // entries of a part

int64_t shared_units(const kh_paged_attention8_args &a) {
  return ceil_div(a.tokens * (a.q_heads / a.cache.kv_heads), KH_WIDE_ROWS) * a.cache.kv_heads;
}

// Rows of a step past which its entries are not shared: parts of more take gigabytes,
// and where sequences have many rows each they read their entries once as it is.
int64_t most_shared_rows(const kh_paged_attention8_args &a) {
  return std::min(int64_t(1) << 22, (narrow_rows_of(KHRT_BF16) + 1) * a.table.seqs * a.cache.kv_heads);
}

SharedPlan shared_plan(const kh_paged_attention8_args &a, size_t workspace_bytes) {
  SharedPlan p{};
  const kh_paged_attention_args plain = as_plain(a, 0);
  const int64_t shared = std::min(a.shared, expected_len(a.table, plain.cache));
  const int64_t rows = a.tokens * a.q_heads, group = a.q_heads / a.cache.kv_heads;
  if (shared <= 0 || a.table.seqs < 2 || rows > most_shared_rows(a)) return p;
  const size_t part = static_cast<size_t>(rows) * part_row_bytes(plain);
  // What the sequences of few rows need not read, against what parts write and
  // read and the launch that joins them.
  const int64_t few = a.table.seqs - a.tokens * group / (narrow_rows_of(KHRT_BF16) + 1);
  p.units = shared_units(a);
  const int64_t most = std::clamp<int64_t>(KH_GEMM_CUS / p.units, 1, std::max<int64_t>(1, shared / kSharedLeast));
  const int64_t splits = std::min<int64_t>(most, static_cast<int64_t>(workspace_bytes / part) - 1);
  if (splits < 1) return p;
  const double saved = static_cast<double>(few - 1) * static_cast<double>(shared * a.cache.kv_heads * 2 * (a.cache.head_dim + 1));
  if (saved < 25e6 + 2.0 * static_cast<double>(splits + 1) * static_cast<double>(part)) return p;
  p.entries = shared;
  p.each = ceil_div(ceil_div(shared, splits), 64) * 64;
  p.splits = ceil_div(shared, p.each);
  p.bytes = static_cast<size_t>(p.splits + 1) * part;
  return p;
}

// What the shared plan of no smaller step takes more than: its parts' rows are at
// most those of a unit to a CU, or those of one part, and it has no more rows than
// may share entries.
size_t shared_workspace(const kh_paged_attention8_args &a) {
  if (a.shared == 0 || a.table.seqs < 2) return 0;
  const int64_t rows = std::min(a.tokens * a.q_heads, most_shared_rows(a));
  return static_cast<size_t>(rows + std::max<int64_t>(rows, KH_GEMM_CUS * KH_WIDE_ROWS)) * part_row_bytes(as_plain(a, 0));
}

}  // namespace

extern "C" {

int kh_qk_norm_rope8(const kh_qk_norm_rope8_args *args, void *stream) {
  const char *op = "qk_norm_rope8";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_qk_norm_rope8_args &a = *args;
    const kh_paged_cache8 &c = a.cache;
    if (int rc = check_cache8(op, c, a.dtype, true)) return rc;
    if (int rc = check_tokens(op, a.tokens, a.q_heads, rows_of(c, a.dtype))) return rc;
    if (!a.q || !a.k || !a.v || !a.q_out || !a.slots) return bad(op, "null buffer");
    if (a.rotary_dim < 0 || a.rotary_dim > c.head_dim || a.rotary_dim % 8 != 0)
      return bad(op, "rotary_dim must be a multiple of 8 up to head_dim");
    if (a.rotary_dim > 0 && (!a.inv_freq || !a.positions)) return bad(op, "null inv_freq or positions");
    if (a.rotary_dim > 0 && (a.axes < 1 || a.axes > 128)) return bad(op, "axes must be in [1, 128]");
    if (a.axis_stride < 0 || a.axis_stride > kMaxStride) return bad(op, "axis_stride must not be negative");
    if (!(a.eps >= 0.0f) || !std::isfinite(a.eps)) return bad(op, "eps must be finite and not negative");
    for (const void *p : {a.q, a.k, a.v, static_cast<const void *>(a.q_out), static_cast<const void *>(a.k_out), a.q_gamma, a.k_gamma})
      if (!aligned(p)) return bad(op, "buffers must be 16-byte aligned");
    const int e = element_bytes(a.dtype);
    if (!stride_ok(a.q_stride, a.tokens, e, 0) || !stride_ok(a.k_stride, a.tokens, e, 0) || !stride_ok(a.v_stride, a.tokens, e, 0))
      return bad(op, "strides must be multiples of 16 bytes, not negative");
    if (!stride_ok(a.q_out_stride, a.tokens, e, a.q_heads * c.head_dim) ||
        (a.k_out != nullptr && !stride_ok(a.k_out_stride, a.tokens, e, c.kv_heads * c.head_dim)))
      return bad(op, "output strides must be multiples of 16 bytes and hold a token");
    if ((a.q_out == a.q && a.q_out_stride != a.q_stride) || (a.k_out == a.k && a.k_out_stride != a.k_stride))
      return bad(op, "in place, input and output strides must be the same");
    for (const void *p : std::initializer_list<const void *>{c.k, c.v, c.k_scale, c.v_scale})
      if (p == a.q || p == a.k || p == a.v || p == a.q_out || p == a.k_out) return bad(op, "the cache must not be one of the rows' buffers");
    if (a.q_out == a.k || a.q_out == a.v || a.q_out == a.k_out || (a.k_out != nullptr && (a.k_out == a.q || a.k_out == a.v)))
      return bad(op, "an output must not be another input or output");

    // As kh_qk_norm_rope shares heads out, and launches.
    const int lanes = c.head_dim <= 64 ? 8 : c.head_dim <= 128 ? 16 : 32;
    const int64_t steps = ceil_div(a.q_heads, 64 / lanes) + 2 * ceil_div(c.kv_heads, 64 / lanes);
    const int64_t parts = std::clamp<int64_t>(ceil_div(16 * KH_GEMM_CUS, a.tokens), 1, steps);
    constexpr int64_t kMost = int64_t(1) << 25;
    const auto row = [](const void *at, int64_t elements, int size) {
      return at != nullptr ? const_cast<char *>(static_cast<const char *>(at)) + elements * size : nullptr;
    };
    for (int64_t t = 0; t < a.tokens; t += kMost) {
      const int64_t tokens = std::min(kMost, a.tokens - t);
      KhRope8Params p{{row(a.q, t * a.q_stride, e), row(a.k, t * a.k_stride, e), row(a.v, t * a.v_stride, e),
                       row(a.q_out, t * a.q_out_stride, e), row(a.k_out, t * a.k_out_stride, e), a.q_gamma, a.k_gamma, a.inv_freq,
                       a.positions != nullptr ? a.positions + t : nullptr, a.slots + t, c.k, c.v, a.q_stride, a.k_stride, a.v_stride,
                       a.q_out_stride, a.k_out_stride, c.k_page_stride, c.k_slot_stride, c.k_head_stride, c.v_page_stride,
                       c.v_slot_stride, c.v_head_stride, c.pages * c.page_size, static_cast<int32_t>(c.page_size),
                       static_cast<int32_t>(tokens), static_cast<int32_t>(a.q_heads), static_cast<int32_t>(c.kv_heads),
                       static_cast<int32_t>(c.head_dim), static_cast<int32_t>(a.rotary_dim), a.interleaved != 0, a.norm != 0,
                       static_cast<int32_t>(parts), a.eps},
                      c.k_scale, c.v_scale, a.pair_axis, a.axis_stride, c.scale_page_stride, c.scale_head_stride,
                      static_cast<int32_t>(std::max<int64_t>(a.axes, 1)), kh_div_by(static_cast<uint32_t>(parts)),
                      kh_div_by(static_cast<uint32_t>(c.page_size)), 1.0 / static_cast<double>(c.head_dim)};
      if (int rc = launch(kRope[lanes / 16][a.dtype], ceil_div(tokens * parts, 4), 1, 256, p, stream)) return rc;
    }
    return 0;
  });
}

int kh_paged_read8(const kh_paged_read8_args *args, void *stream) {
  const char *op = "paged_read8";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_paged_read8_args &a = *args;
    const kh_paged_cache8 &c = a.cache;
    if (int rc = check_cache8(op, c, a.dtype, false)) return rc;
    if (int rc = check_tokens(op, a.tokens, 1, rows_of(c, a.dtype))) return rc;
    if (!a.slots || (!a.k_out && !a.v_out)) return bad(op, "null buffer");
    const int e = element_bytes(a.dtype);
    const int64_t row = c.kv_heads * c.head_dim;
    for (const bool is_v : {false, true}) {
      const void *out = is_v ? a.v_out : a.k_out;
      if (out == nullptr) continue;
      if (!aligned(out)) return bad(op, "buffers must be 16-byte aligned");
      if (!stride_ok(is_v ? a.v_out_stride : a.k_out_stride, a.tokens, e, row))
        return bad(op, "output strides must be multiples of 16 bytes and hold a token");
      for (const void *p : std::initializer_list<const void *>{c.k, c.v, c.k_scale, c.v_scale, a.slots})
        if (p == out) return bad(op, "what is written must not be what is read");
    }
    if (a.k_out == a.v_out) return bad(op, "k_out and v_out must not be the same");
    // Pieces of a token, of which a thread has four on their way; a workgroup takes
    // as many tokens as give it those, and fewer where the chip has room.
    const int64_t pieces = row * e / 16;
    const int64_t each = std::clamp<int64_t>(std::min(4 * 256 / pieces, ceil_div(a.tokens, 4 * KH_GEMM_CUS)), 1, 256);
    constexpr int64_t kMost = int64_t(1) << 23;  // workgroups of a launch
    for (int64_t t = 0; t < a.tokens; t += kMost * each) {
      const int64_t tokens = std::min(kMost * each, a.tokens - t);
      const auto at = [&](void *out, int64_t stride) { return out != nullptr ? static_cast<char *>(out) + t * stride * e : nullptr; };
      KhRead8Params p{static_cast<const uint8_t *>(c.k), static_cast<const uint8_t *>(c.v), c.k_scale, c.v_scale, a.slots + t,
                      at(a.k_out, a.k_out_stride), at(a.v_out, a.v_out_stride), a.k_out_stride, a.v_out_stride, c.pages * c.page_size,
                      static_cast<uint32_t>(c.k_page_stride), static_cast<uint32_t>(c.k_slot_stride),
                      static_cast<uint32_t>(c.k_head_stride), static_cast<uint32_t>(c.v_page_stride),
                      static_cast<uint32_t>(c.v_slot_stride), static_cast<uint32_t>(c.v_head_stride),
                      static_cast<uint32_t>(c.scale_page_stride), static_cast<uint32_t>(c.scale_head_stride),
                      static_cast<int32_t>(c.page_size), static_cast<int32_t>(c.kv_heads), static_cast<int32_t>(c.head_dim),
                      static_cast<int32_t>(tokens), static_cast<int32_t>(each), kh_div_by(static_cast<uint32_t>(pieces)),
                      kh_div_by(static_cast<uint32_t>(c.head_dim * e / 16))};
      if (int rc = launch(kRead[a.dtype], ceil_div(tokens, each), 2, 256, p, stream)) return rc;
    }
    return 0;
  });
}

int kh_paged_attention8_workspace(const kh_paged_attention8_args *args, size_t *bytes) {
  const char *op = "paged_attention8_workspace";
  return guarded(op, [&] {
    if (args == nullptr || bytes == nullptr) return bad(op, "null argument");
    if (int rc = check_attention8(op, *args)) return rc;
    *bytes = attention_workspace(as_plain(*args, 0), {2 * KH_GEMM_CUS, most_together(*args)}) + shared_workspace(*args) + kJoinBytes;
    return 0;
  });
}

int kh_paged_attention8(const kh_paged_attention8_args *args, void *workspace, size_t workspace_bytes, void *stream) {
  const char *op = "paged_attention8";
  return guarded(op, [&] {
    if (args == nullptr) return bad(op, "null arguments");
    const kh_paged_attention8_args &a = *args;
    const kh_paged_cache8 &c = a.cache;
    if (int rc = check_attention8(op, a)) return rc;
    if (!aligned(workspace)) return bad(op, "workspace must be 16-byte aligned");
    if (workspace == nullptr) workspace_bytes = 0;
    const void *const written[] = {a.out, a.lse, workspace_bytes > 0 ? workspace : nullptr};
    const void *const read[] = {a.q, c.k, c.v, c.k_scale, c.v_scale, a.table.pages, a.table.lens, a.q_starts};
    for (int i = 0; i < 3; ++i) {
      if (written[i] == nullptr) continue;
      if (std::find(std::begin(read), std::end(read), written[i]) != std::end(read) || std::find(written, written + i, written[i]) != written + i)
        return bad(op, "what is written must not be what is read, or written already");
    }
    const SharedPlan shared = shared_plan(a, workspace_bytes);
    const bool common = shared.splits > 0;
    const kh_paged_attention_args plain = as_plain(a, shared.entries);
    const int64_t group = a.q_heads / c.kv_heads, rows = a.tokens * a.q_heads, d = c.head_dim;
    const bool even = even_pages8(a);
    // What tells who joins which parts comes last.
    size_t left = workspace_bytes - shared.bytes;
    left -= std::min(left, kJoinBytes);
    // Straight to LDS, two workgroups fill a CU's (rows past 128 elements beside wide
    // ones: one).
    const bool narrow_only = kh_narrow_only(a.tokens, a.table.seqs, group, a.max_new, narrow_rows_of(KHRT_BF16), 256);
    const bool alone = even && !common && narrow_only;
    const int64_t together = even ? heads_together(a, shared.entries) : 1;
    const int64_t whole = common ? kWholeShared : alone && d <= 128 ? kWholeEven : kWholeBlocks;
    const AttentionPlan plan = attention_plan(plain, left, {alone ? 2 * KH_GEMM_CUS : most_groups(plain), together, whole});
    const bool joined = plan.part_bytes + plan.wide_bytes > 0;
    // All rows of parts come first, 16 bytes at a time, then their statistics.
    float *at = static_cast<float *>(workspace);
    const auto take = [&at](int64_t floats) { return std::exchange(at, floats > 0 ? at + floats : at); };
    const int64_t narrow_parts = plan.part_bytes > 0 ? plan.groups * 2 * KH_TILE_ROWS * together : 0;
    const int64_t wide_parts = plan.wide_bytes > 0 ? plan.splits * rows : 0;
    const int64_t common_parts = common ? (shared.splits + 1) * rows : 0;
    float *const part_o = take(narrow_parts * d), *const wide_o = take(wide_parts * d), *const shared_o = take(common_parts * d);
    float *const part_ml = take(narrow_parts * 2), *const wide_ml = take(wide_parts * 2), *const shared_ml = take(common_parts * 2);
    const int64_t wide_blocks = plan.wide_units * plan.splits, shared_blocks = shared.units * shared.splits;
    const auto u32 = [](int64_t x) { return static_cast<uint32_t>(x); };
    const auto i32 = [](int64_t x) { return static_cast<int32_t>(x); };
    KhAttention8Params p{};
    p.cache = {.k = static_cast<const char *>(c.k), .v = static_cast<const char *>(c.v),
               .k_page = u32(c.k_page_stride), .k_slot = u32(c.k_slot_stride), .k_head = u32(c.k_head_stride),
               .v_page = u32(c.v_page_stride), .v_slot = u32(c.v_slot_stride), .v_head = u32(c.v_head_stride),
               .pages = i32(c.pages), .page_size = i32(c.page_size), .kv_heads = i32(c.kv_heads), .head_dim = i32(d),
               .by_page = kh_div_by(u32(c.page_size))};
    p.k_scale = c.k_scale, p.v_scale = c.v_scale;
    p.scale_page = u32(c.scale_page_stride), p.scale_head = u32(c.scale_head_stride);
    p.table = device_table(a.table, plain.cache);
    p.q = a.q, p.out = a.out, p.lse = a.lse, p.q_starts = a.q_starts;
    p.q_stride = a.q_stride, p.out_stride = a.out_stride;
    p.tokens = i32(a.tokens), p.q_heads = i32(a.q_heads), p.group = i32(group), p.window = i32(a.window);
    p.by_group = kh_div_by(u32(group));
    p.part_o = part_o, p.part_ml = part_ml, p.wide_o = wide_o, p.wide_ml = wide_ml, p.shared_o = shared_o, p.shared_ml = shared_ml;
    p.joins = reinterpret_cast<KhJoin *>(at);
    p.groups = i32(plan.groups), p.whole = plan.whole, p.narrow_rows = i32(plan.narrow_rows);
    p.wide_blocks = i32(wide_blocks), p.wide_splits = i32(std::max<int64_t>(plan.splits, 1));
    p.shared = i32(shared.entries), p.shared_blocks = i32(shared_blocks);
    p.shared_splits = i32(std::max<int64_t>(shared.splits, 1)), p.shared_each = i32(shared.each);
    p.even = even, p.together = i32(together), p.head_groups = i32(ceil_div(c.kv_heads, together));
    // Scores are masked before the factor: it is above 0, which a scale of 0 makes up
    // for with queries of 0.
    p.scale_log2 = a.scale == 0.0f ? 1.0f : std::fabs(in_powers_of_two(a.scale));
    p.q_keep = a.scale == 0.0f ? 0u : 0xffffffffu;
    p.q_sign = a.scale < 0.0f ? (element_bytes(a.dtype) == 2 ? 0x80008000u : 0x80000000u) : 0u;
    const Cap cap = cap_of(a.cap, p.scale_log2);
    p.cap_in = cap.in, p.cap_out = cap.out;
    p.cap_near = a.dtype == KHRT_F32 || a.cap > 256.0f || (a.window > 0 && a.window <= KH_FEW_CAPPED);
    const int width = width_of(d);
    const auto &symbols = wide_blocks + shared_blocks > 0 ? kWide : alone ? kAttention : kOdd;
    const unsigned threads = alone ? 64u * kWaves[width] : 256u;
    if (int rc = launch(symbols[width][a.dtype], shared_blocks + wide_blocks + plan.groups, 1, threads, p, stream)) return rc;
    if (joined) {
      const int64_t narrow_joins = plan.part_bytes > 0 ? plan.groups * together : 0;
      const int64_t wide_joins = plan.wide_bytes > 0 ? plan.wide_units * (KH_WIDE_ROWS / KH_TILE_ROWS) : 0;
      // Few units of many parts: a workgroup to 32 columns. MI355X, one sequence of
      // 131071 entries (128 parts) 67 us against 72, 64 of 513 to 8192 (two or three)
      // 117 against 109.
      const int64_t units = std::min(a.tokens, a.table.seqs) * c.kv_heads;
      const int64_t columns = plan.groups * together >= 32 * units ? (width == 0 ? 2 : width == 1 ? 4 : 8) : 1;
      if (int rc = launch(kJoin[width][a.dtype], narrow_joins + wide_joins, columns, 256, p, stream)) return rc;
    }
    if (!common) return 0;
    const int64_t each = 256 / (width == 0 ? 16 : width == 1 ? 32 : 64);
    return launch(kCombine[width][a.dtype], ceil_div(rows, each), 1, 256, p, stream);
  });
}

}  // extern "C"
