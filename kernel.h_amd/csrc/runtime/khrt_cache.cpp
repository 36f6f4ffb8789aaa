// The sequence-cache operators behind the C-ABI (khrt.h, group 8): the checks
// of what the host can see, the launch geometry, and the kernels' parameters.
#include "kernelh/khrt_cache.hpp"

using namespace khrt::cache;

namespace {

// Code objects and symbols by element type.
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
    *bytes = attention_workspace(*args, {most_groups(*args)});
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
    const AttentionPlan plan = attention_plan(a, workspace != nullptr ? workspace_bytes : 0, {most_groups(a)});
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
