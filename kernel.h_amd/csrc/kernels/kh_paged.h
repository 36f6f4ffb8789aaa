// Paged caches of keys and values: the parameters of the kernels over them
// and the index arithmetic that the launcher, the kernels and the CPU checks
// share. Plain C++: included by device and host translation units alike.
//
// Everything that comes from device memory (page numbers, lengths, the
// starts of the sequences' new tokens) is brought into range here before it
// becomes an address: the host never sees it and cannot refuse it.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__) || defined(__HIP__)
#define KH_HD __host__ __device__ __forceinline__
#else
#define KH_HD inline
#endif

// Division of j < 2^31 by a divisor of the launch, as a multiplication. With
// 2^s < by <= 2^(s+1) and mul = 2^(32+s) / by + e, 0 <= e < 1, the product is
// j mul / 2^(32+s) = j / by + j e / 2^(32+s), and j by < 2^(32+s) keeps the last
// term below 1 / by: it never reaches the next quotient. by = 1 has no such
// mul below 2^32 and is marked by mul = 0.
struct KhDiv {
  uint32_t mul, shift, by;
};

KH_HD KhDiv kh_div_by(uint32_t by) {
  KhDiv d{0, 0, by};
  if (by <= 1) return d;
  while ((uint64_t(2) << d.shift) < by) ++d.shift;
  d.mul = static_cast<uint32_t>(((uint64_t(1) << (32 + d.shift)) + by - 1) / by);
  return d;
}

KH_HD uint32_t kh_div(uint32_t j, const KhDiv &d) {
  return d.mul == 0 ? j : static_cast<uint32_t>((static_cast<uint64_t>(j) * d.mul) >> 32) >> d.shift;
}

// A cache and the page table over it. Element e of head h of the entry in
// slot t of page p: k + p k_page + t k_slot + h k_head + e (v alike), strides
// in elements and 64 bits wide: a cache may pass 2^31 elements.
struct KhCache {
  const void *k, *v;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int32_t pages, page_size, kv_heads, head_dim;
  KhDiv by_page;
};

struct KhTable {
  const int32_t *pages;  // [seqs, width]
  const int32_t *lens;   // [seqs]
  int64_t row_stride;
  int32_t seqs, width, capacity;  // capacity: entries a row of the table can hold
};

struct KhSlot {
  int32_t page, slot;  // page < 0: the entry has none
};

// Where entry j of the sequence whose table row is `row` lies.
KH_HD KhSlot kh_slot(const int32_t *row, int32_t width, int32_t pages, const KhDiv &by_page, uint32_t j) {
  const uint32_t i = kh_div(j, by_page);
  KhSlot s;
  s.slot = static_cast<int32_t>(j - i * by_page.by);
  s.page = i < static_cast<uint32_t>(width) ? row[i] : -1;
  if (s.page >= pages) s.page = -1;
  return s;
}

// A sequence's share of a step: entries in the cache, new tokens (the last
// of those entries) and the first of them.
struct KhSeq {
  int32_t n, m, start;
};

KH_HD int32_t kh_clamp(int32_t x, int32_t lo, int32_t hi) { return x < lo ? lo : x > hi ? hi : x; }

KH_HD KhSeq kh_seq(int32_t len, int32_t start, int32_t end, int32_t capacity, int32_t tokens) {
  KhSeq s;
  s.n = kh_clamp(len, 0, capacity);
  s.start = kh_clamp(start, 0, tokens);
  const int32_t e = kh_clamp(end, 0, tokens);
  s.m = e > s.start ? e - s.start : 0;
  return s;
}

// Entries that the new token in place i sees: [first, end), end <= n. Empty
// (first >= end) for a token that lies before the cache's first entry, as
// where a sequence has fewer entries than new tokens.
struct KhSpan {
  int32_t first, end;
};

KH_HD KhSpan kh_seen(const KhSeq &s, int32_t i, int32_t window) {
  KhSpan r;
  r.end = s.n - s.m + i + 1;
  r.first = window > 0 && r.end > window ? r.end - window : 0;
  return r;
}

// The part of a sequence's entries that workgroups share out: all that any of
// its new tokens sees, in chunks of `split_keys`, the last of which takes
// whatever is left past splits * split_keys.
struct KhSplit {
  int32_t first, end, used;
};

KH_HD KhSplit kh_split(const KhSeq &s, int32_t window, int32_t splits, int32_t split_keys, int32_t split) {
  const KhSpan all = kh_seen(s, 0, window);  // the first token's window starts earliest
  const int32_t first = all.first;
  const int32_t keys = s.n > first ? s.n - first : 0;
  KhSplit r;
  r.used = keys == 0 ? 1 : (keys - 1) / split_keys + 1;
  if (r.used > splits) r.used = splits;
  if (split >= r.used) {
    r.first = r.end = s.n;
    return r;
  }
  r.first = first + split * split_keys;
  r.end = split == r.used - 1 ? s.n : r.first + split_keys;
  return r;
}

// qk_norm_rope.hip
struct KhRopeParams {
  const void *q, *k, *v;
  void *q_out, *k_out;
  const void *q_gamma, *k_gamma;
  const float *inv_freq;
  const int64_t *positions, *slots;
  void *k_cache, *v_cache;
  int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int64_t rows;  // slots of the cache: pages * page_size
  int32_t page_size;
  int32_t tokens, q_heads, kv_heads, head_dim, rotary, interleaved, norm, parts;
  float eps;
};

// paged_attention.hip
struct KhAttentionParams {
  KhCache cache;
  KhTable table;
  const void *q;
  void *out;
  float *lse;  // may be null
  const int32_t *q_starts;
  float *part_ml, *part_o;  // splits > 1: [splits][tokens q_heads][2] and [..][head_dim]
  int64_t q_stride, out_stride;
  int32_t tokens, q_heads, group, window, splits, split_keys;
  KhDiv by_group;
  float scale_log2;
};

// paged_weights.hip
struct KhWeightsParams {
  KhCache cache;
  KhTable table;
  const void *q;
  const float *lse;
  const int32_t *q_starts;
  const float *weights_in;  // may be null
  float *weights;
  int64_t q_stride, seq_stride, head_stride;
  int32_t tokens, q_heads, group, window;
  KhDiv by_group;
  float scale_log2;
};

// paged_evict.hip
struct KhEvictParams {
  KhCache cache;
  KhTable table;
  const int32_t *kept_pages;
  int32_t *kept_lens;
  const float *weights_in;
  float *weights;
  int32_t *chosen;  // [seqs][kv_heads][budget]
  int64_t kept_row_stride, in_seq_stride, in_head_stride, seq_stride, head_stride;
  int32_t kept_width, budget, recent, element;
};
