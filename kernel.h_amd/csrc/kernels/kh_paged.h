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

// A cache and the page table over it. Byte e of head h of the entry in slot t
// of page p: k + p k_page + t k_slot + h k_head + e (v alike). Strides are in
// bytes and below 2^32, so that one multiply-add per stride forms the 64-bit
// address: a cache may pass 4 GB, a page may not.
struct KhCache {
  const char *k, *v;
  uint32_t k_page, k_slot, k_head, v_page, v_slot, v_head;
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

// Where the row of that entry starts, past the cache's (and head's) own start.
KH_HD uint64_t kh_row(const KhSlot &s, uint32_t page_stride, uint32_t slot_stride) {
  return static_cast<uint64_t>(static_cast<uint32_t>(s.page)) * page_stride +
         static_cast<uint64_t>(static_cast<uint32_t>(s.slot)) * slot_stride;
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

// The token and the head of its group that row R of a sequence and kv head is.
// A row past the last gives row 0's in its place: what is read there exists and
// is not used. A sequence without new tokens has no row at all, its start may lie
// behind the last token, and nothing may be read for it: token -1.
struct KhQuery {
  int32_t token, head;
};

KH_HD KhQuery kh_query(const KhSeq &s, int32_t group, const KhDiv &by_group, int32_t R) {
  if (s.m == 0) return KhQuery{-1, 0};
  const int32_t real = R < s.m * group ? R : 0, i = static_cast<int32_t>(kh_div(static_cast<uint32_t>(real), by_group));
  return KhQuery{s.start + i, real - i * group};
}

// Of entries [first, end) of the sequence, how many are not its new tokens'.
KH_HD int32_t kh_older(const KhSeq &s, int32_t first, int32_t end) {
  const int32_t older = s.n - s.m < end ? s.n - s.m : end;  // may lie below 0
  return older > first ? older - first : 0;
}

// How paged_attention's narrow form shares out a step. A unit is 16 rows (new
// tokens x heads of a group) of one sequence and kv head against `blocks`
// stretches of KH_STRETCH entries, all that any of the sequence's new tokens
// sees; `whole` makes a unit one indivisible block. The units of all
// sequences, those of a sequence in the order of tiles and heads, follow each
// other in one line of blocks, of which every workgroup gets an equal share:
// however lengths differ, all workgroups are done together.
#define KH_STRETCH 128
#define KH_TILE_ROWS 16

struct KhUnits {
  int32_t first;   // the first entry that any new token sees, down to a multiple of 16
  int32_t blocks;  // of each unit, at least 1: rows that see nothing are written too
  int32_t tiles;   // 0 without new tokens
};

KH_HD KhUnits kh_units(const KhSeq &s, int32_t group, int32_t window, int32_t whole) {
  KhUnits u;
  u.first = kh_seen(s, 0, window).first & ~15;  // the first token's window starts earliest
  const int32_t keys = s.n > u.first ? s.n - u.first : 0;
  u.blocks = whole != 0 || keys == 0 ? 1 : (keys - 1) / KH_STRETCH + 1;
  u.tiles = s.m == 0 ? 0 : (s.m * group - 1) / KH_TILE_ROWS + 1;
  return u;
}

// Blocks of a sequence. The launcher sees to it that all sequences' together
// stay below 2^30 (it makes units whole where they might not).
KH_HD int32_t kh_work(const KhUnits &u, int32_t kv_heads) { return u.tiles * kv_heads * u.blocks; }

// The share of each of at most `most` workgroups: `each` blocks, one more for the
// first `longer` of them. Every one of them gets a block at least, so that each
// part of a unit is one that somebody wrote.
struct KhShares {
  int32_t groups, each, longer;
};

// Of the two workgroups a CU can hold, one does better where each would get a
// single block, and where shares are long (its loads alone fill the memory's
// queues): MI355X, bf16 heads of 128, one workgroup against two, 64 x 4096
// entries 183 us / 193, 1 x 131071 104 / 110, 8 x 1024 16.4 / 18.5; the other way
// 128 x 512 66 / 59, 32 sequences of up to 2000 56 / 45.
#define KH_CUS 256
KH_HD int32_t kh_most(int32_t work, int32_t groups) {
  return (work <= 2 * KH_CUS || work >= 32 * KH_CUS) && groups > KH_CUS ? KH_CUS : groups;
}

KH_HD KhShares kh_shares(int32_t work, int32_t most) {
  KhShares s;
  s.groups = work < most ? work : most;
  s.each = s.groups > 0 ? static_cast<int32_t>(static_cast<uint32_t>(work) / static_cast<uint32_t>(s.groups)) : 0;
  s.longer = work - s.each * s.groups;
  return s;
}

// Walks from unit to unit and from sequence to sequence count from the start
// of the sequence they are in, `in` blocks: what came before may be past 32 bits
// where starts do not ascend and many sequences claim the same tokens. Whether
// block `in` lies behind the sequence's `work` blocks; if so, it is counted from
// there.
KH_HD bool kh_passed(int32_t &in, int32_t work) {
  if (in < work) return false;
  in -= work;
  return true;
}

// Where workgroup g's share starts.
KH_HD int32_t kh_share(const KhShares &s, int32_t g) { return g * s.each + (g < s.longer ? g : s.longer); }

// The workgroup whose share holds block x.
KH_HD int32_t kh_owner(const KhShares &s, int32_t x) {
  const int32_t long_ones = s.longer * (s.each + 1);
  return x < long_ones ? static_cast<int32_t>(static_cast<uint32_t>(x) / static_cast<uint32_t>(s.each + 1))
                       : s.longer + static_cast<int32_t>(static_cast<uint32_t>(x - long_ones) / static_cast<uint32_t>(s.each));
}

// The workgroups that have parts of the unit of `blocks` blocks from block
// `begin` on, of `work` in all. Where counts have passed 32 bits a unit may begin
// before the line's first block or end behind its last: there are no parts there.
// slot: of the first of them, 0 where its share begins in this unit, else 1;
// all others begin theirs in it.
struct KhOwners {
  int32_t first, count, slot;
};

KH_HD KhOwners kh_owners(const KhShares &s, int32_t work, int32_t begin, int32_t blocks) {
  const int64_t end = static_cast<int64_t>(begin) + blocks;
  KhOwners o;
  o.first = kh_owner(s, begin > 0 ? begin : 0);
  o.count = kh_owner(s, static_cast<int32_t>(end < work ? end : work) - 1) - o.first + 1;
  o.slot = kh_share(s, o.first) >= begin ? 0 : 1;
  return o;
}

// Whether a step goes to the narrow form alone, by what the host can know: `few`
// rows to a sequence on the whole, and `most` at the most in one of them. new: the
// most new tokens of a sequence as the caller expects, 0 if it does not say; then
// every sequence is taken to have one at least. A long chunk among single tokens
// would read its entries once for every 16 rows; one that is not there costs the
// launch's idle wide workgroups. MI355X, bf16, 32 heads on 8 of 128, 2000 entries
// each, narrow alone against both: 127 single tokens and a chunk of 33 186 us / 202,
// 64 198 / 200, 128 218 / 202, 512 344 / 203, 896 443 / 212; 64 sequences of 5
// tokens 179 / 184. fp32: a chunk of 128 397 / 414, 256 475 / 408, 896 816 / 568.
// One sequence: whichever form suits its rows.
KH_HD bool kh_narrow_only(int64_t tokens, int64_t seqs, int64_t group, int64_t max_new, int64_t few, int64_t most) {
  if (tokens * group > few * seqs) return false;
  const int64_t left = tokens > seqs ? tokens - seqs + 1 : 1;
  const int64_t longest = max_new > 0 && max_new < tokens ? max_new : max_new > 0 ? tokens : left;
  return longest * group <= (seqs == 1 ? few : most);
}

// The wide form: units of KH_WIDE_ROWS rows of a sequence of more than
// narrow_rows rows and a kv head, each with the entries that its own rows see,
// in up to `splits` parts of whole tiles where units are few.
#define KH_WIDE_ROWS 128

KH_HD int32_t kh_wide_tiles(const KhSeq &s, int32_t group) { return s.m == 0 ? 0 : (s.m * group - 1) / KH_WIDE_ROWS + 1; }

struct KhPart {
  int32_t first, end, used;
};

// Part `split` of entries [first, end): at least 256 entries each but for the
// last, whole tiles of 64.
KH_HD KhPart kh_part(int32_t first, int32_t end, int32_t splits, int32_t split) {
  const int32_t keys = end > first ? end - first : 0;
  KhPart r;
  int32_t each = (keys - 1) / splits / 64 * 64 + 64;
  if (keys == 0 || each < 256) each = 256;
  r.used = keys == 0 ? 1 : (keys - 1) / each + 1;
  r.first = split < r.used ? first + split * each : end;
  r.end = split < r.used - 1 ? r.first + each : end;
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
  // Parts of units that several workgroups work on: [groups][2][rows][head_dim]
  // and, behind them, [groups][2][rows][2] (maximum, sum). Slot 0 is of the
  // unit in which a workgroup's share starts, slot 1 of the one it ends in.
  float *part_o, *part_ml;
  // Parts of the wide units' rows: [wide_splits][tokens q_heads][head_dim] and [..][2].
  float *wide_o, *wide_ml;
  int64_t q_stride, out_stride;
  int32_t tokens, q_heads, group, window, groups, whole;
  int32_t narrow_rows;  // a sequence of more rows is the wide form's
  int32_t wide_blocks, wide_splits;
  int32_t even;  // pages hold a multiple of 16 entries, rows apart, and 16 slots' strides fit 31 bits
  uint32_t q_keep, q_sign;  // q's bits that count (none with a scale of 0); the sign bits where the scale is negative
  KhDiv by_group;
  float scale_log2;  // |scale| log2(e), above 0: maxima may be taken before it
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
  int32_t chunk_keys, chunks, even;  // of a workgroup, a multiple of KH_STRETCH; that the launch has; KhAttentionParams
  int32_t steady;  // 32 rows are whole tokens, and no two tokens of q share bytes
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
  int32_t lanes, chunks;  // paged_evict_move: lanes to a row, workgroups to a sequence
  int32_t heads_inner;    // the heads of an entry lie nearer than its neighbours
  KhDiv by_heads;
};
