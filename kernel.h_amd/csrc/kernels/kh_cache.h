// What the kernels that multiply queries with a paged cache share: how a wave
// holds rows of K, walks pages and loads blocks of entries, and how tiles of
// rows lie in LDS. Element types as in kh_elem.h; parameters P have a `cache`
// and a `table` (kh_paged.h).
#pragma once

#include "kh_elem.h"
#include "kh_paged.h"

namespace kh {

// How a wave holds D columns: a row of K in steps of 64 bytes; of V in `count`
// pieces of `piece` elements a lane, 16 lanes covering `span` columns. A block
// is 16 or 32 entries, 32 where its rows are up to 256 bytes (16-bit elements
// need 32 for their products): with K and V in flight, O and Q at most half
// of the registers a lone wave could have.
template <int D>
struct Form {
  static constexpr int bytes = D * (int)sizeof(elem);
  static constexpr int steps = bytes / 64;
  static constexpr int tiles = kWide && bytes > 256 ? 1 : 2;
  static constexpr int keys = 16 * tiles;
  static constexpr int mine = 4 * tiles;  // entries of a lane
  static constexpr int piece = kWide ? 4 : D / 16 < 8 ? D / 16 : 8;
  static constexpr int span = 16 * piece;
  static constexpr int count = D / span;
  static constexpr int words = piece * (int)sizeof(elem) / 4;
};

// Maximum and sum over the four lanes l % 16 + 16 h: their lanes' values swap
// places between rows of 16 lanes and halves of the wave.
__device__ __forceinline__ float over_rows(float v, bool maximum) {
  const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float x = __uint_as_float(a.x), y = __uint_as_float(a.y);
  v = maximum ? fmaxf(x, y) : x + y;
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float z = __uint_as_float(b.x), w = __uint_as_float(b.y);
  return maximum ? fmaxf(z, w) : z + w;
}

// Natural log of a sum of exponentials held as its binary maximum and 2^lift
// times the sum relative to it.
__device__ __forceinline__ float lse_of(float top, float total, float lift) {
  return total == 0.0f ? -__builtin_inff() : (top + (__builtin_amdgcn_logf(total) - lift)) * 0.69314718055994530942f;
}

__device__ __forceinline__ float over_halves(float v, bool maximum) {
  const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  const float z = __uint_as_float(b.x), w = __uint_as_float(b.y);
  return maximum ? fmaxf(z, w) : z + w;
}

// A word of the page table by way of the scalar cache: for an address that is
// the same in all lanes.
__device__ __forceinline__ int scalar_load(const int32_t *p) {
  typedef const int32_t __attribute__((address_space(4))) *constant;
  return *(constant)(uintptr_t)p;
}

// Page and slot of entry `key`, or of one that is there in its place: nobody
// uses what a load then brings, but every load has an address. EVEN (page_size
// a multiple of 16): the 16 entries from a multiple of 16 on lie in one page
// next to each other, key is such a multiple, and everything about its page is
// the same in all lanes.
template <bool EVEN, class P>
__device__ __forceinline__ KhSlot look_up(const P &p, const int32_t *table, int key, int end) {
  const int inside = key < end ? key : EVEN ? (end - 1) & ~15 : end - 1;
  const uint32_t i = kh_div((uint32_t)inside, p.cache.by_page);  // inside < end <= capacity: i is in the row
  return KhSlot{EVEN ? scalar_load(table + i) : table[i], inside - (int)(i * p.cache.by_page.by)};
}

// Where the rows of a block of entries lie. Loads of absent rows go to the
// cache's first page instead of being skipped: a branch round a load would make
// the wave wait for every load in flight where its paths join.
template <int D, bool EVEN>
struct Block {
  KhSlot at[Form<D>::tiles];  // of entry 16 t + l % 16; EVEN: of entry 16 t
  uint32_t present;           // bit k: entry k of the block has a page, and is one of this workgroup's
};

template <int D, bool EVEN, class P>
__device__ __forceinline__ void find(Block<D, EVEN> &b, const P &p, const int32_t *table, int key0, int end, int r) {
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) b.at[t] = look_up<EVEN>(p, table, key0 + 16 * t + (EVEN ? 0 : r), end);
}

// Done apart from find() so that the page numbers have time to arrive.
template <int D, bool EVEN, class P>
__device__ __forceinline__ void settle(Block<D, EVEN> &b, const P &p, int key0, int end, int r) {
  b.present = 0;
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const bool paged = (uint32_t)b.at[t].page < (uint32_t)p.cache.pages;
    if constexpr (EVEN) {
      const int left = end - key0 - 16 * t;
      b.present |= (!paged || left <= 0 ? 0u : left >= 16 ? 0xffffu : (1u << left) - 1) << (16 * t);
      if (!paged) b.at[t].page = 0;
    } else {
      const bool there = key0 + 16 * t + r < end && paged;
      b.present |= ((uint32_t)__builtin_amdgcn_ballot_w64(there) & 0xffffu) << (16 * t);
      if (!there) b.at[t] = KhSlot{0, 0};
    }
  }
}

// Byte `off` of a row, or its first where the row is shorter.
__device__ __forceinline__ uint32_t within(int off, int row_bytes) { return (uint32_t)(off < row_bytes ? off : 0); }

template <int D, bool EVEN, class P>
__device__ __forceinline__ void load_k(u32x4 (&k)[Form<D>::tiles][Form<D>::steps], const Block<D, EVEN> &b,
                                       const P &p, const char *base, int row_bytes, int r, int h) {
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const char *row = base + kh_row(b.at[t], p.cache.k_page, p.cache.k_slot);
#pragma unroll
    for (int c = 0; c < Form<D>::steps; ++c) {
      const uint32_t off = (EVEN ? (uint32_t)r * p.cache.k_slot : 0u) + within(64 * c + 16 * h, row_bytes);
      k[t][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + off));
    }
  }
}

// Bit n: entry key0 + n is one of those seen, n < 64.
__device__ __forceinline__ uint64_t seen_of(const KhSpan &seen, int key0) {
  const int from = kh_clamp(seen.first - key0, 0, 64), to = kh_clamp(seen.end - key0, 0, 64);
  if (from >= to) return 0;
  return (~uint64_t(0) >> (64 - to)) & (~uint64_t(0) << from);
}

// How a tile of D columns lies in LDS: rows one after another, a row's 16-byte
// pieces at their number exclusive-or a number of the row's (k_turn, v_turn), so
// that the reads of it meet no bank twice.
template <int D>
struct Rows {
  static constexpr int bytes = D * (int)sizeof(elem);
  static constexpr int pieces = bytes / 16;
  static constexpr int tile = bytes > 512 ? 32 : 64;     // rows of a tile
  static constexpr int passes = tile * pieces / 256;     // pieces that a thread brings
  static constexpr int per_wave = 64 / pieces;           // rows that a wave brings in a pass
  static constexpr int share = tile / 4;                 // rows that it brings in all, of four waves
};

// What a row's piece numbers are exclusive-ored with: 16 rows of K in a column
// fill the banks once; so do, of V, the pieces that a product's read takes of 4
// rows (16 bits), or of a row and the one 4 below it (32 bits).
template <int D>
__device__ __forceinline__ int k_turn(int row) {
  return Rows<D>::pieces == 8 ? row >> 1 & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_turn(int row) {
  if constexpr (kWide) return (row >> 2 & 1) * 8;
  return Rows<D>::pieces == 8 ? (row >> 1 & 1) * 4 : (row & 3) * 4;
}

// A operand of K for 32 bytes of the rows of tile kt.
template <int D>
__device__ __forceinline__ u32x4 k_rows(const char *buffer, int kt, int c, int lane) {
  using W = Rows<D>;
  const int r = lane & 31;
  return *reinterpret_cast<const u32x4 *>(buffer + (32 * kt + r) * W::bytes + 16 * ((lane >> 5 ^ k_turn<D>(r)) ^ 2 * c));
}

// Asks the scheduler to read `ahead` operands from LDS before the first of
// `products` matrix instructions, and one more behind each: left to itself it
// reads each right before its product, and the wave waits out LDS every time.
template <int READS, int PRODUCTS, int EACH, int AHEAD>
__device__ __forceinline__ void read_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < PRODUCTS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if (AHEAD + i * EACH < READS) __builtin_amdgcn_sched_group_barrier(0x100, EACH, 0);
  }
}

}  // namespace kh
