// Attention of the new tokens of ragged sequences over a paged cache:
//   x_ij = scale q_i . k_j,  j among the entries that token i sees
//   lse_i = log sum_j exp x_ij,  o_i = sum_j exp(x_ij - lse_i) v_j
// The m new tokens of a sequence of n entries are its last m entries; token i
// sees entries up to its own, n - m + i, and with a window only the last
// `window` of those. A row that sees nothing gives o = 0, lse = -inf.
//
// The heads that share a kv head are rows of one product: row R of a (sequence,
// kv head) is token R / group, head R % group, so that a single token of a
// grouped model already fills part of a tile and reads its keys once.
//
// A step's work is cut into equal shares, one to a workgroup (kh_paged.h,
// KhUnits): a share may end inside a sequence, whose parts a second kernel then
// joins. Whatever the lengths, the chip is full until the end: 64 sequences of
// 513 to 8192 entries (bf16, 32 heads on 8 of 128) take 204 us, 5.6 TB/s of K and V,
// against 224 us with each sequence cut into the best number of equal pieces.
//
// Matrix form, per wave: 16 rows against blocks of 32 entries.
//   S^T = K Q^T   A = rows of K as they lie in memory, 64 bytes of a row in a
//                 step; the result's lane l holds row l % 16 and the entries
//                 4 (l / 16) + i of each half block.
//   O^T += V^T P^T  B = those registers; lane l's eight entries are also the
//                 ones whose rows of V it loads, 16 bytes at 8 (l % 16)
//                 elements (so that 16 lanes read a whole row), and swaps
//                 element by element into A. Nothing crosses lanes, and
//                 nothing goes through LDS but the waves' join at the end.
// Products accumulate in 32 bits. P is rounded to the elements' type for the
// second product, the sum of P is not: the rounding is off by half a step of
// that type at most, as the output's is.
//
// Bound by reading K and V: each wave holds a block of both and has the next
// ones in flight (nontemporal: nobody else reads them), 64 KB to a CU. One
// sequence of 131071 entries takes 104 us, 5.2 TB/s.
//
// Rows of V that no row of the tile sees (past the sequence's end, in pages
// that do not exist) count as zeros. Where some rows of the tile see an entry
// and others do not, 0 x V must be 0 also for infinities and NaN in V: see
// poison().
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

using kh::elem;
using kh::f32x4;
using kh::u32x2;
using kh::u32x4;

constexpr int kRows = KH_TILE_ROWS;
constexpr int kWaves = 4;          // waves of a workgroup; they take blocks of entries in turn
constexpr float kNegBig = -1e30f;  // seed of the running maximum: finite, so that max - max is never NaN

// How a wave holds D columns: a row of K in steps of 64 bytes; of V in `count`
// pieces of `piece` elements a lane, 16 lanes covering `span` columns. A block
// is 16 or 32 entries, 32 where its rows are up to 256 bytes (16-bit elements
// need 32 for their products): with K and V in flight, O and Q at most half
// of the registers a lone wave could have.
template <int D>
struct Form {
  static constexpr int bytes = D * (int)sizeof(elem);
  static constexpr int steps = bytes / 64;
  static constexpr int tiles = kh::kWide && bytes > 256 ? 1 : 2;
  static constexpr int keys = 16 * tiles;
  static constexpr int mine = 4 * tiles;  // entries of a lane
  static constexpr int piece = kh::kWide ? 4 : D / 16 < 8 ? D / 16 : 8;
  static constexpr int span = 16 * piece;
  static constexpr int count = D / span;
  static constexpr int words = piece * (int)sizeof(elem) / 4;
};

// The lane's rows of V, one piece of columns.
template <int D>
struct Piece {
  uint32_t w[Form<D>::mine][Form<D>::words];
};

// Which elements of w are of a kind: ones (of the elements' type) in their places.
// kind 0: NaN, 1: +infinity, 2: -infinity.
__device__ __forceinline__ uint32_t marks(uint32_t w, int kind) {
#if KH_ELEM == 0
  const uint32_t magnitude = w & 0x7fffffffu;
  const bool hit = kind == 0 ? magnitude > 0x7f800000u : w == (kind == 1 ? 0x7f800000u : 0xff800000u);
  return hit ? 0x3f800000u : 0u;
#else
  constexpr uint32_t inf = KH_ELEM == 1 ? 0x7c00u : 0x7f80u, one = KH_ELEM == 1 ? 0x3c00u : 0x3f80u;
  uint32_t r = 0;
#pragma unroll
  for (int b = 0; b < 32; b += 16) {
    const uint32_t x = w >> b & 0xffffu;
    const bool hit = kind == 0 ? (x & 0x7fffu) > inf : x == (kind == 1 ? inf : inf | 0x8000u);
    r |= hit ? one << b : 0u;
  }
  return r;
#endif
}

__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
#if KH_ELEM == 0
  return kh::not_finite(w) ? 0u : w;
#else
  w = kh::not_finite(w & 0xffffu) ? w & 0xffff0000u : w;
  return kh::not_finite(w & 0xffff0000u) ? w & 0xffffu : w;
#endif
}

// o += (element e of this piece of V)^T P^T, p[j] for the lane's entry j;
// KIND >= 0: of the marks of that kind instead of the values.
template <int D>
__device__ __forceinline__ f32x4 pv(const Piece<D> &v, int e, const float (&p)[Form<D>::mine], f32x4 o, int kind = -1) {
#if KH_ELEM == 0
#pragma unroll
  for (int j = 0; j < Form<D>::mine; ++j) {
    const uint32_t w = kind < 0 ? v.w[j][e] : marks(v.w[j][e], kind);
    o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w), p[j], o, 0, 0, 0);
  }
  return o;
#else
  u32x4 a, b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = __builtin_amdgcn_perm(v.w[2 * j + 1][e / 2], v.w[2 * j][e / 2], (e & 1) != 0 ? 0x07060302u : 0x05040100u);
    if (kind >= 0) a[j] = marks(a[j], kind);
    b[j] = kh::pack2(p[2 * j], p[2 * j + 1]);
  }
  return kh::mma16(a, b, o);
#endif
}

// Entries with infinities or NaN in V where rows differ in what they see: adds
// to o what those elements give the rows that do see them, and takes them out
// of v (as zeros). Products of 0/1 marks say which rows meet a NaN, +inf or -inf
// in which column; they are exact, and only blocks at a row's limit with such a
// value come here.
template <int D>
__device__ __forceinline__ void poison(Piece<D> &v, const float (&seen)[Form<D>::mine], f32x4 (&o)[Form<D>::piece]) {
#pragma nounroll
  for (int kind = 0; kind < 3; ++kind) {
    const float add = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
    for (int e = 0; e < Form<D>::piece; ++e) {
      const f32x4 met = pv<D>(v, e, seen, f32x4{0, 0, 0, 0}, kind);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[e][i] = met[i] > 0.0f ? o[e][i] + add : o[e][i];
    }
  }
#pragma unroll
  for (int j = 0; j < Form<D>::mine; ++j)
#pragma unroll
    for (int w = 0; w < Form<D>::words; ++w) v.w[j][w] = without_odd(v.w[j][w]);
}

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

// Natural log of a sum of exponentials held as its binary maximum and the
// sum relative to it.
__device__ __forceinline__ float lse_of(float top, float total) {
  return total == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * 0.69314718055994530942f;
}

// Where the rows of a block of entries lie. Loads of absent rows go to the
// cache's first row instead of being skipped: a branch round a load would make
// the wave wait for every load in flight where its paths join.
template <int D>
struct Block {
  KhSlot at[Form<D>::tiles];  // of entry 16 t + l % 16
  uint32_t present;           // bit k: entry k of the block has a page, and is one of this workgroup's
};

template <int D>
__device__ __forceinline__ void find(Block<D> &b, const KhAttentionParams &p, const int32_t *table, int key0, int end, int r) {
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const int key = key0 + 16 * t + r, inside = key < end ? key : end - 1;
    const uint32_t i = kh_div((uint32_t)inside, p.cache.by_page);
    b.at[t].slot = inside - (int)(i * p.cache.by_page.by);
    b.at[t].page = table[i];  // inside < end <= capacity: i is in the row
  }
}

// Done apart from find() so that the page numbers have time to arrive.
template <int D>
__device__ __forceinline__ void settle(Block<D> &b, const KhAttentionParams &p, int key0, int end, int r) {
  b.present = 0;
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const bool there = key0 + 16 * t + r < end && (uint32_t)b.at[t].page < (uint32_t)p.cache.pages;
    b.present |= ((uint32_t)__builtin_amdgcn_ballot_w64(there) & 0xffffu) << (16 * t);
    if (!there) b.at[t] = KhSlot{0, 0};
  }
}

template <int D>
__device__ __forceinline__ void load_k(u32x4 (&k)[Form<D>::tiles][Form<D>::steps], const Block<D> &b, const KhAttentionParams &p,
                                       const char *base, int row_bytes, int h) {
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const char *row = base + kh_row(b.at[t], p.cache.k_page, p.cache.k_slot);
#pragma unroll
    for (int c = 0; c < Form<D>::steps; ++c) {
      const int off = 64 * c + 16 * h;
      k[t][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + (off < row_bytes ? off : 0)));
    }
  }
}

template <int D>
__device__ __forceinline__ void load_v(Piece<D> (&v)[Form<D>::count], const Block<D> &b, const KhAttentionParams &p,
                                       const char *base, int row_bytes, int r, int h) {
  using F = Form<D>;
#pragma unroll
  for (int t = 0; t < F::tiles; ++t) {
    const uint64_t own = kh_row(b.at[t], p.cache.v_page, p.cache.v_slot);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Entry 4 h + i is the one that lane 4 h + i looked up.
      const uint32_t lo = __shfl((uint32_t)own, 4 * h + i, kh::kWave), hi = __shfl((uint32_t)(own >> 32), 4 * h + i, kh::kWave);
      const char *row = base + ((uint64_t)hi << 32 | lo);
#pragma unroll
      for (int a = 0; a < F::count; ++a) {
        const int off = (a * F::span + F::piece * r) * (int)sizeof(elem);
        const char *from = row + (off < row_bytes ? off : 0);
        uint32_t(&w)[F::words] = v[a].w[4 * t + i];
        if constexpr (F::words == 4) {
          const u32x4 g = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from));
          w[0] = g.x, w[1] = g.y, w[2] = g.z, w[3] = g.w;
        } else {
          const u32x2 g = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(from));
          w[0] = g.x, w[1] = g.y;
        }
      }
    }
  }
}

__device__ __forceinline__ KhSeq sequence(const KhAttentionParams &p, int seq) {
  return kh_seq(p.table.lens[seq], p.q_starts[seq], p.q_starts[seq + 1], p.table.capacity, p.tokens);
}

// Sum over the lanes up to this one: within rows of 16 lanes, then each row's
// last lane to the rows behind it.
__device__ __forceinline__ int up_to(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);   // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);   // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);   // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// The step's blocks, and of the first 64 sequences, one to a lane, what they
// are and how many blocks they have.
struct Line {
  KhSeq s;
  int own, upto, all;
};

// Blocks of the lane's sequence; 0 past the last.
__device__ __forceinline__ int work_of(const KhAttentionParams &p, int seq, KhSeq &s) {
  s = KhSeq{0, 0, 0};
  if (seq < p.table.seqs) s = sequence(p, seq);
  return kh_work(kh_units(s, p.group, p.window, p.whole), p.cache.kv_heads);
}

__device__ __forceinline__ Line line_of(const KhAttentionParams &p) {
  const int lane = kh::lane_id();
  Line l;
  l.own = work_of(p, lane, l.s);
  l.upto = up_to(l.own);
  l.all = __builtin_amdgcn_readlane(l.upto, kh::kWave - 1);
  for (int s0 = kh::kWave; s0 < p.table.seqs; s0 += kh::kWave) {
    KhSeq s;
    l.all += __builtin_amdgcn_readlane(up_to(work_of(p, s0 + lane, s)), kh::kWave - 1);
  }
  return l;
}

// The sequence that block x (less than all) is of, and the blocks before that
// sequence.
__device__ __forceinline__ int sequence_at(const KhAttentionParams &p, const Line &l, int x, KhSeq &s, int &before) {
  const int lane = kh::lane_id();
  int own = l.own, upto = l.upto;
  KhSeq mine = l.s;
  for (int s0 = 0;; s0 += kh::kWave) {
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > x);
    if (past != 0) {
      const int first = __builtin_ctzll(past);
      before = __builtin_amdgcn_readlane(upto - own, first);
      s.n = __builtin_amdgcn_readlane(mine.n, first);
      s.m = __builtin_amdgcn_readlane(mine.m, first);
      s.start = __builtin_amdgcn_readlane(mine.start, first);
      return s0 + first;
    }
    const int sum = __builtin_amdgcn_readlane(upto, kh::kWave - 1);
    own = work_of(p, s0 + kh::kWave + lane, mine);
    upto = sum + up_to(own);
  }
}

template <int D>
__device__ __forceinline__ void attention(const KhAttentionParams &p, float *lds) {
  using F = Form<D>;
  const int lane = kh::lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kh::kWave);
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);

  const Line line = line_of(p);
  const KhShares shares = kh_shares(line.all, kh_most(line.all, p.groups));
  if ((int)blockIdx.x >= shares.groups) return;
  const int start = kh_share(shares, (int)blockIdx.x), end = kh_share(shares, (int)blockIdx.x + 1);
  // The join area: each wave's maxima and sums of its rows, what each row's
  // sum is multiplied by, and each wave's part of O.
  float *ml = lds, *inv = lds + kWaves * kRows * 2, *part = inv + kRows;
  constexpr int kPitch = D + 4;
  int before;  // blocks of the sequences before this one
  KhSeq s;
  int seq = sequence_at(p, line, start, s, before);
  KhUnits units = kh_units(s, p.group, p.window, p.whole);

  for (int at = start; at < end;) {
    while (at >= before + kh_work(units, p.cache.kv_heads)) {
      before += kh_work(units, p.cache.kv_heads);
      s = sequence(p, ++seq);
      units = kh_units(s, p.group, p.window, p.whole);
    }
    const uint32_t unit = (uint32_t)(at - before) / (uint32_t)units.blocks;
    const int tile = (int)(unit / (uint32_t)p.cache.kv_heads), head = (int)(unit - (uint32_t)tile * (uint32_t)p.cache.kv_heads);
    const int block0 = at - before - (int)unit * units.blocks;
    const int block1 = end - at < units.blocks - block0 ? block0 + end - at : units.blocks;
    const bool alone = block0 == 0 && block1 == units.blocks;
    const int slot = at == start ? 0 : 1;
    at += block1 - block0;
    const int from = units.first + block0 * KH_STRETCH, to = block1 == units.blocks ? s.n : units.first + block1 * KH_STRETCH;
    const int rows = s.m * p.group;  // < 2^31: tokens x q_heads is
    const int row0 = tile * kRows;
    const int32_t *table = p.table.pages + seq * p.table.row_stride;
    const char *kbase = p.cache.k + (uint64_t)head * p.cache.k_head;
    const char *vbase = p.cache.v + (uint64_t)head * p.cache.v_head;

    const int R = row0 + r;
    const bool mine = R < rows;
    const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
    const int i_first = (int)kh_div(row0, p.by_group);
    const int i_last = (int)kh_div(row0 + kRows < rows ? row0 + kRows - 1 : rows - 1, p.by_group);
    const KhSpan seen = kh_seen(s, i, p.window);
    const KhSpan low = kh_seen(s, i_first, p.window), high = kh_seen(s, i_last, p.window);
    const int key_first = low.first > from ? low.first : from;
    const int key_end = high.end < to ? high.end : to;

    u32x4 q[F::steps];
    const elem *qp = static_cast<const elem *>(p.q) + (int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d;
#pragma unroll
    for (int c = 0; c < F::steps; ++c) {
      q[c] = u32x4{0, 0, 0, 0};
      if (mine && 64 * c + 16 * h < row_bytes) q[c] = *reinterpret_cast<const u32x4 *>(qp + (64 * c + 16 * h) / (int)sizeof(elem));
    }

    float m = kNegBig, l = 0.0f;  // of row l % 16; l of this lane's entries alone
    f32x4 o[F::count][F::piece];
#pragma unroll
    for (int a = 0; a < F::count; ++a)
#pragma unroll
      for (int e = 0; e < F::piece; ++e) o[a][e] = f32x4{0, 0, 0, 0};

    // K and V are a block ahead of their use, the page numbers two: K's next
    // block goes out as soon as the scores have taken its registers' content,
    // V's when the products have.
    int key0 = key_first + wave * F::keys;
    if (key0 < key_end) {
      constexpr int kStep = kWaves * F::keys;
      u32x4 k[F::tiles][F::steps];
      Piece<D> v[F::count];
      Block<D> now, next;
      find<D>(now, p, table, key0, key_end, r);
      find<D>(next, p, table, key0 + kStep, key_end, r);
      settle<D>(now, p, key0, key_end, r);
      load_k<D>(k, now, p, kbase, row_bytes, h);
      load_v<D>(v, now, p, vbase, row_bytes, r, h);
      for (; key0 < key_end; key0 += kStep) {
        const uint32_t present = now.present;
        float y[F::mine];
        if (d != D) {
          // Columns past the row's end were read from its start.
#pragma unroll
          for (int c = 0; c < F::steps; ++c)
            if (64 * c + 16 * h >= row_bytes) {
#pragma unroll
              for (int t = 0; t < F::tiles; ++t) k[t][c] = u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int t = 0; t < F::tiles; ++t) {
          f32x4 x = {0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < F::steps; ++c) x = kh::mma16(k[t][c], q[c], x);
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * t + e] = x[e] * p.scale_log2;
        }
        now = next;
        settle<D>(now, p, key0 + kStep, key_end, r);
        load_k<D>(k, now, p, kbase, row_bytes, h);
        find<D>(next, p, table, key0 + 2 * kStep, key_end, r);

        // Every row sees every entry of the block: no mask.
        const bool whole = present == (F::keys == 32 ? 0xffffffffu : 0xffffu) && key0 + F::keys <= low.end && key0 >= high.first;
        float on[F::mine];
        bool odd = false;
        if (!whole) {
#pragma unroll
          for (int j = 0; j < F::mine; ++j) {
            const int n = 16 * (j / 4) + 4 * h + j % 4, key = key0 + n;
            const bool there = (present >> n & 1) != 0;
            const bool sees = mine && key >= seen.first && key < seen.end && there;
            on[j] = sees ? 1.0f : 0.0f;
            y[j] = sees ? y[j] : -__builtin_inff();
#pragma unroll
            for (int a = 0; a < F::count; ++a)
#pragma unroll
              for (int w = 0; w < F::words; ++w) {
                v[a].w[j][w] = there ? v[a].w[j][w] : 0u;
                odd |= kh::not_finite(v[a].w[j][w]);
              }
          }
        }
        float top = y[0];
#pragma unroll
        for (int j = 1; j < F::mine; ++j) top = fmaxf(top, y[j]);
        top = fmaxf(m, over_rows(top, true));
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float fade = kh::exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int a = 0; a < F::count; ++a)
#pragma unroll
            for (int e = 0; e < F::piece; ++e) o[a][e] *= fade;
        }
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < F::mine; ++j) {
          y[j] = kh::exp2_hw(y[j] - m);
          sum += y[j];
        }
        l += sum;
        // After the fading: an infinity does not survive a factor of zero.
        if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll
          for (int a = 0; a < F::count; ++a) poison<D>(v[a], on, o[a]);
        }
#pragma unroll
        for (int a = 0; a < F::count; ++a)
#pragma unroll
          for (int e = 0; e < F::piece; ++e) o[a][e] = pv<D>(v[a], e, y, o[a][e]);
        load_v<D>(v, now, p, vbase, row_bytes, r, h);
      }
    }

    // Join the waves: rescale to the rows' common maximum, add in wave order.
    l = over_rows(l, false);
    if (h == 0) {
      ml[(wave * kRows + r) * 2] = m;
      ml[(wave * kRows + r) * 2 + 1] = l;
    }
    kh::lds_barrier();
    float top = kNegBig;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * kRows + r) * 2]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += ml[(w * kRows + r) * 2 + 1] * kh::exp2_hw(ml[(w * kRows + r) * 2] - top);
    const float fade = kh::exp2_hw(m - top);
#pragma unroll
    for (int a = 0; a < F::count; ++a)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
        for (int e = 0; e < F::piece; ++e)
          part[(wave * kRows + r) * kPitch + a * F::span + F::piece * (4 * h + i4) + e] = o[a][e][i4] * fade;
    const int64_t row_of = (int64_t)(s.start + i) * p.q_heads + hq;  // this lane's row
    if (wave == 0 && h == 0) {
      inv[r] = alone ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
      if (mine && alone && p.lse != nullptr) p.lse[row_of] = lse_of(top, total);
      if (!alone) {
        float *ml_to = p.part_ml + ((int64_t)blockIdx.x * 2 + slot) * kRows * 2 + r * 2;
        ml_to[0] = top;
        ml_to[1] = total;
      }
    }
    kh::lds_barrier();
    for (int x = threadIdx.x; x < kRows * (D / 4); x += kWaves * kh::kWave) {
      const int row = x / (D / 4), col = x % (D / 4) * 4, RR = row0 + row;
      if (RR >= rows || col >= d) continue;
      const int ii = (int)kh_div(RR, p.by_group), hh = head * p.group + RR - ii * p.group;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += part[(w * kRows + row) * kPitch + col + e];
        y[e] = sum * inv[row];
      }
      if (alone) {
        kh::store4(static_cast<elem *>(p.out) + (int64_t)(s.start + ii) * p.out_stride + (int64_t)hh * d + col, y);
      } else {
        float *o_to = p.part_o + (((int64_t)blockIdx.x * 2 + slot) * kRows + row) * d + col;
        *reinterpret_cast<f32x4 *>(o_to) = f32x4{y[0], y[1], y[2], y[3]};
      }
    }
    kh::lds_barrier();  // before the next unit writes the join area
  }
}

// Joins the parts of units that several workgroups worked on: a workgroup per
// row, its waves taking the parts in turn. `lds` holds kWaves x 256 + kWaves floats.
__device__ __forceinline__ void join(const KhAttentionParams &p, float *lds) {
  constexpr int kMost = 256;
  const int lane = kh::lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kh::kWave);
  const int token = (int)(blockIdx.x / (uint32_t)p.q_heads), hq = (int)(blockIdx.x % (uint32_t)p.q_heads);
  // The token's sequence, the blocks before it and all blocks. Tokens of no
  // sequence have no parts.
  int work = 0, before = -1;
  KhSeq s{0, 0, 0};
  for (int s0 = 0; s0 < p.table.seqs; s0 += kh::kWave) {
    KhSeq mine;
    const int own = work_of(p, s0 + lane, mine), upto = up_to(own);
    const uint64_t here = __builtin_amdgcn_ballot_w64(token >= mine.start && token - mine.start < mine.m);
    if (here != 0) {
      const int first = __builtin_ctzll(here);
      before = work + __builtin_amdgcn_readlane(upto - own, first);
      s.n = __builtin_amdgcn_readlane(mine.n, first);
      s.m = __builtin_amdgcn_readlane(mine.m, first);
      s.start = __builtin_amdgcn_readlane(mine.start, first);
    }
    work += __builtin_amdgcn_readlane(upto, kh::kWave - 1);
  }
  if (before < 0) return;
  const KhUnits units = kh_units(s, p.group, p.window, p.whole);
  const int head = hq / p.group, R = (token - s.start) * p.group + hq - head * p.group, tile = R / kRows;
  const int begin = before + (tile * p.cache.kv_heads + head) * units.blocks, end = begin + units.blocks;
  const KhShares shares = kh_shares(work, kh_most(work, p.groups));
  const int g0 = kh_owner(shares, begin), g1 = kh_owner(shares, end - 1);
  if (g0 == g1) return;  // one workgroup had the whole unit
  // The first part ends its workgroup's share unless that began in this unit;
  // all others begin theirs.
  const int slot0 = kh_share(shares, g0) >= begin ? 0 : 1;
  const int64_t row = R - tile * kRows;
  auto place = [&](int g) { return ((int64_t)g * 2 + (g == g0 ? slot0 : 0)) * kRows + row; };
  float top = kNegBig;
  for (int g = g0 + lane; g <= g1; g += kh::kWave) top = fmaxf(top, p.part_ml[place(g) * 2]);
  top = kh::wave_max(top);
  const int d = p.cache.head_dim;
  f32x4 o = {0, 0, 0, 0};
  float total = 0.0f;
  const bool live = 4 * lane < d;
#pragma unroll 4
  for (int g = g0 + wave; g <= g1; g += kWaves) {
    const int64_t at = place(g);
    const float w = kh::exp2_hw(p.part_ml[at * 2] - top);
    total += p.part_ml[at * 2 + 1] * w;
    if (live) o += *reinterpret_cast<const f32x4 *>(p.part_o + at * d + 4 * lane) * w;
  }
  if (live) *reinterpret_cast<f32x4 *>(lds + wave * kMost + 4 * lane) = o;
  float *sums = lds + kWaves * kMost;
  if (lane == 0) sums[wave] = total;
  kh::lds_barrier();
  if (wave != 0) return;
  total = sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) {
    total += sums[w];
    if (live) o += *reinterpret_cast<const f32x4 *>(lds + w * kMost + 4 * lane);
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (live) {
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    kh::store4(static_cast<elem *>(p.out) + (int64_t)token * p.out_stride + (int64_t)hq * d + 4 * lane, y);
  }
  if (lane == 0 && p.lse != nullptr) p.lse[blockIdx.x] = lse_of(top, total);
}

}  // namespace

// Two workgroups to a CU, so that one's loads are in flight while the other
// multiplies; a wave of the widest rows needs the registers of both.
#define KH_ATTENTION(D)                                                                                     \
  extern "C" __global__ void __launch_bounds__(256, D > 128 ? 1 : 2) KH_TYPED(paged_attention_##D)(const KhAttentionParams p) { \
    __shared__ float lds[kWaves * kRows * 2 + kRows + kWaves * kRows * (D + 4)];                             \
    attention<D>(p, lds);                                                                                    \
  }
KH_ATTENTION(64)
KH_ATTENTION(128)
KH_ATTENTION(256)
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_attention_join)(const KhAttentionParams p) {
  __shared__ __attribute__((aligned(16))) float lds[kWaves * 256 + kWaves];
  join(p, lds);
}
