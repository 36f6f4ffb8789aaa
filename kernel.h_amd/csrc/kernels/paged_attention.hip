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
// 513 to 8192 entries (bf16, 32 heads on 8 of 128) take 199 us, 5.7 TB/s of K and V,
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
// that type at most, as the output's is. fp16 ends soon below one, so there P and
// its sums are 2^15 times their value (kLift): entries a 2^25th of the largest, of
// which a long cache may hold many, would be in the sum alone.
//
// Bound by reading K and V: each wave holds a block of both and has the next
// ones in flight (nontemporal: nobody else reads them), 64 KB to a CU. One
// sequence of 131071 entries takes 103 us, 5.2 TB/s.
//
// Rows of V that no row of the tile sees (past the sequence's end, in pages
// that do not exist) count as zeros. Where some rows of the tile see an entry
// and others do not, infinities and NaN in V are kept out of the products and
// added to the rows that do see them.
#include "kh_cache.h"

namespace {

using namespace kh;
using kh::elem;
using kh::f32x16;
using kh::f32x4;
using kh::u32x2;
using kh::u32x4;

constexpr int kRows = KH_TILE_ROWS;
constexpr int kWaves = 4;          // waves of a workgroup; they take blocks of entries in turn
constexpr float kSeed = -3.402823466e38f;  // of the running maximum: no finite score lies below it, and max - max is never NaN
constexpr float kLift = KH_ELEM == 1 ? 15.0f : 0.0f;  // fp16 holds 2^kLift times what the largest score can be off by (2^0.25)
constexpr float kFine = 4194304.0f;        // 2^22, see coarse()

// The lane's rows of V, one piece of columns.
template <int D>
struct Piece {
  uint32_t w[Form<D>::mine][Form<D>::words];
};

// w with zeros for infinities and NaN.
__device__ __forceinline__ uint32_t without_odd(uint32_t w) {
#if KH_ELEM == 0
  return kh::not_finite(w) ? 0u : w;
#else
  w = kh::not_finite(w & 0xffffu) ? w & 0xffff0000u : w;
  return kh::not_finite(w & 0xffff0000u) ? w & 0xffffu : w;
#endif
}

// o += (element e of this piece of V)^T P^T, p[j] for the lane's entry j.
template <int D>
__device__ __forceinline__ f32x4 pv(const Piece<D> &v, int e, const float (&p)[Form<D>::mine], f32x4 o) {
#if KH_ELEM == 0
#pragma unroll
  for (int j = 0; j < Form<D>::mine; ++j)
    o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v.w[j][e]), p[j], o, 0, 0, 0);
  return o;
#else
  u32x4 a, b;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    a[j] = __builtin_amdgcn_perm(v.w[2 * j + 1][e / 2], v.w[2 * j][e / 2], (e & 1) != 0 ? 0x07060302u : 0x05040100u);
    b[j] = kh::pack2(p[2 * j], p[2 * j + 1]);
  }
  return kh::mma16(a, b, o);
#endif
}

// Four elements of a row of V, zeros but for infinities and NaN.
__device__ __forceinline__ f32x4 odd_of(const char *at) {
  float x[4];
  kh::load4(x, reinterpret_cast<const elem *>(at));
  f32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = (__float_as_uint(x[i]) & 0x7fffffffu) >= 0x7f800000u ? x[i] : 0.0f;
  return y;
}

template <int D, bool EVEN>
__device__ __forceinline__ void load_v(Piece<D> (&v)[Form<D>::count], const Block<D, EVEN> &b, const KhAttentionParams &p,
                                       const char *base, int row_bytes, int r, int h) {
  using F = Form<D>;
#pragma unroll
  for (int t = 0; t < F::tiles; ++t) {
    const uint64_t own = kh_row(b.at[t], p.cache.v_page, p.cache.v_slot);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const char *row = base + own;
      if constexpr (!EVEN) {
        // Entry 4 h + i is the one that lane 4 h + i looked up.
        const uint32_t lo = __shfl((uint32_t)own, 4 * h + i, kh::kWave), hi = __shfl((uint32_t)(own >> 32), 4 * h + i, kh::kWave);
        row = base + ((uint64_t)hi << 32 | lo);
      }
#pragma unroll
      for (int a = 0; a < F::count; ++a) {
        const char *from = row + ((EVEN ? (uint32_t)(4 * h + i) * p.cache.v_slot : 0u) +
                                  within((a * F::span + F::piece * r) * (int)sizeof(elem), row_bytes));
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

// h, worked out where it is used: on a path that is hardly ever taken, what
// follows from it is not to be kept in registers across the loop round it.
__device__ __forceinline__ int apart(int h) {
  asm volatile("" : "+v"(h));
  return h;
}

// 2^x takes scores times a factor less the row's maximum m (in powers of two) and
// more kLift:
// one multiply-add, exact but for its last rounding, while m itself was rounded.
// The largest score is so off by half a step of m: 2^-2 at kFine, whole powers of
// two further up. Where the wave has such maxima (coarse), the products are
// rounded as m was before it is taken from them (less), and nothing else is done.
__device__ __forceinline__ bool coarse(float m) { return __builtin_amdgcn_ballot_w64(__builtin_fabsf(m) > kFine) != 0; }

template <int N, class X>
__device__ __forceinline__ void less(X &x, float factor, float m) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float y = x[j] * factor;
    asm volatile("" : "+v"(y));  // not fused with the subtraction
    x[j] = y - m;
  }
}

__device__ __forceinline__ KhSeq sequence(const KhAttentionParams &p, int seq) {
  return kh_seq(p.table.lens[seq], p.q_starts[seq], p.q_starts[seq + 1], p.table.capacity, p.tokens);
}

// The step's blocks, and of the first 64 sequences, one to a lane, what they
// are and how many blocks they have.
struct Line {
  KhSeq s;
  int own, upto, all;
};

// Blocks of the lane's sequence, or units where `wide`; 0 past the last.
__device__ __forceinline__ int work_of(const KhAttentionParams &p, int seq, bool wide, KhSeq &s) {
  s = KhSeq{0, 0, 0};
  if (seq < p.table.seqs) s = sequence(p, seq);
  const bool is_wide = s.m * p.group > p.narrow_rows;
  if (is_wide != wide) return 0;
  return wide ? kh_wide_tiles(s, p.group) * p.cache.kv_heads
              : kh_work(kh_units(s, p.group, p.window, p.whole), p.cache.kv_heads);
}

__device__ __forceinline__ Line line_of(const KhAttentionParams &p, bool wide) {
  const int lane = kh::lane_id();
  Line l;
  l.own = work_of(p, lane, wide, l.s);
  l.upto = up_to(l.own);
  l.all = __builtin_amdgcn_readlane(l.upto, kh::kWave - 1);
  for (int s0 = kh::kWave; s0 < p.table.seqs; s0 += kh::kWave) {
    KhSeq s;
    l.all += __builtin_amdgcn_readlane(up_to(work_of(p, s0 + lane, wide, s)), kh::kWave - 1);
  }
  return l;
}

// The sequence that block x (less than all) is of, and the blocks before that
// sequence. -1 if there is none: starts that do not ascend can make the counts
// wrap, and every walk over the sequences ends at the last one all the same.
__device__ __forceinline__ int sequence_at(const KhAttentionParams &p, const Line &l, int x, bool wide, KhSeq &s, int &before) {
  const int lane = kh::lane_id();
  int own = l.own, upto = l.upto;
  KhSeq mine = l.s;
  for (int s0 = 0; s0 < p.table.seqs; s0 += kh::kWave) {
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
    own = work_of(p, s0 + kh::kWave + lane, wide, mine);
    upto = sum + up_to(own);
  }
  return -1;
}

// Behind a launch's wide workgroups one to a CU cannot be had: where the idle ones
// of them leave first, two of the others come to lie on one CU beside empty ones.
__device__ __forceinline__ KhShares shares_of(const KhAttentionParams &p, const Line &line) {
  return kh_shares(line.all, p.wide_blocks > 0 ? p.groups : kh_most(line.all, p.groups));
}

template <int D, bool EVEN>
__device__ __forceinline__ void narrow(const KhAttentionParams &p, int block, float *lds) {
  using F = Form<D>;
  const int lane = kh::lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kh::kWave);
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);

  const Line line = line_of(p, false);
  const KhShares shares = shares_of(p, line);
  if (block >= shares.groups) return;
  const int start = kh_share(shares, block), end = kh_share(shares, block + 1);
  // The join area: each wave's maxima and sums of its rows, what each row's
  // sum is multiplied by, and each wave's part of O.
  float *ml = lds, *inv = lds + kWaves * kRows * 2, *part = inv + kRows;
  constexpr int kPitch = D + 4;
  int before;  // blocks of the sequences before this one
  KhSeq s;
  int seq = sequence_at(p, line, start, false, s, before);
  if (seq < 0) return;
  KhUnits units = kh_units(s, p.group, p.window, p.whole);

  for (int at = start, in = start - before; at < end;) {
    while (kh_passed(in, kh_work(units, p.cache.kv_heads))) {
      // The next sequence of few rows: wide() has the others.
      do {
        if (++seq >= p.table.seqs) return;
        s = sequence(p, seq);
      } while (s.m * p.group > p.narrow_rows);
      units = kh_units(s, p.group, p.window, p.whole);
    }
    const uint32_t unit = (uint32_t)in / (uint32_t)units.blocks;
    const int tile = (int)(unit / (uint32_t)p.cache.kv_heads), head = (int)(unit - (uint32_t)tile * (uint32_t)p.cache.kv_heads);
    const int block0 = in - (int)unit * units.blocks;
    const int block1 = end - at < units.blocks - block0 ? block0 + end - at : units.blocks;
    const bool alone = block0 == 0 && block1 == units.blocks;
    const int slot = at == start ? 0 : 1;
    at += block1 - block0, in += block1 - block0;
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
    const int key_first = (low.first > from ? low.first : from) & ~15;  // from is a multiple of 16
    const int key_end = high.end < to ? high.end : to;

    u32x4 q[F::steps];
    const char *qp = static_cast<const char *>(p.q) + ((int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d) * (int)sizeof(elem);
#pragma unroll
    for (int c = 0; c < F::steps; ++c) {
      // From an address that is there in any case, as the rows of K and V.
      const u32x4 x = *reinterpret_cast<const u32x4 *>(qp + within(64 * c + 16 * h, row_bytes)) & p.q_keep ^ p.q_sign;
      q[c] = mine && 64 * c + 16 * h < row_bytes ? x : u32x4{0, 0, 0, 0};
    }

    // Of row l % 16; l of this lane's entries alone. A row that there is none of has
    // no scores, and no maximum to look after either.
    float m = mine ? kSeed : 0.0f, l = 0.0f;
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
      Block<D, EVEN> now, next;
      find<D, EVEN>(now, p, table, key0, key_end, r);
      find<D, EVEN>(next, p, table, key0 + kStep, key_end, r);
      settle<D, EVEN>(now, p, key0, key_end, r);
      load_k<D, EVEN>(k, now, p, kbase, row_bytes, r, h);
      // K goes out before V here as in the loop: the wait for K at its top then
      // leaves V in flight.
      __builtin_amdgcn_sched_barrier(0);
      load_v<D, EVEN>(v, now, p, vbase, row_bytes, r, h);
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
          for (int e = 0; e < 4; ++e) y[4 * t + e] = x[e];
        }
        now = next;
        settle<D, EVEN>(now, p, key0 + kStep, key_end, r);
        load_k<D, EVEN>(k, now, p, kbase, row_bytes, r, h);
        find<D, EVEN>(next, p, table, key0 + 2 * kStep, key_end, r);

        // Every row sees every entry of the block: no mask.
        const bool whole = present == (F::keys == 32 ? 0xffffffffu : 0xffffu) && key0 + F::keys <= low.end && key0 >= high.first;
        uint32_t odds = 0;  // bit n: entry n of the block, in this lane's columns
        if (!whole) {
          // Of the lane's entries: those that its row sees, and those that are there.
          const uint32_t sees = (mine ? (uint32_t)seen_of(seen, key0) & present : 0u) >> 4 * h, there = present >> 4 * h;
#pragma unroll
          for (int j = 0; j < F::mine; ++j) {
            const uint32_t bit = 1u << (16 * (j / 4) + j % 4);
            y[j] = (sees & bit) != 0 ? y[j] : -__builtin_inff();
#pragma unroll
            for (int a = 0; a < F::count; ++a)
#pragma unroll
              for (int w = 0; w < F::words; ++w) {
                v[a].w[j][w] = (there & bit) != 0 ? v[a].w[j][w] : 0u;
                odds |= kh::not_finite(v[a].w[j][w]) ? bit : 0u;
              }
          }
          odds <<= 4 * h;
        }
        float top = y[0];
#pragma unroll
        for (int j = 1; j < F::mine; ++j) top = fmaxf(top, y[j]);
        top = fmaxf(m, over_rows(top, true) * p.scale_log2);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float fade = kh::exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int a = 0; a < F::count; ++a)
#pragma unroll
            for (int e = 0; e < F::piece; ++e) o[a][e] *= fade;
        }
        const bool far = coarse(m);
        const float factor = far ? 1.0f : p.scale_log2, shift = far ? kLift : kLift - m;
        if (far) less<F::mine>(y, p.scale_log2, m);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < F::mine; ++j) {
          y[j] = kh::exp2_hw(fmaf(y[j], factor, shift));
          sum += y[j];
        }
        l += sum;
        if (__builtin_amdgcn_ballot_w64(odds != 0) != 0) {
          // Infinities and NaN in V where rows differ in what they see: 0 x V would
          // reach the rows that do not. They leave the products as zeros and are
          // added, read once more, to the rows that do see them (after the
          // fading: an infinity does not survive a factor of zero).
          for (int n = 0; n < F::keys; ++n) {
            if (__builtin_amdgcn_ballot_w64((odds >> n & 1) != 0) == 0) continue;
            const int key = key0 + n;
            const KhSlot at = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)key);
            const char *row = vbase + kh_row(at, p.cache.v_page, p.cache.v_slot);
            if (mine && key >= seen.first && key < seen.end) {
              const int h1 = apart(h);
#pragma unroll
              for (int a = 0; a < F::count; ++a)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
                  for (int e = 0; e < F::piece; e += 4) {
                    const int col = a * F::span + F::piece * (4 * h1 + i4) + e;
                    if (col >= d) continue;
                    const f32x4 x = odd_of(row + col * (int)sizeof(elem));
#pragma unroll
                    for (int b = 0; b < 4; ++b) o[a][e + b][i4] += x[b];
                  }
            }
          }
          // Its loads end here: one that the compiler took for still on its way would
          // have the common path wait for all, the next block among them.
          kh::vm_wait<0>();
#pragma unroll
          for (int a = 0; a < F::count; ++a)
#pragma unroll
            for (int j = 0; j < F::mine; ++j)
#pragma unroll
              for (int w = 0; w < F::words; ++w) v[a].w[j][w] = without_odd(v[a].w[j][w]);
        }
#pragma unroll
        for (int a = 0; a < F::count; ++a)
#pragma unroll
          for (int e = 0; e < F::piece; ++e) o[a][e] = pv<D>(v[a], e, y, o[a][e]);
        load_v<D, EVEN>(v, now, p, vbase, row_bytes, r, h);
      }
    }

    // Join the waves: rescale to the rows' common maximum, add in wave order.
    l = over_rows(l, false);
    if (h == 0) {
      ml[(wave * kRows + r) * 2] = m;
      ml[(wave * kRows + r) * 2 + 1] = l;
    }
    kh::lds_barrier();
    float top = kSeed;
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
      if (mine && alone && p.lse != nullptr) p.lse[row_of] = lse_of(top, total, kLift);
      if (!alone) {
        float *ml_to = p.part_ml + ((int64_t)block * 2 + slot) * kRows * 2 + r * 2;
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
        float *o_to = p.part_o + (((int64_t)block * 2 + slot) * kRows + row) * d + col;
        *reinterpret_cast<f32x4 *>(o_to) = f32x4{y[0], y[1], y[2], y[3]};
      }
    }
    kh::lds_barrier();  // before the next unit writes the join area
  }
}

// ---- many rows: chunks of prompts
//
// A workgroup takes 128 rows, 32 to a wave, of one sequence and kv head, and
// brings tiles of K and V through LDS for all of them, a tile ahead. Per wave
//   S^T = K Q^T     32 x 32 tiles, A = rows of K from LDS, B = Q in registers
//   O^T += V^T P^T  B = S^T's registers as they are, A = V read across its rows
//                   (16 bits), or row by row (32 bits, one row to a product)
// with the running maximum and sum of row l % 32 in lanes l and l ^ 32.
//
// Tiles of pages of a multiple of 16 entries go straight to LDS (a wave's load
// brings whole rows of one page; its resource ends where the page's entries
// do, so that absent rows and columns past the row's end arrive as zeros);
// others through registers. A row's 16-byte pieces lie at their number
// exclusive-or a number of the row's, so that neither kind of read meets a bank
// twice (measured: no conflicts).
//
// A wave does a tile's two products and the softmax between them one after the
// other, with two waves to a SIMD to fill each other's gaps: the matrix units are
// busy for 96 us of the 277 to 281 (271 to 308 from one card to another) that 2048
// new tokens of 8192 entries take (bf16, 32 heads on 8 of 128), 865 TFLOP/s. A large
// library product reaches 1228.
template <int D>
struct Wide {
  static constexpr int bytes = D * (int)sizeof(elem);
  static constexpr int steps = bytes / 32;
  static constexpr int keys = Rows<D>::tile;  // entries of a tile
  static constexpr int tiles = keys / 32, runs = keys / 16;
  static constexpr int dts = D / 32;
  static constexpr int pieces = Rows<D>::pieces, passes = Rows<D>::passes, rows = Rows<D>::per_wave, share = Rows<D>::share;
  static constexpr int v_at = keys * bytes, marks_at = 2 * v_at, buffer = marks_at + keys;
  static constexpr int lds = 2 * buffer;
};
constexpr int kWideRows = 32;                  // of a wave
constexpr int kWideTile = kWaves * kWideRows;  // of a workgroup

// The first row that the wave brings in pass i.
template <int D>
__device__ __forceinline__ int first_row(int i, int wave) {
  return wave * Wide<D>::share + i * Wide<D>::rows;
}

constexpr uint8_t kThere = 1, kOdd = 2;  // marks of a row in LDS

// A tile on its way. EVEN: lane n has found run n % runs.
template <int D, bool EVEN>
struct Stage {
  KhSlot at[EVEN ? 1 : Wide<D>::passes];
  u32x4 k[EVEN ? 1 : Wide<D>::passes], v[EVEN ? 1 : Wide<D>::passes];
};

template <int D, bool EVEN>
__device__ __forceinline__ void seek(Stage<D, EVEN> &g, const KhAttentionParams &p, const int32_t *table, int key0, int end, int lane, int wave) {
  using W = Wide<D>;
  if constexpr (EVEN) {
    const int key = key0 + 16 * (lane % W::runs), last = (end - 1) & ~15;
    const uint32_t inside = (uint32_t)(key < last ? key : last), i = kh_div(inside, p.cache.by_page);
    g.at[0] = KhSlot{table[i], (int)(inside - i * p.cache.by_page.by)};
  } else {
#pragma unroll
    for (int i = 0; i < W::passes; ++i)
      g.at[i] = look_up<false>(p, table, key0 + first_row<D>(i, wave) + lane / W::pieces, end);
  }
}

// What a lane brings of a row of K and of V in each pass: where from, past the
// wave's first row.
template <int D>
struct Lanes {
  uint32_t k[Wide<D>::passes], v[Wide<D>::passes];
};

template <int D>
__device__ __forceinline__ Lanes<D> lanes_of(const KhAttentionParams &p, int row_bytes, int lane, int wave) {
  using W = Wide<D>;
  Lanes<D> l;
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const int own = i * W::rows + lane / W::pieces, row = wave * W::share + own;
    const int kc = 16 * (lane % W::pieces ^ k_turn<D>(row)), vc = 16 * (lane % W::pieces ^ v_turn<D>(row));
    l.k[i] = kc < row_bytes ? (uint32_t)own * p.cache.k_slot + (uint32_t)kc : kh::kOutside;
    l.v[i] = vc < row_bytes ? (uint32_t)own * p.cache.v_slot + (uint32_t)vc : kh::kOutside;
  }
  return l;
}

// Sends a tile's rows to LDS, and says which entries are there.
template <int D>
__device__ __forceinline__ uint64_t send(const Stage<D, true> &g, const Lanes<D> &l, const KhAttentionParams &p, const char *kbase,
                                         const char *vbase, int key0, int end, const char *buffer, int wave) {
  using W = Wide<D>;
  // Runs with a page; of a run past the end the last one's was found.
  const uint32_t paged = (uint32_t)__builtin_amdgcn_ballot_w64((uint32_t)g.at[0].page < (uint32_t)p.cache.pages);
  const int left = end - key0;
  uint64_t present = W::keys == 64 ? ~uint64_t(0) : (uint64_t(1) << W::keys % 64) - 1;
  if ((paged & ((1u << W::runs) - 1)) != (1u << W::runs) - 1 || left < W::keys) {
    present = left <= 0 ? 0 : left < W::keys ? (uint64_t(1) << left) - 1 : present;
#pragma unroll
    for (int n = 0; n < W::runs; ++n)
      if ((paged >> n & 1) == 0) present &= ~(uint64_t(0xffff) << (16 * n));
  }
  const int row = wave * W::share, run = row / 16;
  KhSlot at = {__builtin_amdgcn_readlane(g.at[0].page, run), __builtin_amdgcn_readlane(g.at[0].slot, run) + (row & 15)};
  if ((paged >> run & 1) == 0) at.page = 0;
  const uint32_t real = (uint32_t)__builtin_popcountll(present >> row & ((uint64_t(1) << W::share) - 1));
  const uint64_t k = (uint64_t)reinterpret_cast<uintptr_t>(kbase) + kh_row(at, p.cache.k_page, p.cache.k_slot);
  const uint64_t v = (uint64_t)reinterpret_cast<uintptr_t>(vbase) + kh_row(at, p.cache.v_page, p.cache.v_slot);
  // Addresses have 48 bits: the resource's stride, above them, is zero.
  const u32x4 rk = {(uint32_t)k, (uint32_t)(k >> 32), real * p.cache.k_slot, 0x00020000u};
  const u32x4 rv = {(uint32_t)v, (uint32_t)(v >> 32), real * p.cache.v_slot, 0x00020000u};
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(buffer) + (uint32_t)(row * W::bytes);
#pragma unroll
  for (int i = 0; i < W::passes; ++i) kh::dma16(rk, l.k[i], lds + (uint32_t)(i * W::rows * W::bytes));
#pragma unroll
  for (int i = 0; i < W::passes; ++i) kh::dma16(rv, l.v[i], lds + (uint32_t)(W::v_at + i * W::rows * W::bytes));
  return present;
}

// Starts a tile's loads into registers.
template <int D>
__device__ __forceinline__ void fetch(Stage<D, false> &g, const KhAttentionParams &p, const char *kbase, const char *vbase, int key0,
                                      int end, int row_bytes, int lane, int wave) {
  using W = Wide<D>;
  const int own = lane / W::pieces;
  const uint32_t off = within(16 * (lane % W::pieces), row_bytes);
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    if (key0 + first_row<D>(i, wave) + own >= end || (uint32_t)g.at[i].page >= (uint32_t)p.cache.pages) g.at[i] = KhSlot{-1, 0};
    const KhSlot at = g.at[i].page < 0 ? KhSlot{0, 0} : g.at[i];
    g.k[i] = *reinterpret_cast<const u32x4 *>(kbase + kh_row(at, p.cache.k_page, p.cache.k_slot) + off);
    g.v[i] = *reinterpret_cast<const u32x4 *>(vbase + kh_row(at, p.cache.v_page, p.cache.v_slot) + off);
  }
}

// From registers to LDS, with zeros for absent rows and columns past the row's
// end. The lane that brought a row's first piece marks the row.
template <int D>
__device__ __forceinline__ void put(const Stage<D, false> &g, char *buffer, int row_bytes, int lane, int wave) {
  using W = Wide<D>;
  const int own = lane / W::pieces, piece = lane % W::pieces;
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const int row = first_row<D>(i, wave) + own;
    const bool there = g.at[i].page >= 0, real = there && 16 * piece < row_bytes;
    const u32x4 zero = {0, 0, 0, 0};
    *reinterpret_cast<u32x4 *>(buffer + row * W::bytes + 16 * (piece ^ k_turn<D>(row))) = real ? g.k[i] : zero;
    *reinterpret_cast<u32x4 *>(buffer + W::v_at + row * W::bytes + 16 * (piece ^ v_turn<D>(row))) = real ? g.v[i] : zero;
    if (piece == 0) buffer[W::marks_at + row] = there ? kThere : 0;
  }
}

// In a tile of which rows of the unit see different entries: takes infinities
// and NaN out of V and marks the rows that had some. Between barriers.
template <int D>
__device__ __forceinline__ void clean(char *buffer, int lane, int wave) {
  using W = Wide<D>;
  const int own = lane / W::pieces, piece = lane % W::pieces;
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const int row = first_row<D>(i, wave) + own;
    u32x4 *at = reinterpret_cast<u32x4 *>(buffer + W::v_at + row * W::bytes + 16 * piece);
    const u32x4 v = *at;
    const bool odd = kh::not_finite(v.x) | kh::not_finite(v.y) | kh::not_finite(v.z) | kh::not_finite(v.w);
    const uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
    if (odd) *at = u32x4{without_odd(v.x), without_odd(v.y), without_odd(v.z), without_odd(v.w)};
    const uint64_t lanes = W::pieces == 64 ? ~uint64_t(0) : ((uint64_t(1) << W::pieces % 64) - 1) << (own * W::pieces);
    if (piece == 0) {
      uint8_t *mark = reinterpret_cast<uint8_t *>(buffer + W::marks_at + row);
      *mark = (uint8_t)((*mark & kThere) | ((odds & lanes) != 0 ? kOdd : 0));
    }
  }
}

// A operand of V^T for columns 32 dt .. and the entries that step c of tile kt's
// scores hold (16 bits: half a tile, 32 bits: a quarter).
template <int D>
__device__ __forceinline__ u32x4 v_across(const char *buffer, int kt, int c, int dt, int lane) {
  using W = Wide<D>;
  u32x4 a = {0, 0, 0, 0};
#if KH_ELEM == 0
  // Four products, of registers 4 c .. + 3 of the scores.
  const int h = lane >> 5, x = lane & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = *reinterpret_cast<const uint32_t *>(buffer + W::v_at + (32 * kt + 8 * c + 4 * h + i) * W::bytes + 128 * (dt ^ h) + 4 * x);
#else
  const int r = (lane & 15) / 4, turn = W::pieces == 8 ? r >> 1 : r;
  const char *at = buffer + W::v_at + (32 * kt + 16 * c + 4 * (lane >> 5) + r) * W::bytes + 64 * (dt ^ turn) + 32 * (lane >> 4 & 1) +
                   8 * (lane & 3);
  const u32x2 lo = kh::read_across(at), hi = kh::read_across(at + 8 * W::bytes);
  a = u32x4{lo.x, lo.y, hi.x, hi.y};
#endif
  return a;
}

// B operand of P^T for that step.
__device__ __forceinline__ u32x4 p_of(const f32x16 &s, int c) {
#if KH_ELEM == 0
  return u32x4{__float_as_uint(s[4 * c]), __float_as_uint(s[4 * c + 1]), __float_as_uint(s[4 * c + 2]), __float_as_uint(s[4 * c + 3])};
#else
  return u32x4{kh::pack2(s[8 * c], s[8 * c + 1]), kh::pack2(s[8 * c + 2], s[8 * c + 3]), kh::pack2(s[8 * c + 4], s[8 * c + 5]),
               kh::pack2(s[8 * c + 6], s[8 * c + 7])};
#endif
}
constexpr int kPvSteps = kh::kWide ? 4 : 2;  // of a 32-entry tile

// A wide unit: its rows and all entries that any of them sees. A sequence's units
// go from its last tile on: with causal rows the longest first.
struct WideUnit {
  int head, tile0, tile_end, first, end;
};

__device__ __forceinline__ WideUnit wide_unit(const KhAttentionParams &p, const KhSeq &s, int in_seq) {
  const int rows = s.m * p.group, turn = in_seq / p.cache.kv_heads;
  WideUnit u;
  u.head = in_seq - turn * p.cache.kv_heads;
  u.tile0 = (kh_wide_tiles(s, p.group) - 1 - turn) * kWideTile;
  u.tile_end = u.tile0 + kWideTile < rows ? u.tile0 + kWideTile : rows;
  u.first = kh_seen(s, (int)kh_div(u.tile0, p.by_group), p.window).first & ~15;
  u.end = kh_seen(s, (int)kh_div(u.tile_end - 1, p.by_group), p.window).end;
  return u;
}

template <int D, bool EVEN>
__device__ __forceinline__ void wide(const KhAttentionParams &p, int block, char *lds) {
  using W = Wide<D>;
  const int tid = threadIdx.x, lane = kh::lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kh::kWave);
  const int r = lane & 31, h = lane >> 5;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);
  const int split = block % p.wide_splits, unit = block / p.wide_splits;
  KhSeq s;
  int before;
  const Line line = line_of(p, true);
  if (unit >= line.all) return;
  const int seq = sequence_at(p, line, unit, true, s, before);
  if (seq < 0) return;
  const WideUnit u = wide_unit(p, s, unit - before);
  const KhPart part = kh_part(u.first, u.end, p.wide_splits, split);
  if (split >= part.used) return;

  const int rows = u.tile_end, head = u.head;
  const int row0 = u.tile0 + wave * kWideRows, R = row0 + r;
  const bool mine = R < rows;
  const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
  const int last_row = row0 + kWideRows < rows ? row0 + kWideRows - 1 : rows - 1;
  const bool any = row0 < rows;
  const KhSpan seen = kh_seen(s, i, p.window);
  const KhSpan low = kh_seen(s, any ? (int)kh_div(row0, p.by_group) : 0, p.window);
  const KhSpan high = kh_seen(s, any ? (int)kh_div(last_row, p.by_group) : 0, p.window);
  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const char *kbase = p.cache.k + (uint64_t)head * p.cache.k_head;
  const char *vbase = p.cache.v + (uint64_t)head * p.cache.v_head;

  u32x4 q[W::steps];
  const char *qp = static_cast<const char *>(p.q) + ((int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d) * (int)sizeof(elem);
#pragma unroll
  for (int c = 0; c < W::steps; ++c) {
    const u32x4 x = *reinterpret_cast<const u32x4 *>(qp + within(32 * c + 16 * h, row_bytes)) & p.q_keep ^ p.q_sign;
    q[c] = mine && 32 * c + 16 * h < row_bytes ? x : u32x4{0, 0, 0, 0};
  }
  float m = mine ? kSeed : 0.0f, l = 0.0f;
  f32x16 o[W::dts];
#pragma unroll
  for (int a = 0; a < W::dts; ++a) o[a] = f32x16{};

  // Whether rows of the unit differ in what they see of the tile at key0.
  const int all_end = kh_seen(s, (int)kh_div(u.tile0, p.by_group), p.window).end;
  const int all_first = kh_seen(s, (int)kh_div(u.tile_end - 1, p.by_group), p.window).first;
  auto mixed = [&](int key0) { return key0 + W::keys > all_end || key0 < all_first; };
  if (part.first < part.end) {
    Stage<D, EVEN> g;
    uint64_t here = 0, next = 0;  // entries that are there, of this tile and the next
    seek<D, EVEN>(g, p, table, part.first, part.end, lane, wave);
    Lanes<D> lanes;
    if constexpr (EVEN) {
      lanes = lanes_of<D>(p, row_bytes, lane, wave);
      next = send<D>(g, lanes, p, kbase, vbase, part.first, part.end, lds, wave);
      seek<D, EVEN>(g, p, table, part.first + W::keys, part.end, lane, wave);
    } else {
      fetch<D>(g, p, kbase, vbase, part.first, part.end, row_bytes, lane, wave);
    }
    int cur = 0;
    for (int key0 = part.first; key0 < part.end; key0 += W::keys, cur ^= 1) {
      char *buffer = lds + cur * W::buffer;
      here = next;
      // One barrier: this tile is there for everyone, and everyone is done with
      // the tile whose place the next one takes.
      if constexpr (EVEN) {
        kh::vm_wait<0>();
        kh::lds_barrier();
        if (mixed(key0)) {
          clean<D>(buffer, lane, wave);
          kh::lds_barrier();
        }
        // The page numbers of the tile after that go out first: whoever waits for
        // them does not wait for the tile.
        const Stage<D, EVEN> found = g;
        seek<D, EVEN>(g, p, table, key0 + 2 * W::keys, part.end, lane, wave);
        next = send<D>(found, lanes, p, kbase, vbase, key0 + W::keys, part.end, lds + (cur ^ 1) * W::buffer, wave);
      } else {
        put<D>(g, buffer, row_bytes, lane, wave);
        seek<D, EVEN>(g, p, table, key0 + W::keys, part.end, lane, wave);
        fetch<D>(g, p, kbase, vbase, key0 + W::keys, part.end, row_bytes, lane, wave);
        kh::lds_barrier();
        if (mixed(key0)) {
          clean<D>(buffer, lane, wave);
          kh::lds_barrier();
        }
      }
      // Nothing to do for a wave none of whose rows sees any of the tile.
      if (any && key0 < high.end && key0 + W::keys > low.first) {
        f32x16 x[W::tiles];
#pragma unroll
        for (int kt = 0; kt < W::tiles; ++kt) x[kt] = f32x16{};
#pragma unroll
        for (int c = 0; c < W::steps; ++c)
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) x[kt] = kh::mma32(k_rows<D>(buffer, kt, c, lane), q[c], x[kt]);
        if constexpr (!kh::kWide) read_ahead<W::steps * W::tiles, W::steps * W::tiles, 1, 6>();
        uint64_t present = here, odds = 0;
        if constexpr (EVEN) present |= W::keys == 64 ? 0 : ~uint64_t(0) << W::keys % 64;
        if (!EVEN || mixed(key0)) {
          const uint32_t mark = lane < W::keys ? (uint8_t)buffer[W::marks_at + lane] : kThere;
          if (!EVEN) present = __builtin_amdgcn_ballot_w64((mark & kThere) != 0);
          if (mixed(key0)) odds = __builtin_amdgcn_ballot_w64((mark & kOdd) != 0);
        }
        const bool whole = present == ~uint64_t(0) && key0 + W::keys <= low.end && key0 >= high.first;
        if (!whole) {
          const uint64_t sees = mine ? seen_of(seen, key0) & present : 0;
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) {
            const uint32_t own = (uint32_t)(sees >> 32 * kt) >> 4 * h;
#pragma unroll
            for (int j = 0; j < 16; ++j) x[kt][j] = (own >> (8 * (j / 4) + j % 4) & 1) != 0 ? x[kt][j] : -__builtin_inff();
          }
        }
        float top = x[0][0];
#pragma unroll
        for (int kt = 0; kt < W::tiles; ++kt)
#pragma unroll
          for (int j = 0; j < 16; ++j) top = fmaxf(top, x[kt][j]);
        top = fmaxf(m, over_halves(top, true) * p.scale_log2);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float fade = kh::exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int a = 0; a < W::dts; ++a) o[a] *= fade;
        }
        const bool far = coarse(m);
        const float factor = far ? 1.0f : p.scale_log2, shift = far ? kLift : kLift - m;
        if (far) {
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) less<16>(x[kt], p.scale_log2, m);
        }
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < W::tiles; ++kt)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            x[kt][j] = kh::exp2_hw(fmaf(x[kt][j], factor, shift));
            sum += x[kt][j];
          }
        l += sum;
        // As in narrow(): what was kept out of the products.
        for (uint64_t left = odds; left != 0; left &= left - 1) {
          const int key = key0 + __builtin_ctzll(left);
          const KhSlot at = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)key);
          const char *row = vbase + kh_row(at, p.cache.v_page, p.cache.v_slot);
          if (mine && key >= seen.first && key < seen.end) {
            const int h1 = apart(h);
#pragma unroll
            for (int dt = 0; dt < W::dts; ++dt)
#pragma unroll
              for (int j = 0; j < 16; j += 4) {
                const int col = 32 * dt + 2 * j + 4 * h1;
                if (col >= d) continue;
                const f32x4 y = odd_of(row + col * (int)sizeof(elem));
#pragma unroll
                for (int b = 0; b < 4; ++b) o[dt][j + b] += y[b];
              }
          }
        }
        // Operands of V are read a step ahead of their products.
        constexpr int kAll = W::tiles * kPvSteps;
        u32x4 a[2][W::dts];
#pragma unroll
        for (int dt = 0; dt < W::dts; ++dt) a[0][dt] = v_across<D>(buffer, 0, 0, dt, lane);
#pragma unroll
        for (int n = 0; n < kAll; ++n) {
          if (n + 1 < kAll) {
#pragma unroll
            for (int dt = 0; dt < W::dts; ++dt) a[(n + 1) % 2][dt] = v_across<D>(buffer, (n + 1) / kPvSteps, (n + 1) % kPvSteps, dt, lane);
          }
          __builtin_amdgcn_sched_barrier(0);
          const u32x4 b = p_of(x[n / kPvSteps], n % kPvSteps);
#pragma unroll
          for (int dt = 0; dt < W::dts; ++dt) o[dt] = kh::mma32(a[n % 2][dt], b, o[dt]);
        }
      }
    }
  }

  kh::vm_wait<0>();  // nothing is on its way to LDS that the workgroup may give back
  const float total = over_halves(l, false);
  if (!mine) return;
  const int64_t row = (int64_t)(s.start + i) * p.q_heads + hq;
  const bool alone = part.used == 1;
  const int64_t at_row = (int64_t)split * p.tokens * p.q_heads + row;
  if (h == 0) {
    if (alone) {
      if (p.lse != nullptr) p.lse[row] = lse_of(m, total, kLift);
    } else {
      p.wide_ml[at_row * 2] = m;
      p.wide_ml[at_row * 2 + 1] = total;
    }
  }
  const float inv = !alone ? 1.0f : total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int dt = 0; dt < W::dts; ++dt)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int col = 32 * dt + 2 * j + 4 * h;
      if (col >= d) continue;
      const float y[4] = {o[dt][j] * inv, o[dt][j + 1] * inv, o[dt][j + 2] * inv, o[dt][j + 3] * inv};
      if (alone)
        kh::store4(static_cast<elem *>(p.out) + (int64_t)(s.start + i) * p.out_stride + (int64_t)hq * d + col, y);
      else
        *reinterpret_cast<f32x4 *>(p.wide_o + at_row * d + col) = f32x4{y[0], y[1], y[2], y[3]};
    }
}

// Up to 16 rows whose parts several workgroups have: row x of part k is at
// place base(k) + x of the parts' arrays (narrow), or base(k) + the row's own
// place among all rows (wide).
struct Parts {
  const float *ml, *o;
  int64_t first, others, step;  // base of part 0, of part 1, and from there on
  int count;
  int R0, rows;  // the rows of the sequence that they are
  int head;
  bool wide;
};

// The unit that workgroup g's share starts inside of, if it is the first to do
// so: every unit of the narrow form in parts has one such.
__device__ __forceinline__ bool narrow_parts(const KhAttentionParams &p, int g, KhSeq &s, Parts &parts) {
  const Line line = line_of(p, false);
  const KhShares shares = shares_of(p, line);
  if (g == 0 || g >= shares.groups) return false;
  const int at = kh_share(shares, g);
  int before;
  if (sequence_at(p, line, at, false, s, before) < 0) return false;
  const KhUnits units = kh_units(s, p.group, p.window, p.whole);
  const int unit = (int)((uint32_t)(at - before) / (uint32_t)units.blocks);
  const int begin = before + unit * units.blocks;
  const KhOwners owners = kh_owners(shares, line.all, begin, units.blocks);
  if (at == begin || owners.first != g - 1) return false;
  const int tile = unit / p.cache.kv_heads, rows = s.m * p.group - tile * kRows;
  parts = Parts{p.part_ml, p.part_o, ((int64_t)owners.first * 2 + owners.slot) * kRows, (int64_t)g * 2 * kRows, 2 * kRows,
                owners.count, tile * kRows, rows < kRows ? rows : kRows,
                unit - tile * p.cache.kv_heads, false};
  return true;
}

__device__ __forceinline__ bool wide_parts(const KhAttentionParams &p, int unit, int row0, KhSeq &s, Parts &parts) {
  const Line line = line_of(p, true);
  int before;
  if (unit >= line.all || sequence_at(p, line, unit, true, s, before) < 0) return false;
  const WideUnit u = wide_unit(p, s, unit - before);
  const int R0 = u.tile0 + row0, rows = u.tile_end - R0, count = kh_part(u.first, u.end, p.wide_splits, 0).used;
  if (count == 1 || rows <= 0) return false;
  const int64_t all = (int64_t)p.tokens * p.q_heads;
  parts = Parts{p.wide_ml, p.wide_o, 0, all, all, count, R0, rows < kRows ? rows : kRows, u.head, true};
  return true;
}

constexpr int kJoinParts = 64;  // statistics brought to LDS at a time
constexpr int kJoinAhead = 16;  // parts whose rows are in flight

// Joins the parts of 16 rows: a workgroup for every workgroup's start, then one
// for each 16 rows of the wide units. A thread has 4 columns of a row, and where
// that leaves threads over (few rows), only each second or fourth part of it.
// The parts were written through other L2s, so that each round of loads takes
// its time: bound by how many there are in a row.
template <int D>
__device__ __forceinline__ void join(const KhAttentionParams &p, float *lds) {
  constexpr int kCols = D / 4;
  const int tid = threadIdx.x, d = p.cache.head_dim;
  const int narrow_blocks = p.whole ? 0 : p.groups, block = (int)blockIdx.x - narrow_blocks;
  constexpr int kPer = kWideTile / kRows;
  KhSeq s{0, 0, 0};
  Parts parts{};
  if (!(block < 0 ? narrow_parts(p, (int)blockIdx.x, s, parts) : wide_parts(p, block / kPer, block % kPer * kRows, s, parts))) return;
  auto base = [&](int k) { return k == 0 ? parts.first : parts.others + (k - 1) * parts.step; };
  auto place_of = [&](int row) {
    if (!parts.wide) return (int64_t)row;
    const int R = parts.R0 + row, i = (int)kh_div(R, p.by_group);
    return (int64_t)(s.start + i) * p.q_heads + parts.head * p.group + R - i * p.group;
  };
  // Rows rounded up to a power of two, times columns: items; threads that share one.
  const int rows2 = parts.rows <= 1 ? 1 : parts.rows <= 2 ? 2 : parts.rows <= 4 ? 4 : parts.rows <= 8 ? 8 : 16;
  const int items = rows2 * kCols, shares = items >= 256 ? 1 : 256 / items < 4 ? 256 / items : 4;
  for (int item0 = 0; item0 < items; item0 += 256) {
    const int share = tid / items, item = item0 + tid % items;  // item0 > 0: shares = 1
    const int row = item / kCols, col = item % kCols * 4;
    const bool live = row < parts.rows && col < d && share < shares;
    const int64_t place = place_of(live ? row : 0);
    f32x4 o = {0, 0, 0, 0};
    float m = kSeed, total = 0.0f;
    for (int k0 = 0; k0 < parts.count; k0 += kJoinParts) {
      const int here = parts.count - k0 < kJoinParts ? parts.count - k0 : kJoinParts;
      for (int x = tid; x < here * kRows; x += 256) {
        const int k = x / kRows, r = x % kRows;
        const float *from = parts.ml + (base(k0 + k) + place_of(r < parts.rows ? r : 0)) * 2;
        lds[2 * x] = from[0], lds[2 * x + 1] = from[1];
      }
      kh::lds_barrier();
      if (live) {
        float top = m;
        for (int k = 0; k < here; ++k) top = fmaxf(top, lds[2 * (k * kRows + row)]);
        const float fade = kh::exp2_hw(m - top);
        m = top, total *= fade, o *= fade;
        for (int k1 = share; k1 < here; k1 += kJoinAhead * shares) {
          f32x4 x[kJoinAhead];
#pragma unroll
          for (int j = 0; j < kJoinAhead; ++j) {
            const int k = k1 + j * shares;
            x[j] = *reinterpret_cast<const f32x4 *>(parts.o + (base(k0 + (k < here ? k : here - 1)) + place) * d + col);
          }
#pragma unroll
          for (int j = 0; j < kJoinAhead; ++j) {
            const int k = k1 + j * shares;
            if (k < here) {
              const float w = kh::exp2_hw(lds[2 * (k * kRows + row)] - top);
              total += lds[2 * (k * kRows + row) + 1] * w;
              o += x[j] * w;
            }
          }
        }
      }
      kh::lds_barrier();
    }
    // The shares' sums, in their order.
    if (shares > 1) {
      float *sum = lds + 5 * tid;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = o[e];
      sum[4] = total;
      kh::lds_barrier();
      if (share == 0)
        for (int k = 1; k < shares; ++k) {
          const float *other = lds + 5 * (tid + k * items);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] += other[e];
          total += other[4];
        }
    }
    if (!live || share != 0) continue;
    const int R = parts.R0 + row, i = (int)kh_div(R, p.by_group), hq = parts.head * p.group + R - i * p.group;
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
    kh::store4(static_cast<elem *>(p.out) + (int64_t)(s.start + i) * p.out_stride + (int64_t)hq * d + col, y);
    if (col == 0 && p.lse != nullptr) p.lse[(int64_t)(s.start + i) * p.q_heads + hq] = lse_of(m, total, kLift);
  }
}

}  // namespace

// Two workgroups to a CU, so that one's loads are in flight while the other
// multiplies; a wave of the widest rows needs the registers of both.
#define KH_ATTENTION(D, PER_CU)                                                                                  \
  extern "C" __global__ void __launch_bounds__(256, PER_CU) KH_TYPED(paged_attention_##D)(const KhAttentionParams p) { \
    __shared__ float lds[kWaves * kRows * 2 + kRows + kWaves * kRows * (D + 4)];                                 \
    if (p.even)                                                                                                  \
      narrow<D, true>(p, (int)blockIdx.x, lds);                                                                  \
    else                                                                                                         \
      narrow<D, false>(p, (int)blockIdx.x, lds);                                                                 \
  }
KH_ATTENTION(64, 2)
KH_ATTENTION(128, 2)
KH_ATTENTION(256, 1)
// Steps with sequences of many rows: their workgroups first, the longest there are.
template <int D, bool EVEN>
__device__ __forceinline__ void either(const KhAttentionParams &p, char *lds) {
  if ((int)blockIdx.x < p.wide_blocks)
    wide<D, EVEN>(p, (int)blockIdx.x, lds);
  else
    narrow<D, EVEN>(p, (int)blockIdx.x - p.wide_blocks, reinterpret_cast<float *>(lds));
}
#define KH_ATTENTION_WIDE(D, PER_CU)                                                                              \
  extern "C" __global__ void __launch_bounds__(256, PER_CU) KH_TYPED(paged_attention_wide_##D)(const KhAttentionParams p) { \
    __shared__ __attribute__((aligned(16))) char lds[Wide<D>::lds];                                               \
    if (p.even)                                                                                                   \
      either<D, true>(p, lds);                                                                                    \
    else                                                                                                          \
      either<D, false>(p, lds);                                                                                   \
  }
KH_ATTENTION_WIDE(64, 2)
KH_ATTENTION_WIDE(128, kh::kWide ? 1 : 2)
KH_ATTENTION_WIDE(256, 1)
#define KH_ATTENTION_JOIN(D)                                                                                       \
  extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_attention_join_##D)(const KhAttentionParams p) { \
    __shared__ float lds[kJoinParts * kRows * 2];                                                                   \
    join<D>(p, lds);                                                                                                \
  }
KH_ATTENTION_JOIN(64)
KH_ATTENTION_JOIN(128)
KH_ATTENTION_JOIN(256)
