// Attention of the new tokens of ragged sequences over a paged cache in 8 bits:
//   x_ij = scale q_i . k_j, or cap tanh(scale q_i . k_j / cap)
//   lse_i = log sum_j exp x_ij,  o_i = sum_j exp(x_ij - lse_i) v_j
// over the entries j that token i sees, as in paged_attention.hip; k_j and v_j are
// e4m3 numbers times a power of two of their row.
//
// Such a row is exact in bf16, and the conversion takes the power of two along, so
// that every product is one of bf16 numbers, whatever the type of q and out: q is
// the sum of kParts bf16 numbers (bf16 one, fp16 two, fp32 three of 8 bits each:
// exact), and so is P for the second product (off by half a step of bf16, 2^-17 and
// 2^-24). Sums are in 32 bits. Against products of fp32 this is a third of the time
// of the matrix units, and 8 bits times 8 bits would need K and V's other operand
// in e4m3, 4 bits of it.
//
// Few rows to a sequence: 16 rows of a wave against blocks of entries, in shares of the
// step as in paged_attention.hip.
//   S^T = K Q^T     the result's lane l holds row l % 16 and entries 4 (l / 16) + i
//                   of each 16: a row's softmax crosses lanes twice.
//   O^T += V^T P^T  P as the lanes hold it, in bf16.
// In two forms: narrow_even() for pages of whole sixteens (K and V straight to LDS, blocks
// of 32 entries), narrow() for others (K and V in registers, blocks of 64, and of 32 with
// rows past 128 elements). Bound by reading K and V: MI355X, bf16,
// 8 kv heads of 128, 64 sequences of 513 to 8192 entries 110 us, 5.2 TB/s, with
// pages of 24 slots 138; one of 131071 59-67 us, 4.0-4.6 TB/s with the launch of the join
// and both kernels' ends; four of 1024, 16 heads of 64 in fp32, 14 us, of which the
// two launches are ten.
//
// Many rows (wide): 128 rows of a workgroup against tiles of 64 entries, which go
// to LDS as bf16: each byte is converted once for 128 rows. Bound by what the waves
// issue, the softmax's and the conversions' instructions (54% of the time) and the
// matrix units' (32%) in turn: a chunk of 2048 at 8192 entries, 32 heads on 8 of
// 128, bf16, 283 to 305 us, 795 to 855 TFLOP/s.
//
// Entries that all sequences share are worked on by wide units whose rows are all
// tokens of the step; their parts and the sequences' own are joined row by row.
#include "kh_step.h"

#if KH_ELEM != 2
#error "the products are of bf16 numbers; KH_ROWS is the type of q and out"
#endif

namespace {

using namespace kh;

#if KH_ROWS == 0
using row_t = float;
constexpr int kParts = 3;
#elif KH_ROWS == 1
using row_t = _Float16;
constexpr int kParts = 2;
#else
using row_t = __bf16;
constexpr int kParts = 1;
#endif

// Four floats in the rows' type, rounded to nearest even.
__device__ __forceinline__ void store_row(row_t *p, const float (&x)[4]) {
#if KH_ROWS == 0
  *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
#else
  typedef row_t Two __attribute__((ext_vector_type(2)));
  const Two a = {static_cast<row_t>(x[0]), static_cast<row_t>(x[1])}, b = {static_cast<row_t>(x[2]), static_cast<row_t>(x[3])};
  *reinterpret_cast<u32x2 *>(p) = u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
#endif
}

// Eight numbers as kParts of bf16: the leading bits, the next ones of what is
// left, exact but for the last part's rounding. What is left of an infinity is
// nothing.
__device__ __forceinline__ void in_parts(u32x4 (&part)[kParts], const float (&x)[8], bool any) {
  float left[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) left[j] = x[j];
#pragma unroll
  for (int n = 0; n < kParts; ++n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = left[2 * j], b = left[2 * j + 1];
      if (n == kParts - 1) {
        part[n][j] = pack2(a, b);
        continue;
      }
      const uint32_t wa = __float_as_uint(a), wb = __float_as_uint(b);
      part[n][j] = __builtin_amdgcn_perm(wb, wa, 0x07060302u);
      left[2 * j] = a - __uint_as_float(wa & 0xffff0000u);
      left[2 * j + 1] = b - __uint_as_float(wb & 0xffff0000u);
      if (any) {
        if ((wa & 0x7fffffffu) == 0x7f800000u) left[2 * j] = 0.0f;
        if ((wb & 0x7fffffffu) == 0x7f800000u) left[2 * j + 1] = 0.0f;
      }
    }
  }
}

// Eight elements of q.
__device__ __forceinline__ void load_q(u32x4 (&part)[kParts], const row_t *at, bool real, const KhAttention8Params &p) {
  const u32x4 *from = reinterpret_cast<const u32x4 *>(at);
  const u32x4 zero = {0, 0, 0, 0};
  const u32x4 w = real ? from[0] & p.q_keep ^ p.q_sign : zero;
#if KH_ROWS == 2
  part[0] = w;
#else
  float x[8];
#if KH_ROWS == 1
  typedef _Float16 Two __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t word = w[j];
    const Two t = __builtin_bit_cast(Two, word);
    x[2 * j] = static_cast<float>(t.x), x[2 * j + 1] = static_cast<float>(t.y);
  }
#else
  const u32x4 v = real ? from[1] & p.q_keep ^ p.q_sign : zero;
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(w[j]), x[4 + j] = __uint_as_float(v[j]);
#endif
  in_parts(part, x, true);
#endif
}

// The power of two that a scale's byte stands for.
__device__ __forceinline__ float power_of(uint32_t byte) {
  const uint32_t up = byte > KH_SCALE_LEAST ? byte : KH_SCALE_LEAST, b = up < KH_SCALE_MOST ? up : KH_SCALE_MOST;
  return __uint_as_float(b << 23);
}

// Two of a word's four numbers, times a power of two, in bf16: exact.
template <bool UPPER>
__device__ __forceinline__ uint32_t widen(uint32_t w, float power) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, power, UPPER));
}

// The top bit of each byte of w that is a NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u & 0x80808080u; }

// w with zeros for NaN.
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
  const uint32_t n = nan_bytes(w);
  return w & ~((n >> 7) * 0xffu);
}

// Scores over the cap, capped: tanh(y cap_in / (2 log2 e)), which cap_out takes back to
// scores in powers of two. By way of t = 2^(y cap_in) it is 1 - 2 / (t + 1), off by
// some 2^-23 of the cap. near: what lies below a quarter of the cap comes from the
// power series (first term left out 2e-10 of the score), 16 instructions a score instead
// of 5. Few rows have the time for it (64 sequences of 513 to 8192 entries 112 us with
// either); chunks feel every instruction. Of a chunk's 16-bit rows' weights 2^-23 of a
// cap up to 256 is nothing (2^-15 of a weight), nor is it of their lse over many entries.
// Rows of fp32, under larger caps or windows of few entries (cap_near), and waves with a
// row that sees no more than KH_FEW_CAPPED, whose lse is as far off as each of them, take
// the series there too: what the row sees decides, not what else the step holds (16
// chunks of up to 301 of 4001 fp16 tokens, windows of 1000, 86 us, all by the series 104).
template <int N, class X>
__device__ __forceinline__ void cap(X &y, const KhAttention8Params &p, bool near) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float x = y[j] * p.cap_in;
    float r = fmaf(-2.0f, __builtin_amdgcn_rcpf(exp2_hw(x) + 1.0f), 1.0f);
    if (near) {
      const float a = x * 0.34657359027997265471f, z = a * a;  // log(2) / 2
      const float series = a + a * z * (-1.0f / 3 + z * (2.0f / 15 + z * (-17.0f / 315 + z * (62.0f / 2835 + z * (-1382.0f / 155925)))));
      r = z < 0.0625f ? series : r;
    }
    y[j] = r;
  }
}

// ---- few rows

template <int D>
struct Few {
  static constexpr int steps = D / 64;                // loads of 16 bytes of a lane to a row of K
  static constexpr int tiles = D > 128 ? 2 : 4;
  static constexpr int keys = 16 * tiles;             // entries of a block
  static constexpr int mine = 4 * tiles;              // of a lane
  static constexpr int piece = D / 16, words = D / 64;  // columns of V of a lane
};

// Where a block's rows lie.
template <int D>
struct Stretch {
  KhSlot at[Few<D>::tiles];  // of entry 16 t + l % 16
  uint64_t present;
};

template <int D>
__device__ __forceinline__ void find(Stretch<D> &b, const KhAttention8Params &p, const int32_t *table, int key0, int end, int lane) {
#pragma unroll
  for (int t = 0; t < Few<D>::tiles; ++t) b.at[t] = look_up<false>(p, table, key0 + 16 * t + lane % 16, end);
}

// Absent rows are read from the cache's first page: kh_cache.h, Block.
template <int D>
__device__ __forceinline__ void settle(Stretch<D> &b, const KhAttention8Params &p, int key0, int end, int lane) {
  b.present = 0;
#pragma unroll
  for (int t = 0; t < Few<D>::tiles; ++t) {
    const bool there = key0 + 16 * t + lane % 16 < end && (uint32_t)b.at[t].page < (uint32_t)p.cache.pages;
    b.present |= (__builtin_amdgcn_ballot_w64(there) & 0xffffu) << (16 * t);
    if (!there) b.at[t] = KhSlot{0, 0};
  }
}

// A block's rows of K: lane l has 16 bytes at 16 (l / 16) of each 64 of entry l % 16,
// and that entry's scale.
template <int D>
struct RowsOfK {
  u32x4 w[Few<D>::tiles][Few<D>::steps];
  uint32_t scale[Few<D>::tiles];
};

// Of V: D / 16 columns of the lane's entries, and the scale of entry l % 16.
template <int D>
struct RowsOfV {
  uint32_t w[Few<D>::mine][Few<D>::words];
  uint32_t scale[Few<D>::tiles];
};

template <int D>
__device__ __forceinline__ void load_k(RowsOfK<D> &k, const Stretch<D> &b, const KhAttention8Params &p, const char *base,
                                       const uint8_t *scales, int row_bytes, int h) {
  using F = Few<D>;
#pragma unroll
  for (int t = 0; t < F::tiles; ++t) {
    const char *row = base + kh_row(b.at[t], p.cache.k_page, p.cache.k_slot);
#pragma unroll
    for (int c = 0; c < F::steps; ++c)
      k.w[t][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + within(64 * c + 16 * h, row_bytes)));
    k.scale[t] = scales[(uint64_t)(uint32_t)b.at[t].page * p.scale_page + (uint32_t)b.at[t].slot];
  }
}

template <int D>
__device__ __forceinline__ void load_v(RowsOfV<D> &v, const Stretch<D> &b, const KhAttention8Params &p, const char *base,
                                       const uint8_t *scales, int row_bytes, int r, int h) {
  using F = Few<D>;
#pragma unroll
  for (int t = 0; t < F::tiles; ++t) {
    const uint64_t own = kh_row(b.at[t], p.cache.v_page, p.cache.v_slot);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Entry 4 h + i is the one that lane 4 h + i looked up.
      const uint32_t lo = __shfl((uint32_t)own, 4 * h + i, kWave), hi = __shfl((uint32_t)(own >> 32), 4 * h + i, kWave);
      const char *from = base + ((uint64_t)hi << 32 | lo) + within(F::piece * r, row_bytes);
      uint32_t(&w)[F::words] = v.w[4 * t + i];
      if constexpr (F::words == 4) {
        const u32x4 g = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from));
        w[0] = g.x, w[1] = g.y, w[2] = g.z, w[3] = g.w;
      } else if constexpr (F::words == 2) {
        const u32x2 g = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(from));
        w[0] = g.x, w[1] = g.y;
      } else {
        w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(from));
      }
    }
    v.scale[t] = scales[(uint64_t)(uint32_t)b.at[t].page * p.scale_page + (uint32_t)b.at[t].slot];
  }
}

// The scales' powers of the lane's entries of 32, half `g` of the block.
template <int D>
__device__ __forceinline__ void powers_of(float (&power)[8], const RowsOfV<D> &v, int g, int h) {
#pragma unroll
  for (int j = 0; j < 8; ++j) power[j] = power_of(__shfl(v.scale[2 * g + j / 4], 4 * h + j % 4, kWave));
}

// Writes of results: to out, or where sequences share entries to the parts that
// combine() joins.
__device__ __forceinline__ void finish(const KhAttention8Params &p, int token, int hq, int col, const f32x4 &o, float m, float total) {
  const int d = p.cache.head_dim;
  const int64_t row = (int64_t)token * p.q_heads + hq;
  if (p.shared > 0) {
    const int64_t at = (int64_t)p.shared_splits * p.tokens * p.q_heads + row;
    *reinterpret_cast<f32x4 *>(p.shared_o + at * d + col) = o;
    if (col == 0) p.shared_ml[2 * at] = m, p.shared_ml[2 * at + 1] = total;
    return;
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  store_row(static_cast<row_t *>(p.out) + (int64_t)token * p.out_stride + (int64_t)hq * d + col, y);
  if (col == 0 && p.lse != nullptr) p.lse[row] = lse_of(m, total, 0.0f);
}

// Writes down what workgroup `block` is the second to work on: the unit, of the
// sequence s with `before` blocks before it, that its share starts inside of.
__device__ __forceinline__ void tell(const KhAttention8Params &p, const Line &line, const KhShares &shares, int block, int start,
                                     int seq, const KhSeq &s, int before) {
  if (p.whole != 0 || threadIdx.x != 0) return;
  KhJoin j{};
  if (block > 0 && block < shares.groups && seq >= 0) {
    const KhUnits units = kh_units_of(p, s);
    const int unit = (int)((uint32_t)(start - before) / (uint32_t)units.blocks), begin = before + unit * units.blocks;
    const KhOwners owners = kh_owners(shares, line.all, begin, units.blocks);
    if (start != begin && owners.first == block - 1) {
      const int tile = unit / p.head_groups, rows = s.m * p.group - tile * kRows;
      j = KhJoin{owners.count, owners.first, owners.slot, s.start, tile * kRows, rows < kRows ? rows : kRows,
                 (unit - tile * p.head_groups) * p.together, 0};
    }
  }
  p.joins[block] = j;
}

__device__ __forceinline__ bool told_parts(const KhAttention8Params &p, int block, KhSeq &s, Parts &parts) {
  const int g = block / p.together, nth = block - g * p.together;
  const KhJoin j = p.joins[g];
  if (j.count == 0 || j.head0 + nth >= p.cache.kv_heads) return false;
  s.start = j.start;
  parts = Parts{p.part_ml, p.part_o, (((int64_t)j.first * 2 + j.slot) * p.together + nth) * kRows,
                ((int64_t)g * 2 * p.together + nth) * kRows, 2 * p.together * kRows, j.count, j.row0, j.rows, j.head0 + nth, false};
  return true;
}

template <int D>
__device__ __forceinline__ void narrow(const KhAttention8Params &p, int block, float *lds) {
  using F = Few<D>;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim;

  const Line line = line_of(p, false);
  const KhShares shares = shares_of(p, line);
  KhSeq s{0, 0, 0};
  int seq = -1, before = 0;  // blocks of the sequences before this one
  const int start = kh_share(shares, block), end = kh_share(shares, block + 1);
  if (block < shares.groups) seq = sequence_at(p, line, start, false, s, before);
  tell(p, line, shares, block, start, seq, s, before);
  if (seq < 0) return;
  // The join area: each wave's maxima and sums of its rows, the rows' own of the
  // workgroup, and each wave's part of O.
  float *ml = lds, *both = lds + kWaves * kRows * 2, *part = both + kRows * 2;
  constexpr int kPitch = D + 4;
  KhUnits units = kh_units_of(p, s);
  const float factor0 = p.cap_in != 0.0f ? p.cap_out : p.scale_log2;

  for (int at = start, in = start - before; at < end;) {
    while (kh_passed(in, kh_work(units, p.cache.kv_heads))) {
      // The next sequence of few rows: wide() has the others.
      do {
        if (++seq >= p.table.seqs) return;
        s = sequence(p, seq);
      } while (s.m * p.group > p.narrow_rows);
      units = kh_units_of(p, s);
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
    const uint8_t *kscales = p.k_scale + (uint64_t)head * p.scale_head, *vscales = p.v_scale + (uint64_t)head * p.scale_head;

    const int R = row0 + r;
    const bool mine = R < rows;
    const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
    const int i_first = (int)kh_div(row0, p.by_group);
    const int i_last = (int)kh_div(row0 + kRows < rows ? row0 + kRows - 1 : rows - 1, p.by_group);
    const KhSpan seen = kh_span_of(p, s, i);
    const KhSpan low = kh_span_of(p, s, i_first), high = kh_span_of(p, s, i_last);
    const int key_first = (low.first > from ? low.first : from) & ~15;  // from is a multiple of 16
    const int key_end = high.end < to ? high.end : to;

    // q's columns as K's bytes lie: of each 64, 16 of a lane, in two steps.
    u32x4 q[2 * F::steps][kParts];
    const row_t *qp = static_cast<const row_t *>(p.q) + ((int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d);
#pragma unroll
    for (int c = 0; c < 2 * F::steps; ++c) {
      const int col = 64 * (c / 2) + 16 * h + 8 * (c % 2);
      // From an address that is there in any case, as the rows of K and V.
      load_q(q[c], qp + within(col, d), mine && col < d, p);
    }

    // Of row l % 16; l of this lane's entries alone. A row that there is none of has
    // no scores, and no maximum to look after either.
    float m = mine ? kSeed : 0.0f, l = 0.0f;
    f32x4 o[F::piece];
#pragma unroll
    for (int e = 0; e < F::piece; ++e) o[e] = f32x4{0, 0, 0, 0};

    // K and V are a block ahead of their use, the page numbers two: K's next
    // block goes out as soon as the scores have taken its registers' content,
    // V's when the products have.
    int key0 = key_first + wave * F::keys;
    if (key0 < key_end) {
      constexpr int kStep = kWaves * F::keys;
      RowsOfK<D> k;
      RowsOfV<D> v;
      Stretch<D> now, next;
      find<D>(now, p, table, key0, key_end, lane);
      find<D>(next, p, table, key0 + kStep, key_end, lane);
      settle<D>(now, p, key0, key_end, lane);
      load_k<D>(k, now, p, kbase, kscales, d, h);
      // K goes out before V here as in the loop: the wait for K at its top then
      // leaves V in flight.
      __builtin_amdgcn_sched_barrier(0);
      load_v<D>(v, now, p, vbase, vscales, d, r, h);
      for (; key0 < key_end; key0 += kStep) {
        const uint64_t present = now.present;
        float y[F::mine];
        if (d != D) {
          // Columns past the row's end were read from its start.
#pragma unroll
          for (int c = 0; c < F::steps; ++c)
            if (64 * c + 16 * h >= d) {
#pragma unroll
              for (int t = 0; t < F::tiles; ++t) k.w[t][c] = u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int t = 0; t < F::tiles; ++t) {
          f32x4 x = {0, 0, 0, 0};
          const float power = power_of(k.scale[t]);
#pragma unroll
          for (int c = 0; c < 2 * F::steps; ++c) {
            const uint32_t w0 = k.w[t][c / 2][2 * (c % 2)], w1 = k.w[t][c / 2][2 * (c % 2) + 1];
            const u32x4 a = {widen<false>(w0, power), widen<true>(w0, power), widen<false>(w1, power), widen<true>(w1, power)};
#pragma unroll
            for (int n = 0; n < kParts; ++n) x = mma16(a, q[c][n], x);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * t + e] = x[e];
        }
        now = next;
        settle<D>(now, p, key0 + kStep, key_end, lane);
        load_k<D>(k, now, p, kbase, kscales, d, h);
        find<D>(next, p, table, key0 + 2 * kStep, key_end, lane);

        if (p.cap_in != 0.0f) {
          cap<F::mine>(y, p, true);
        }
        // Every row sees every entry of the block: no mask.
        const bool whole = present == ~uint64_t(0) >> (64 - F::keys) && key0 + F::keys <= low.end && key0 >= high.first;
        uint64_t odds = 0;  // bit n: entry n of the block, in this lane's columns
        if (!whole) {
          // Of the lane's entries: those that its row sees, and those that are there.
          const uint64_t sees = (mine ? seen_of(seen, key0) & present : 0) >> 4 * h, there = present >> 4 * h;
#pragma unroll
          for (int j = 0; j < F::mine; ++j) {
            const uint64_t bit = uint64_t(1) << (16 * (j / 4) + j % 4);
            y[j] = (sees & bit) != 0 ? y[j] : -__builtin_inff();
#pragma unroll
            for (int w = 0; w < F::words; ++w) {
              v.w[j][w] = (there & bit) != 0 ? v.w[j][w] : 0u;
              odds |= nan_bytes(v.w[j][w]) != 0 ? bit : 0;
            }
          }
          odds <<= 4 * h;
        }
        float top = y[0];
#pragma unroll
        for (int j = 1; j < F::mine; ++j) top = fmaxf(top, y[j]);
        top = fmaxf(m, over_rows(top, true) * factor0);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {
          const float fade = exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int e = 0; e < F::piece; ++e) o[e] *= fade;
        }
        const bool far = coarse(m);
        const float factor = far ? 1.0f : factor0, shift = far ? 0.0f : -m;
        if (far) less<F::mine>(y, factor0, m);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < F::mine; ++j) {
          y[j] = exp2_hw(fmaf(y[j], factor, shift));
          sum += y[j];
        }
        l += sum;
        if (__builtin_amdgcn_ballot_w64(odds != 0) != 0) {
          // NaN in V where rows differ in what they see: 0 x V would reach the rows
          // that do not. They leave the products as zeros and are added, read once
          // more, to the rows that do see them.
          for (int n = 0; n < F::keys; ++n) {
            if (__builtin_amdgcn_ballot_w64((odds >> n & 1) != 0) == 0) continue;
            const int key = key0 + n;
            const KhSlot at_key = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)key);
            const char *row = vbase + kh_row(at_key, p.cache.v_page, p.cache.v_slot);
            if (mine && key >= seen.first && key < seen.end) {
              const int h1 = apart(h);
#pragma unroll
              for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
                for (int e = 0; e < F::piece; e += 4) {
                  const int col = F::piece * (4 * h1 + i4) + e;
                  if (col >= d) continue;
                  const uint32_t odd = nan_bytes(*reinterpret_cast<const uint32_t *>(row + col));
#pragma unroll
                  for (int b = 0; b < 4; ++b)
                    if ((odd >> 8 * b & 0x80u) != 0) o[e + b][i4] = __builtin_nanf("");
                }
            }
          }
          // Its loads end here: one that the compiler took for still on its way would
          // have the common path wait for all, the next block among them.
          vm_wait<0>();
#pragma unroll
          for (int j = 0; j < F::mine; ++j)
#pragma unroll
            for (int w = 0; w < F::words; ++w) v.w[j][w] = without_nan(v.w[j][w]);
        }
#pragma unroll
        for (int g = 0; g < F::tiles / 2; ++g) {
          u32x4 b[kParts];
          const float eight[8] = {y[8 * g], y[8 * g + 1], y[8 * g + 2], y[8 * g + 3], y[8 * g + 4], y[8 * g + 5], y[8 * g + 6], y[8 * g + 7]};
          in_parts(b, eight, false);
          float power[8];
          powers_of<D>(power, v, g, h);
#pragma unroll
          for (int e = 0; e < F::piece; e += 2) {
            uint32_t x[8];  // columns e and e + 1 of the eight entries
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const uint32_t w = v.w[8 * g + j][e / 4];
              x[j] = (e & 2) != 0 ? widen<true>(w, power[j]) : widen<false>(w, power[j]);
            }
            u32x4 a0, a1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              a0[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
              a1[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int n = 0; n < kParts; ++n) {
              o[e] = mma16(a0, b[n], o[e]);
              o[e + 1] = mma16(a1, b[n], o[e + 1]);
            }
          }
        }
        load_v<D>(v, now, p, vbase, vscales, d, r, h);
      }
    }

    // Join the waves: rescale to the rows' common maximum, add in wave order.
    l = over_rows(l, false);
    if (h == 0) {
      ml[(wave * kRows + r) * 2] = m;
      ml[(wave * kRows + r) * 2 + 1] = l;
    }
    lds_barrier();
    float top = kSeed;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * kRows + r) * 2]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += ml[(w * kRows + r) * 2 + 1] * exp2_hw(ml[(w * kRows + r) * 2] - top);
    const float fade = exp2_hw(m - top);
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
      for (int e = 0; e < F::piece; ++e) part[(wave * kRows + r) * kPitch + F::piece * (4 * h + i4) + e] = o[e][i4] * fade;
    if (wave == 0 && h == 0) {
      both[2 * r] = top, both[2 * r + 1] = total;
      if (!alone) {
        float *ml_to = p.part_ml + ((int64_t)block * 2 + slot) * kRows * 2 + r * 2;
        ml_to[0] = top;
        ml_to[1] = total;
      }
    }
    lds_barrier();
    for (int x = threadIdx.x; x < kRows * (D / 4); x += kWaves * kWave) {
      const int row = x / (D / 4), col = x % (D / 4) * 4, RR = row0 + row;
      if (RR >= rows || col >= d) continue;
      const int ii = (int)kh_div(RR, p.by_group), hh = head * p.group + RR - ii * p.group;
      f32x4 y = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) y += *reinterpret_cast<const f32x4 *>(part + (w * kRows + row) * kPitch + col);
      if (alone)
        finish(p, s.start + ii, hh, col, y, both[2 * row], both[2 * row + 1]);
      else
        *reinterpret_cast<f32x4 *>(p.part_o + (((int64_t)block * 2 + slot) * kRows + row) * d + col) = y;
    }
    lds_barrier();  // before the next unit writes the join area
  }
}

// ---- few rows, pages of whole sixteens
//
// The same products with K and V straight to LDS, whole rows at a time (a load of
// 64 bytes of each row, as the matrix operand lies, takes the memory 17% longer),
// two blocks ahead of their use. A wave has its own LDS, and nobody waits for
// others: two buffers of a block's rows of K, and of V, their scales' bytes, the
// powers of two these stand for, and the page numbers of the next blocks, 64
// tiles' at a time.
//   S^T   A = 16 bytes of a row of K, two steps' operands.
//   O^T   A = eight entries of a column of V, read across its rows; V's powers
//         of two are multiplied into P, and lane l ends with columns
//         16 c + 4 (l / 16) + i of row l % 16.
// A row's 16-byte pieces lie at their number exclusive-or a number of the row's, so
// that 16 rows of K in a column, and the rows of V that two groups of 16 lanes read
// across, fill the banks once.
template <int D>
struct Ring {
  static constexpr int tiles = 2, keys = 16 * tiles, mine = 4 * tiles;  // entries of a block, and of a lane
  static constexpr int pieces = D / 16, rows = 64 / pieces;  // rows that a load brings
  static constexpr int loads = 16 / rows;                    // of a tile
  static constexpr int ops = tiles * loads + 1;              // of a block's rows of K, or V, and their scales
  static constexpr int block = keys * D;
  static constexpr int k_at = 0, v_at = 2 * block, scales_at = 4 * block;  // scales: [K, V][2 buffers][256]
  static constexpr int powers_at = scales_at + 4 * 256, pages_at = powers_at + 2 * 256;  // powers: [K, V][64] floats
  static constexpr int places_at = pages_at + 256, there_at = places_at + 64 * 32;  // of 64 tiles
  static constexpr int lds = there_at + 64 * 2;   // of a wave
  static constexpr int ahead = 64 / tiles;        // blocks whose pages are found at a time
};

template <int D>
__device__ __forceinline__ int k_swap(int row) {
  return D == 64 ? row >> 2 & 3 : D == 128 ? row >> 1 & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int v_swap(int row) {
  return D == 64 ? (row >> 2 & 1) | (row >> 3 & 2) : D == 128 ? (row >> 1 & 3) | (row >> 2 & 4) : (row & 7) | (row >> 1 & 8);
}

// Of 8 x 16 bytes in LDS that the 16 lanes of a row point at (lane 2 r + c: row r,
// columns 8 c ..), lane i receives column i, its eight rows in order.
__device__ __forceinline__ u32x2 read_across8(const char *p) {
  typedef int Two __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                                       (__attribute__((address_space(3))) Two *)const_cast<char *>(p)));
}

// What was read from LDS has arrived: what it was read from may be written.
__device__ __forceinline__ void read_out() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ uint32_t lds_of(const char *p) { return (uint32_t)reinterpret_cast<uintptr_t>(p); }

// Asks for the page numbers of 64 tiles, those of `ahead` blocks of the wave's, the
// first at key0 and `step` entries apart: lane n the n-th's.
template <class F>
__device__ __forceinline__ void ask(const KhAttention8Params &p, const int32_t *table, int key0, int step, int end, char *own, int lane) {
  // In 64 bits: blocks that are asked for may lie past 2^31.
  const int64_t key = (int64_t)key0 + (int64_t)(lane / F::tiles) * step + 16 * (lane % F::tiles);
  const int last = (end - 1) & ~15;
  const uint32_t inside = (uint32_t)(key < last ? key : last);
  const uint32_t i = __umulhi(inside, p.cache.by_page.mul) >> p.cache.by_page.shift;  // kh_div: pages hold 16 entries at least
  const uint64_t at = reinterpret_cast<uintptr_t>(table);
  dma4(u32x4{(uint32_t)at, (uint32_t)(at >> 32), (uint32_t)p.table.width * 4u, 0x00020000u}, 4 * i, lds_of(own + F::pages_at));
}

// From page numbers to where the tiles' rows lie, a lane each: two resources' words
// but the last, the scales' place, and which entries are there. A resource ends
// where the tile's entries do: absent rows arrive as zeros.
template <class F>
__device__ __forceinline__ void place(const KhAttention8Params &p, const char *kbase, const char *vbase, int key0, int step, int end,
                                      char *own, int lane) {
  const int64_t far = (int64_t)key0 + (int64_t)(lane / F::tiles) * step + 16 * (lane % F::tiles);
  const int key = (int)(far < end ? far : 0), left = far < end ? (end - key < 16 ? end - key : 16) : 0;
  const int page = reinterpret_cast<const int32_t *>(own + F::pages_at)[lane];
  const bool there = left > 0 && (uint32_t)page < (uint32_t)p.cache.pages;
  const uint32_t i = __umulhi((uint32_t)key, p.cache.by_page.mul) >> p.cache.by_page.shift;
  const KhSlot at = there ? KhSlot{page, key - (int)(i * p.cache.by_page.by)} : KhSlot{0, 0};
  const uint32_t rows = there ? (uint32_t)left : 0;
  // Addresses have 48 bits: the resource's stride, above them, is zero.
  const uint64_t k = reinterpret_cast<uintptr_t>(kbase) + kh_row(at, p.cache.k_page, p.cache.k_slot);
  const uint64_t v = reinterpret_cast<uintptr_t>(vbase) + kh_row(at, p.cache.v_page, p.cache.v_slot);
  u32x4 *to = reinterpret_cast<u32x4 *>(own + F::places_at) + 2 * lane;
  to[0] = u32x4{(uint32_t)k, (uint32_t)(k >> 32), rows * p.cache.k_slot, (uint32_t)at.page * p.scale_page + (uint32_t)at.slot};
  to[1] = u32x4{(uint32_t)v, (uint32_t)(v >> 32), rows * p.cache.v_slot, 0u};
  reinterpret_cast<uint16_t *>(own + F::there_at)[lane] = (uint16_t)((1u << rows) - 1);
}

// The loads of a tile: dma16 (kh_elem.h) 1, 2 or 4 times, 1 KB further in LDS each.
#define KH_DMA_NEXT(n) "s_add_u32 m0, m0, 0x400\n\ts_nop 0\n\tbuffer_load_dwordx4 %" #n ", %3, 0 offen nt lds\n\t"
#define KH_DMA_TILE(more, ...)                                     \
  asm volatile(                                                    \
      "s_mov_b32 %0, m0\n\t"                                       \
      "s_mov_b32 m0, %1\n\t"                                       \
      "s_nop 2\n\t"                                                \
      "buffer_load_dwordx4 %2, %3, 0 offen nt lds\n\t" more           \
      "s_mov_b32 m0, %0"                                           \
      : "=&s"(saved)                                               \
      : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff[0]), "s"(rsrc) __VA_ARGS__ \
      : "memory", "scc")
template <int LOADS>
__device__ __forceinline__ void dma_tile(u32x4 rsrc, const uint32_t (&voff)[LOADS], uint32_t lds) {
#pragma unroll
  for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
  uint32_t saved;
  if constexpr (LOADS == 1)
    KH_DMA_TILE("");
  else if constexpr (LOADS == 2)
    KH_DMA_TILE(KH_DMA_NEXT(4), , "v"(voff[1]));
  else
    KH_DMA_TILE(KH_DMA_NEXT(4) KH_DMA_NEXT(5) KH_DMA_NEXT(6), , "v"(voff[1]), "v"(voff[2]), "v"(voff[3]));
}
#undef KH_DMA_TILE
#undef KH_DMA_NEXT

// Sends a block's rows of K, or of V (which: 0 or 1), and their scales to LDS; n: its
// number among those placed, `ahead` for one that there is none of. voff: what a
// lane brings of a tile's rows in each load, tiles of even and odd number.
template <class F>
__device__ __forceinline__ void send(const KhAttention8Params &p, const char *own, int n, int which, const uint32_t (&voff)[2][F::loads],
                                     const uint8_t *scales, const char *to, const char *scales_to, int lane) {
  const u32x4 *places = reinterpret_cast<const u32x4 *>(own + F::places_at) + 2 * F::tiles * (n % F::ahead);
  const uint32_t scale = places[2 * (lane / 4 % F::tiles)].w + 4u * (uint32_t)(lane % 4);
#pragma unroll
  for (int t = 0; t < F::tiles; ++t) {
    u32x4 r = places[2 * t + which];
    r.z = n < F::ahead ? r.z : 0u;
    r.w = 0x00020000u;
    dma_tile<F::loads>(r, voff[t % 2], lds_of(to) + (uint32_t)(t * F::loads * 1024));
  }
  const uint64_t at = reinterpret_cast<uintptr_t>(scales);
  const uint32_t size = (uint32_t)(p.cache.pages - 1) * p.scale_page + (uint32_t)p.cache.page_size;
  dma4(u32x4{(uint32_t)at, (uint32_t)(at >> 32), size, 0x00020000u}, scale, lds_of(scales_to));
}

// Which entries of a placed block are there.
template <class F>
__device__ __forceinline__ uint64_t there_of(const char *own, int n) {
  const uint16_t *at = reinterpret_cast<const uint16_t *>(own + F::there_at) + F::tiles * (n % F::ahead);
  const uint32_t there = (uint32_t)__builtin_amdgcn_readfirstlane(*reinterpret_cast<const uint32_t *>(at));
  return n < F::ahead ? there : 0;
}

template <int D, int WAVES>
__device__ __forceinline__ void narrow_even(const KhAttention8Params &p, int block, char *lds) {
  using F = Ring<D>;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim;

  const Line line = line_of(p, false);
  const KhShares shares = shares_of(p, line);
  KhSeq s{0, 0, 0};
  int seq = -1, before = 0;  // blocks of the sequences before this one
  const int start = kh_share(shares, block), end = kh_share(shares, block + 1);
  if (block < shares.groups) seq = sequence_at(p, line, start, false, s, before);
  tell(p, line, shares, block, start, seq, s, before);
  if (seq < 0) return;
  // The join area, behind which nobody's loads are on their way any more: each
  // wave's maxima and sums of its rows, the rows' own of the workgroup, and each
  // wave's part of O.
  float *ml = reinterpret_cast<float *>(lds), *both = ml + WAVES * kRows * 2, *part = both + WAVES * kRows * 2;
  constexpr int kPitch = D + 4;
  char *own = lds + wave * F::lds;
  float *powers = reinterpret_cast<float *>(own + F::powers_at);
  KhUnits units = kh_units_of(p, s);
  const float factor0 = p.cap_in != 0.0f ? p.cap_out : p.scale_log2;

  uint32_t k_off[2][F::loads], v_off[2][F::loads];
#pragma unroll
  for (int i = 0; i < F::loads; ++i)
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) {
      const int row = i * F::rows + lane / F::pieces, piece = lane % F::pieces;
      const int kc = 16 * (piece ^ k_swap<D>(row)), vc = 16 * (piece ^ v_swap<D>(row + 16 * odd));
      k_off[odd][i] = kc < d ? (uint32_t)row * p.cache.k_slot + (uint32_t)kc : kOutside;
      v_off[odd][i] = vc < d ? (uint32_t)row * p.cache.v_slot + (uint32_t)vc : kOutside;
    }

  // Of two workgroups on a CU the older one's waves go first, and the other one would
  // end alone, some 15% later. So the second goes first for half of its share, the
  // older one after that (64 sequences of 513 to 8192 entries, 122 us without, 114
  // with).
  const int second = block >= shares.groups / 2 && shares.groups > KH_CUS;
  int first_half = second ? (end - start) * (KH_STRETCH / 2) : 0;  // entries until then
  if (second) __builtin_amdgcn_s_setprio(1);
  for (int at = start, in = start - before; at < end;) {
    while (kh_passed(in, kh_work(units, p.head_groups))) {
      // The next sequence of few rows: wide() has the others.
      do {
        if (++seq >= p.table.seqs) return;
        s = sequence(p, seq);
      } while (s.m * p.group > p.narrow_rows);
      units = kh_units_of(p, s);
    }
    const uint32_t unit = (uint32_t)in / (uint32_t)units.blocks;
    const int tile = (int)(unit / (uint32_t)p.head_groups), head0 = (int)(unit - (uint32_t)tile * (uint32_t)p.head_groups) * p.together;
    // The waves share the unit's heads out, and a head's share the entries.
    const int heads = p.cache.kv_heads - head0 < p.together ? p.cache.kv_heads - head0 : p.together;
    const int per_head = heads == 1 ? WAVES : heads == 2 ? WAVES / 2 : 1;
    const int nth = wave / per_head, head = head0 + (nth < heads ? nth : 0);
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
    const uint8_t *kscales = p.k_scale + (uint64_t)head * p.scale_head, *vscales = p.v_scale + (uint64_t)head * p.scale_head;

    const int R = row0 + r;
    const bool mine = R < rows;
    const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
    const int i_first = (int)kh_div(row0, p.by_group);
    const int i_last = (int)kh_div(row0 + kRows < rows ? row0 + kRows - 1 : rows - 1, p.by_group);
    const KhSpan seen = kh_span_of(p, s, i);
    const KhSpan low = kh_span_of(p, s, i_first), high = kh_span_of(p, s, i_last);
    const int key_first = (low.first > from ? low.first : from) & ~15;  // from is a multiple of 16
    const int key_end = high.end < to ? high.end : to;

    // Of row l % 16; l of this lane's entries alone. A row that there is none of has
    // no scores, and no maximum to look after either.
    float m = mine ? kSeed : 0.0f, l = 0.0f;
    f32x4 o[F::pieces];
#pragma unroll
    for (int c = 0; c < F::pieces; ++c) o[c] = f32x4{0, 0, 0, 0};

    int key0 = nth < heads ? key_first + wave % per_head * F::keys : key_end;
    if (key0 < key_end) {
      const int kStep = per_head * F::keys;
      uint64_t present[2];
      ask<F>(p, table, key0, kStep, key_end, own, lane);
      // q's columns as K's bytes lie: of each 64, 16 of a lane, in two steps.
      u32x4 q[D / 32][kParts];
      const row_t *qp = static_cast<const row_t *>(p.q) + ((int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d);
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const int col = 64 * (c / 2) + 16 * h + 8 * (c % 2);
        // From an address that is there in any case.
        load_q(q[c], qp + within(col, d), mine && col < d, p);
      }
      arrived<0>();
      place<F>(p, kbase, vbase, key0, kStep, key_end, own, lane);
      int placed = 0;  // blocks from the first of those placed to this one
      read_out();
      if (key_end - key0 > F::ahead * kStep) ask<F>(p, table, key0 + F::ahead * kStep, kStep, key_end, own, lane);
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        present[n] = there_of<F>(own, n);
        send<F>(p, own, n, 0, k_off, kscales, own + F::k_at + n * F::block, own + F::scales_at + n * 256, lane);
        send<F>(p, own, n, 1, v_off, vscales, own + F::v_at + n * F::block, own + F::scales_at + 512 + n * 256, lane);
      }
      for (int n = 0; key0 < key_end; ++n, key0 += kStep) {
        const int b = n & 1;
        first_half -= kStep;
        if (first_half < 0) __builtin_amdgcn_s_setprio(0);
        const uint64_t here = present[0];
        // Of K, V of this block, K, V of the next: all but the first may be on their way.
        arrived<3 * F::ops>();
        const char *kb = own + F::k_at + b * F::block;
        powers[lane] = power_of((uint8_t)own[F::scales_at + b * 256 + lane % F::keys]);
        float y[F::mine];
#pragma unroll
        for (int t = 0; t < F::tiles; ++t) {
          f32x4 x = {0, 0, 0, 0};
          const float power = powers[16 * t + r];
          const char *row = kb + (16 * t + r) * D;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(row + 16 * ((4 * c + h) ^ k_swap<D>(r)));
            const u32x4 a0 = {widen<false>(w.x, power), widen<true>(w.x, power), widen<false>(w.y, power), widen<true>(w.y, power)};
            const u32x4 a1 = {widen<false>(w.z, power), widen<true>(w.z, power), widen<false>(w.w, power), widen<true>(w.w, power)};
#pragma unroll
            for (int n1 = 0; n1 < kParts; ++n1) x = mma16(a0, q[2 * c][n1], x);
#pragma unroll
            for (int n1 = 0; n1 < kParts; ++n1) x = mma16(a1, q[2 * c + 1][n1], x);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * t + e] = x[e];
        }
        // The block after the next takes this one's place. The page numbers of the
        // next `ahead` blocks were asked for as many ago.
        if (placed + 2 == F::ahead && key_end - key0 > 2 * kStep) [[unlikely]] {
          place<F>(p, kbase, vbase, key0 + 2 * kStep, kStep, key_end, own, lane);
          placed = -2;
          read_out();
          if (key_end - key0 > (2 + F::ahead) * kStep) ask<F>(p, table, key0 + (2 + F::ahead) * kStep, kStep, key_end, own, lane);
        }
        const int then = key_end - key0 > 2 * kStep ? placed + 2 : F::ahead;
        ++placed;
        present[0] = present[1], present[1] = there_of<F>(own, then);
        read_out();
        send<F>(p, own, then, 0, k_off, kscales, kb, own + F::scales_at + b * 256, lane);

        if (p.cap_in != 0.0f) [[unlikely]] {
          cap<F::mine>(y, p, true);
        }
        // Every row sees every entry of the block: no mask.
        const bool whole = here == ~uint64_t(0) >> (64 - F::keys) && key0 + F::keys <= low.end && key0 >= high.first;
        if (!whole) [[unlikely]] {
          const uint64_t sees = (mine ? seen_of(seen, key0) & here : 0) >> 4 * h;
#pragma unroll
          for (int j = 0; j < F::mine; ++j) y[j] = (sees >> (16 * (j / 4) + j % 4) & 1) != 0 ? y[j] : -__builtin_inff();
        }
        float top = y[0];
#pragma unroll
        for (int j = 1; j < F::mine; ++j) top = fmaxf(top, y[j]);
        top = fmaxf(m, over_rows(top, true) * factor0);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) [[unlikely]] {
          const float fade = exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int c = 0; c < F::pieces; ++c) o[c] *= fade;
        }
        const bool far = coarse(m);
        const float factor = far ? 1.0f : factor0, shift = far ? 0.0f : -m;
        if (far) [[unlikely]] less<F::mine>(y, factor0, m);
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < F::mine; ++j) {
          y[j] = exp2_hw(fmaf(y[j], factor, shift));
          sum += y[j];
        }
        l += sum;

        // Of V of this block, K, V of the next, K of the one after it.
        arrived<3 * F::ops>();
        char *vb = own + F::v_at + b * F::block;
        powers[64 + lane] = power_of((uint8_t)own[F::scales_at + 512 + b * 256 + lane % F::keys]);
        if (!whole) [[unlikely]] {
          // NaN in V where rows differ in what they see: 0 x V would reach the rows
          // that do not. They are added to the rows that do see them, and leave the
          // products as zeros.
#pragma unroll 1
          for (int at16 = 0; at16 < F::block; at16 += 1024) {
            u32x4 *mine16 = reinterpret_cast<u32x4 *>(vb + at16 + 16 * lane);
            const u32x4 w = *mine16;
            const bool odd = (nan_bytes(w.x) | nan_bytes(w.y) | nan_bytes(w.z) | nan_bytes(w.w)) != 0;
            uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
            if (odds == 0) continue;
            while (odds != 0) {
              const int in1024 = __builtin_ctzll(odds) / F::pieces;
              odds &= ~(((uint64_t(1) << F::pieces) - 1) << (in1024 * F::pieces));
              const int row = at16 / D + in1024, key = key0 + row;
              if (!(mine && key >= seen.first && key < seen.end)) continue;
#pragma unroll
              for (int c = 0; c < F::pieces; ++c) {
                const uint32_t n4 = nan_bytes(*reinterpret_cast<const uint32_t *>(vb + row * D + 16 * (c ^ v_swap<D>(row)) + 4 * h));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if ((n4 >> 8 * e & 0x80u) != 0) o[c][e] = __builtin_nanf("");
              }
            }
            *mine16 = u32x4{without_nan(w.x), without_nan(w.y), without_nan(w.z), without_nan(w.w)};
          }
        }
        // The row that lane 2 x + c of 16 points at, of 32 entries: x % 4 of the
        // lane's four of each 16.
        const int across = 16 * (r / 8) + 4 * h + r / 2 % 4;
#pragma unroll
        for (int g = 0; g < F::tiles / 2; ++g) {
          u32x4 bp[kParts];
          const f32x4 p0 = *reinterpret_cast<const f32x4 *>(powers + 64 + 32 * g + 4 * h);
          const f32x4 p1 = *reinterpret_cast<const f32x4 *>(powers + 64 + 32 * g + 16 + 4 * h);
          float eight[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) eight[j] = y[8 * g + j] * p0[j], eight[4 + j] = y[8 * g + 4 + j] * p1[j];
          in_parts(bp, eight, false);
          const char *row = vb + (32 * g + across) * D + 8 * (r % 2);
#pragma unroll
          for (int c = 0; c < F::pieces; ++c) {
            const u32x2 w = read_across8(row + 16 * (c ^ v_swap<D>(across)));
            const u32x4 a = {widen<false>(w.x, 1.0f), widen<true>(w.x, 1.0f), widen<false>(w.y, 1.0f), widen<true>(w.y, 1.0f)};
#pragma unroll
            for (int n1 = 0; n1 < kParts; ++n1) o[c] = mma16(a, bp[n1], o[c]);
          }
        }
        read_out();
        send<F>(p, own, then, 1, v_off, vscales, vb, own + F::scales_at + 512 + b * 256, lane);
      }
    }

    // Join the waves: rescale to the rows' common maximum, add in wave order.
    l = over_rows(l, false);
    vm_wait<0>();
    lds_barrier();  // everyone's last loads have come to LDS
    if (h == 0) {
      ml[(wave * kRows + r) * 2] = m;
      ml[(wave * kRows + r) * 2 + 1] = l;
    }
    lds_barrier();
    const int wave0 = nth * per_head;  // the head's first wave
    float top = kSeed;
    for (int w = 0; w < per_head; ++w) top = fmaxf(top, ml[((wave0 + w) * kRows + r) * 2]);
    float total = 0.0f;
    for (int w = 0; w < per_head; ++w) total += ml[((wave0 + w) * kRows + r) * 2 + 1] * exp2_hw(ml[((wave0 + w) * kRows + r) * 2] - top);
    const float fade = exp2_hw(m - top);
#pragma unroll
    for (int c = 0; c < F::pieces; ++c) *reinterpret_cast<f32x4 *>(part + (wave * kRows + r) * kPitch + 16 * c + 4 * h) = o[c] * fade;
    if (wave == wave0 && nth < heads && h == 0) {
      both[2 * (nth * kRows + r)] = top, both[2 * (nth * kRows + r) + 1] = total;
      if (!alone) {
        float *ml_to = p.part_ml + ((((int64_t)block * 2 + slot) * p.together + nth) * kRows + r) * 2;
        ml_to[0] = top;
        ml_to[1] = total;
      }
    }
    lds_barrier();
    for (int x = threadIdx.x; x < heads * kRows * (D / 4); x += WAVES * kWave) {
      const int of = x / (kRows * (D / 4)), row = x / (D / 4) % kRows, col = x % (D / 4) * 4, RR = row0 + row;
      if (RR >= rows || col >= d) continue;
      const int ii = (int)kh_div(RR, p.by_group), hh = (head0 + of) * p.group + RR - ii * p.group;
      f32x4 y = {0, 0, 0, 0};
      for (int w = 0; w < per_head; ++w) y += *reinterpret_cast<const f32x4 *>(part + ((of * per_head + w) * kRows + row) * kPitch + col);
      if (alone)
        finish(p, s.start + ii, hh, col, y, both[2 * (of * kRows + row)], both[2 * (of * kRows + row) + 1]);
      else
        *reinterpret_cast<f32x4 *>(p.part_o + ((((int64_t)block * 2 + slot) * p.together + of) * kRows + row) * d + col) = y;
    }
    lds_barrier();  // before the next unit's loads come to the join area
  }
}

// ---- many rows: chunks of prompts, and entries that all sequences share

template <int D>
struct Many {
  static constexpr int bytes = 2 * D;                 // of a row in LDS
  static constexpr int steps = bytes / 32;
  static constexpr int keys = 64, tiles = keys / 32;  // entries of a tile
  static constexpr int dts = D / 32;
  static constexpr int pieces = D / 16;               // of 16 bytes of a row of the cache
  static constexpr int rows = 256 / pieces, passes = keys / rows;  // rows that the workgroup brings at a time
  static constexpr int v_at = keys * bytes, marks_at = 2 * v_at, buffer = marks_at + keys;
  static constexpr int lds = 2 * buffer;
  // The columns of piece n of eight of a row in LDS. A thread brings sixteen: the first
  // eight of all threads come before the second ones, so that neighbours write to
  // neighbouring banks (a chunk of 2048 at 8192 entries 288 us, in the columns' own
  // order 295).
  static __device__ constexpr int column(int n) { return n < pieces ? 16 * n : 16 * (n - pieces) + 8; }
};
static_assert(Rows<64>::tile == 64 && Rows<128>::tile == 64 && Rows<256>::tile == 64);

constexpr uint8_t kThere = 1, kOdd = 2;  // marks of a row in LDS

// A tile on its way: a thread brings 16 bytes of a row of K and of V in each pass.
template <int D>
struct Tile {
  KhSlot found[Many<D>::passes], at[Many<D>::passes];
  u32x4 k[Many<D>::passes], v[Many<D>::passes];
  uint32_t k_scale[Many<D>::passes], v_scale[Many<D>::passes];
};

template <int D>
__device__ __forceinline__ void seek(Tile<D> &g, const KhAttention8Params &p, const int32_t *table, int key0, int end, int tid) {
  using W = Many<D>;
#pragma unroll
  for (int i = 0; i < W::passes; ++i) g.found[i] = look_up<false>(p, table, key0 + i * W::rows + tid / W::pieces, end);
}

// Starts the loads of the tile that was sought.
template <int D>
__device__ __forceinline__ void fetch(Tile<D> &g, const KhAttention8Params &p, int head, int key0, int end, int tid) {
  using W = Many<D>;
  const int own = tid / W::pieces;
  const uint32_t off = within(16 * (tid % W::pieces), p.cache.head_dim);
  const uint64_t scale0 = (uint64_t)head * p.scale_head;
  const char *kbase = p.cache.k + (uint64_t)head * p.cache.k_head, *vbase = p.cache.v + (uint64_t)head * p.cache.v_head;
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const bool there = key0 + i * W::rows + own < end && (uint32_t)g.found[i].page < (uint32_t)p.cache.pages;
    g.at[i] = there ? g.found[i] : KhSlot{-1, 0};
    const KhSlot at = there ? g.found[i] : KhSlot{0, 0};
    g.k[i] = *reinterpret_cast<const u32x4 *>(kbase + kh_row(at, p.cache.k_page, p.cache.k_slot) + off);
    g.v[i] = *reinterpret_cast<const u32x4 *>(vbase + kh_row(at, p.cache.v_page, p.cache.v_slot) + off);
    const uint64_t scale = scale0 + (uint64_t)(uint32_t)at.page * p.scale_page + (uint32_t)at.slot;
    g.k_scale[i] = p.k_scale[scale];
    g.v_scale[i] = p.v_scale[scale];
  }
}

// Sixteen numbers as two pieces of eight in bf16.
__device__ __forceinline__ void widen16(u32x4 &a, u32x4 &b, u32x4 w, float power) {
  a = u32x4{widen<false>(w.x, power), widen<true>(w.x, power), widen<false>(w.y, power), widen<true>(w.y, power)};
  b = u32x4{widen<false>(w.z, power), widen<true>(w.z, power), widen<false>(w.w, power), widen<true>(w.w, power)};
}

// From registers to LDS as bf16. Columns past the row's end are copies of its first:
// q has zeros there, and nobody takes them from O. Absent rows of K have no score; of V
// they are zeros. Where rows of the unit see different entries of the tile (mixed), NaN
// in V become zeros and their row is marked.
template <int D>
__device__ __forceinline__ void put(const Tile<D> &g, char *buffer, bool mixed, int tid) {
  using W = Many<D>;
  const int own = tid / W::pieces, piece = tid % W::pieces, lane = lane_id();
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const int row = i * W::rows + own;
    const bool there = g.at[i].page >= 0;
    u32x4 v = g.v[i];
    uint8_t mark = there ? kThere : 0;
    if (__builtin_amdgcn_ballot_w64(!there) != 0) [[unlikely]] v = there ? v : u32x4{0, 0, 0, 0};
    if (mixed) [[unlikely]] {
      const bool odd = (nan_bytes(v.x) | nan_bytes(v.y) | nan_bytes(v.z) | nan_bytes(v.w)) != 0;
      const uint64_t odds = __builtin_amdgcn_ballot_w64(odd);
      if (odds != 0) {
        v = u32x4{without_nan(v.x), without_nan(v.y), without_nan(v.z), without_nan(v.w)};
        if ((odds >> (lane - piece) & ((uint64_t(1) << W::pieces) - 1)) != 0) mark |= kOdd;
      }
    }
    u32x4 a, b;
    widen16(a, b, g.k[i], power_of(g.k_scale[i]));
    char *to = buffer + row * W::bytes;
    *reinterpret_cast<u32x4 *>(to + 16 * (piece ^ k_turn<D>(row))) = a;
    *reinterpret_cast<u32x4 *>(to + 16 * (W::pieces + piece ^ k_turn<D>(row))) = b;
    widen16(a, b, v, power_of(g.v_scale[i]));
    to += W::v_at;
    *reinterpret_cast<u32x4 *>(to + 16 * (piece ^ v_turn<D>(row))) = a;
    *reinterpret_cast<u32x4 *>(to + 16 * (W::pieces + piece ^ v_turn<D>(row))) = b;
    if (piece == 0) buffer[W::marks_at + row] = (char)mark;
  }
}

// A operand of V^T for columns 32 dt .. and 16 entries, half c of 32.
template <int D>
__device__ __forceinline__ u32x4 v_across(const char *buffer, int kt, int c, int dt, int lane) {
  using W = Many<D>;
  const int r = (lane & 15) / 4, turn = Rows<D>::pieces == 8 ? r >> 1 : r;
  const char *at = buffer + W::v_at + (32 * kt + 16 * c + 4 * (lane >> 5) + r) * W::bytes + 64 * (dt ^ turn) + 32 * (lane >> 4 & 1) +
                   8 * (lane & 3);
  const u32x2 lo = read_across(at), hi = read_across(at + 8 * W::bytes);
  return u32x4{lo.x, lo.y, hi.x, hi.y};
}

// Least and most of a value over the wave.
__device__ __forceinline__ int least(int v) {
#pragma unroll
  for (int n = 1; n < kWave; n *= 2) {
    const int w = __shfl_xor(v, n, kWave);
    v = w < v ? w : v;
  }
  return __builtin_amdgcn_readfirstlane(v);
}

// Block `block` of the wide ones; `common`: of those over the entries that all
// sequences share.
template <int D>
__device__ __forceinline__ void wide(const KhAttention8Params &p, int block, bool common, char *lds) {
  using W = Many<D>;
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 31, h = lane >> 5;
  const int d = p.cache.head_dim;
  const int splits = common ? p.shared_splits : p.wide_splits;
  const int split = block % splits, unit = block / splits;

  // The lane's row, what it sees, and the entries of this part.
  int head, token = 0, hq, seq = 0;
  bool mine, nobody = false, alone;
  KhSpan seen = {0, 0};
  KhPart part;
  if (common) {
    if (p.shared == 0) return;
    head = unit % p.cache.kv_heads;
    const int R = unit / p.cache.kv_heads * kWideTile + wave * kWideRows + r, rows = p.tokens * p.group;
    const bool row = R < rows;
    token = row ? (int)kh_div(R, p.by_group) : 0;
    hq = head * p.group + (row ? R - token * p.group : 0);
    const int of = kh_sequence_of(p.q_starts, p.table.seqs, token);
    const KhSeq s = sequence(p, of);
    const int i = token - s.start;
    mine = row && i >= 0 && i < s.m;
    nobody = row && !mine;
    if (mine) {
      seen = kh_seen(s, i, p.window);
      seen.end = seen.end < p.shared ? seen.end : p.shared;
    }
    alone = false;
    part = KhPart{split * p.shared_each, (split + 1) * p.shared_each < p.shared ? (split + 1) * p.shared_each : p.shared, splits};
  } else {
    KhSeq s;
    int before;
    const Line line = line_of(p, true);
    if (unit >= line.all) return;
    seq = sequence_at(p, line, unit, true, s, before);
    if (seq < 0) return;
    const WideUnit u = wide_unit(p, s, unit - before);
    part = kh_part(u.first, u.end, splits, split);
    if (split >= part.used) return;
    alone = part.used == 1;
    head = u.head;
    const int R = u.tile0 + wave * kWideRows + r;
    mine = R < u.tile_end;
    const int i = mine ? (int)kh_div(R, p.by_group) : 0;
    token = s.start + i;
    hq = head * p.group + (mine ? R - i * p.group : 0);
    if (mine) seen = kh_span_of(p, s, i);
  }
  const bool any = __builtin_amdgcn_ballot_w64(mine) != 0;
  // Least and most of the rows' spans, of the wave and of the workgroup.
  constexpr int kFar = 0x7fffffff;
  const KhSpan low = {least(mine ? seen.first : kFar), least(mine ? seen.end : kFar)};
  const KhSpan high = {-least(mine ? -seen.first : kFar), -least(mine ? -seen.end : kFar)};
  int *spans = reinterpret_cast<int *>(lds);
  if (lane == 0) {
    int *to = spans + 4 * wave;
    to[0] = low.first, to[1] = low.end, to[2] = any ? high.first : -kFar, to[3] = any ? high.end : -kFar;
  }
  lds_barrier();
  int all_end = kFar, all_first = -kFar, part_first = kFar, part_end = -kFar;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int *s = spans + 4 * w;
    part_first = s[0] < part_first ? s[0] : part_first;
    all_end = s[1] < all_end ? s[1] : all_end;
    all_first = s[2] > all_first ? s[2] : all_first;
    part_end = s[3] > part_end ? s[3] : part_end;
  }
  part_first = __builtin_amdgcn_readfirstlane(part_first), all_end = __builtin_amdgcn_readfirstlane(all_end);
  all_first = __builtin_amdgcn_readfirstlane(all_first), part_end = __builtin_amdgcn_readfirstlane(part_end);
  lds_barrier();
  // Tiles that none of the rows sees are passed over.
  if (part_end < part.end) part.end = part_end;
  if (part_first > part.first) part.first = part_first < part.end ? part_first & ~15 : part.end;

  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const char *vbase = p.cache.v + (uint64_t)head * p.cache.v_head;
  const float factor0 = p.cap_in != 0.0f ? p.cap_out : p.scale_log2;

  u32x4 q[W::steps][kParts];
  const row_t *qp = static_cast<const row_t *>(p.q) + ((int64_t)token * p.q_stride + (int64_t)hq * d);
#pragma unroll
  for (int c = 0; c < W::steps; ++c) {
    const int col = W::column(2 * c) + 16 * h;
    load_q(q[c], qp + within(col, d), mine && col < d, p);
  }
  float m = mine ? kSeed : 0.0f, l = 0.0f;
  f32x16 o[W::dts];
#pragma unroll
  for (int a = 0; a < W::dts; ++a) o[a] = f32x16{};

  // Whether rows of the unit differ in what they see of the tile at key0.
  auto mixed = [&](int key0) { return key0 + W::keys > all_end || key0 < all_first; };
  if (part.first < part.end) {
    Tile<D> g;
    seek<D>(g, p, table, part.first, part.end, tid);
    fetch<D>(g, p, head, part.first, part.end, tid);
    seek<D>(g, p, table, part.first + W::keys, part.end, tid);
    int cur = 0;
    for (int key0 = part.first; key0 < part.end; key0 += W::keys, cur ^= 1) {
      char *buffer = lds + cur * W::buffer;
      put<D>(g, buffer, mixed(key0), tid);
      // The page numbers of the tile after the next go out behind its loads.
      fetch<D>(g, p, head, key0 + W::keys, part.end, tid);
      seek<D>(g, p, table, key0 + 2 * W::keys, part.end, tid);
      // One barrier: this tile is there for everyone, and everyone is done with
      // the tile whose place the next one takes.
      lds_barrier();
      // Nothing to do for a wave none of whose rows sees any of the tile.
      if (any && key0 < high.end && key0 + W::keys > low.first) {
        f32x16 x[W::tiles];
#pragma unroll
        for (int kt = 0; kt < W::tiles; ++kt) x[kt] = f32x16{};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < W::steps; ++c)
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) {
            const u32x4 a = k_rows<D>(buffer, kt, c, lane);
#pragma unroll
            for (int n = 0; n < kParts; ++n) x[kt] = mma32(a, q[c][n], x[kt]);
          }
        if constexpr (kParts == 1) read_ahead<W::steps * W::tiles, W::steps * W::tiles, 1, 6>();
        __builtin_amdgcn_s_setprio(0);
        const uint32_t mark = (uint8_t)buffer[W::marks_at + lane];
        const uint64_t present = __builtin_amdgcn_ballot_w64((mark & kThere) != 0);
        const uint64_t odds = mixed(key0) ? __builtin_amdgcn_ballot_w64((mark & kOdd) != 0) : 0;
        if (p.cap_in != 0.0f) [[unlikely]] {
          const bool near = p.cap_near || low.end <= KH_FEW_CAPPED;
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) {
            if (near)
              cap<16>(x[kt], p, true);
            else
              cap<16>(x[kt], p, false);
          }
        }
        const bool whole = present == ~uint64_t(0) && key0 + W::keys <= low.end && key0 >= high.first;
        if (!whole) [[unlikely]] {
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
        top = fmaxf(m, over_halves(top, true) * factor0);
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) [[unlikely]] {
          const float fade = exp2_hw(m - top);
          m = top;
          l *= fade;
#pragma unroll
          for (int a = 0; a < W::dts; ++a) o[a] *= fade;
        }
        const bool far = coarse(m);
        const float factor = far ? 1.0f : factor0, shift = far ? 0.0f : -m;
        if (far) [[unlikely]] {
#pragma unroll
          for (int kt = 0; kt < W::tiles; ++kt) less<16>(x[kt], factor0, m);
        }
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < W::tiles; ++kt)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            x[kt][j] = exp2_hw(fmaf(x[kt][j], factor, shift));
            sum += x[kt][j];
          }
        l += sum;
        // As in narrow(): what was kept out of the products.
        if (odds != 0) [[unlikely]]
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
                const int col = W::column(4 * dt + j / 4) + 4 * h1;
                if (col >= d) continue;
                const uint32_t odd = nan_bytes(*reinterpret_cast<const uint32_t *>(row + col));
#pragma unroll
                for (int b = 0; b < 4; ++b)
                  if ((odd >> 8 * b & 0x80u) != 0) o[dt][j + b] = __builtin_nanf("");
              }
          }
        }
        __builtin_amdgcn_s_setprio(1);
        // Operands of V are read a step ahead of their products.
        constexpr int kAll = W::tiles * 2;
        u32x4 a[2][W::dts];
#pragma unroll
        for (int dt = 0; dt < W::dts; ++dt) a[0][dt] = v_across<D>(buffer, 0, 0, dt, lane);
#pragma unroll
        for (int n = 0; n < kAll; ++n) {
          if (n + 1 < kAll) {
#pragma unroll
            for (int dt = 0; dt < W::dts; ++dt) a[(n + 1) % 2][dt] = v_across<D>(buffer, (n + 1) / 2, (n + 1) % 2, dt, lane);
          }
          __builtin_amdgcn_sched_barrier(0);
          const f32x16 &y = x[n / 2];
          const int j0 = 8 * (n % 2);
          const float eight[8] = {y[j0], y[j0 + 1], y[j0 + 2], y[j0 + 3], y[j0 + 4], y[j0 + 5], y[j0 + 6], y[j0 + 7]};
          u32x4 b[kParts];
          in_parts(b, eight, false);
#pragma unroll
          for (int dt = 0; dt < W::dts; ++dt)
#pragma unroll
            for (int i = 0; i < kParts; ++i) o[dt] = mma32(a[n % 2][dt], b[i], o[dt]);
        }
        __builtin_amdgcn_s_setprio(0);
      }
    }
  }

  const float total = over_halves(l, false);
  const int64_t rows = (int64_t)p.tokens * p.q_heads, row = (int64_t)token * p.q_heads + hq;
  float *part_o = common ? p.shared_o : p.wide_o, *part_ml = common ? p.shared_ml : p.wide_ml;
  const int64_t at_row = (int64_t)split * rows + row;
  if (nobody && h == 0) part_ml[2 * at_row + 1] = -1.0f;  // combine() leaves such a row alone
  if (!mine) return;
  if (!alone && h == 0) part_ml[2 * at_row] = m, part_ml[2 * at_row + 1] = total;
#pragma unroll
  for (int dt = 0; dt < W::dts; ++dt)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int col = W::column(4 * dt + j / 4) + 4 * h;
      if (col >= d) continue;
      const f32x4 y = {o[dt][j], o[dt][j + 1], o[dt][j + 2], o[dt][j + 3]};
      if (alone)
        finish(p, token, hq, col, y, m, total);
      else
        *reinterpret_cast<f32x4 *>(part_o + at_row * d + col) = y;
    }
}

// Joins what the shared entries' parts and the sequences' own entries gave each row:
// D / 4 lanes to a row, four columns each. Its statistics come a part to a lane, and
// with them the first rows.
template <int D>
__device__ __forceinline__ void combine(const KhAttention8Params &p) {
  constexpr int kLanes = D / 4, kAhead = 16;
  const int d = p.cache.head_dim, lane = threadIdx.x % kLanes, col = lane * 4, count = p.shared_splits + 1;
  const int64_t rows = (int64_t)p.tokens * p.q_heads;
  const int64_t at = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int64_t row = at < rows ? at : rows - 1;
  const float *ml = p.shared_ml + 2 * row, *from = p.shared_o + row * d + (col < d ? col : 0);
  f32x4 x[kAhead];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) x[j] = *reinterpret_cast<const f32x4 *>(from + (int64_t)(k0 + j < count ? k0 + j : count - 1) * rows * d);
  };
  fetch(0);
  const bool nobodys = ml[1] < 0.0f;
  float top = kSeed, total = 0.0f;
  for (int k = lane; k < count; k += kLanes) top = fmaxf(top, ml[2 * (int64_t)k * rows]);
#pragma unroll
  for (int n = 1; n < kLanes; n *= 2) top = fmaxf(top, __shfl_xor(top, n, kWave));
  f32x4 o = {0, 0, 0, 0};
  for (int k0 = 0; k0 < count; k0 += kLanes) {
    const int mine = k0 + lane < count ? k0 + lane : count - 1;
    const float w = k0 + lane < count ? exp2_hw(ml[2 * (int64_t)mine * rows] - top) : 0.0f;
    total += ml[2 * (int64_t)mine * rows + 1] * w;
    for (int k1 = k0; k1 < count && k1 < k0 + kLanes; k1 += kAhead) {
      if (k1 != 0) fetch(k1);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const float f = __shfl(w, (int)(threadIdx.x % kWave / kLanes * kLanes) + (k1 - k0 + j) % kLanes, kWave);
        if (k1 + j < count) o += x[j] * f;
      }
    }
  }
#pragma unroll
  for (int n = 1; n < kLanes; n *= 2) total += __shfl_xor(total, n, kWave);
  // Every lane takes part in the exchanges above.
  if (p.shared == 0 || at >= rows || nobodys || col >= d) return;
  const int token = (int)(row / p.q_heads), hq = (int)(row - (int64_t)token * p.q_heads);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  const float y[4] = {o.x * inv, o.y * inv, o.z * inv, o.w * inv};
  store_row(static_cast<row_t *>(p.out) + (int64_t)token * p.out_stride + (int64_t)hq * d + col, y);
  if (col == 0 && p.lse != nullptr) p.lse[row] = lse_of(top, total, 0.0f);
}

constexpr int kJoinMost = 128;

struct JoinLds {
  float weights[kJoinMost * kRows];  // of a part's row against the row's maximum so far
  float tops[kWaves * kRows], fades[kRows], totals[kWaves * kRows];
  float sums[256 * 4];
};

// Joins the parts of 16 rows. They were written through other L2s, so that each round
// of loads takes its time: the statistics of AT parts and AHEAD of its rows come to a
// thread in one. Statistics lie a part's row to a lane, which works out what the row
// counts for once for all columns. A thread has 4 columns of a row, and where that
// leaves threads over (few rows), only each second to eighth part of it.
template <int D, int AT, int AHEAD>
__device__ __forceinline__ void join_rows(const KhAttention8Params &p, JoinLds &lds, const KhSeq &s, const Parts &parts) {
  constexpr int kMine = AT * kRows / 256;
  const int shift = __builtin_ctz(D / 4) - __builtin_ctz(gridDim.y), cols = 1 << shift;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid / kWave, d = p.cache.head_dim;
  auto base = [&](int k) { return k == 0 ? parts.first : parts.others + (k - 1) * parts.step; };
  auto place_of = [&](int row) {
    if (!parts.wide) return (int64_t)row;
    const int R = parts.R0 + row, i = (int)kh_div(R, p.by_group);
    return (int64_t)(s.start + i) * p.q_heads + parts.head * p.group + R - i * p.group;
  };
  // Rows rounded up to a power of two, times columns: items; threads that share one.
  const int rows2 = parts.rows <= 1 ? 1 : parts.rows <= 2 ? 2 : parts.rows <= 4 ? 4 : parts.rows <= 8 ? 8 : 16;
  const int items = rows2 * cols, shares = items >= 256 ? 1 : 256 / items < 8 ? 256 / items : 8;
  const int own = tid % kRows;  // whose statistics the thread has, of parts tid / 16, ..
  const float *ml = parts.ml + 2 * place_of(own < parts.rows ? own : 0);
  for (int item0 = 0; item0 < items; item0 += 256) {
    const int share = tid / items, item = item0 + tid % items;  // item0 > 0: shares = 1
    const int row = item >> shift, col = (item & (cols - 1)) * 4 + (int)blockIdx.y * 4 * cols;
    const bool live = row < parts.rows && col < d && share < shares;
    const float *from = parts.o + place_of(live ? row : 0) * d + (live ? col : 0);
    f32x4 o = {0, 0, 0, 0};
    float m = kSeed, total = 0.0f;  // of row `own`
    for (int k0 = 0; k0 < parts.count; k0 += AT) {
      const int here = parts.count - k0 < AT ? parts.count - k0 : AT;
      f32x4 x[AHEAD];
      auto fetch = [&](int k1) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int k = k1 + j * shares;
          x[j] = *reinterpret_cast<const f32x4 *>(from + base(k0 + (k < here ? k : here - 1)) * d);
        }
      };
      // The first rows come with the statistics.
      if (live) fetch(share);
      f32x2 mine[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int k = tid / kRows + 256 / kRows * i;
        mine[i] = *reinterpret_cast<const f32x2 *>(ml + 2 * base(k0 + (k < here ? k : here - 1)));
        if (k >= here) mine[i] = f32x2{kSeed, 0.0f};
      }
      float top = mine[0].x;
#pragma unroll
      for (int i = 1; i < kMine; ++i) top = fmaxf(top, mine[i].x);
#pragma unroll
      for (int n = kRows; n < kWave; n *= 2) top = fmaxf(top, __shfl_xor(top, n, kWave));
      if (lane < kRows) lds.tops[wave * kRows + lane] = top;
      lds_barrier();
      top = m;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) top = fmaxf(top, lds.tops[w * kRows + own]);
      const float fade = exp2_hw(m - top);
      m = top, total *= fade;
      if (tid < kRows) lds.fades[tid] = fade;
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const float weight = exp2_hw(mine[i].x - top);
        total += mine[i].y * weight;
        lds.weights[256 * i + tid] = weight;
      }
      lds_barrier();
      if (live) {
        o *= lds.fades[row];
        for (int k1 = share; k1 < here; k1 += AHEAD * shares) {
          if (k1 != share) fetch(k1);
#pragma unroll
          for (int j = 0; j < AHEAD; ++j) {
            const int k = k1 + j * shares;
            if (k < here) o += x[j] * lds.weights[k * kRows + row];
          }
        }
      }
      lds_barrier();
    }
#pragma unroll
    for (int n = kRows; n < kWave; n *= 2) total += __shfl_xor(total, n, kWave);
    if (lane < kRows) lds.totals[wave * kRows + lane] = total, lds.tops[wave * kRows + lane] = m;
    if (shares > 1) *reinterpret_cast<f32x4 *>(lds.sums + 4 * tid) = o;
    lds_barrier();
    if (live && share == 0) {
      // The shares' sums, in their order.
      for (int k = 1; k < shares; ++k) o += *reinterpret_cast<const f32x4 *>(lds.sums + 4 * (tid + k * items));
      float all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) all += lds.totals[w * kRows + row];
      const int R = parts.R0 + row, i = (int)kh_div(R, p.by_group);
      finish(p, s.start + i, parts.head * p.group + R - i * p.group, col, o, lds.tops[row], all);
    }
    lds_barrier();
  }
}

// A workgroup for every workgroup's start and head, as that one told it, then one for
// each 16 rows of the wide units; a grid's y shares out the columns. Parts of up to
// 16 take fewer loads: four sequences of 2000 entries 16.6 us, by the other form 18.3
template <int D>
__device__ __forceinline__ void join_told(const KhAttention8Params &p, JoinLds &lds) {
  constexpr int kPer = kWideTile / kRows;
  const int narrow_blocks = p.whole ? 0 : p.groups * p.together, block = (int)blockIdx.x - narrow_blocks;
  KhSeq s{0, 0, 0};
  Parts parts{};
  if (!(block < 0 ? told_parts(p, (int)blockIdx.x, s, parts) : wide_parts(p, block / kPer, block % kPer * kRows, s, parts))) return;
  if (parts.count <= 16)
    join_rows<D, 16, 4>(p, lds, s, parts);
  else
    join_rows<D, kJoinMost, 16>(p, lds, s, parts);
}

// As far as sequence 0 reaches: its row of the table is the one that is read.
__device__ __forceinline__ void settle_shared(KhAttention8Params &p) {
  if (p.shared == 0) return;
  const int n = kh_clamp(scalar_load(p.table.lens), 0, p.table.capacity);
  p.shared = n < p.shared ? n : p.shared;
}

}  // namespace

#if KH_ROWS == 0
#define KH_TYPED8(name) KH_PASTE(name, f32)
#elif KH_ROWS == 1
#define KH_TYPED8(name) KH_PASTE(name, f16)
#else
#define KH_TYPED8(name) KH_PASTE(name, bf16)
#endif

#define KH_ATTENTION8(D, WAVES, PER_CU)                                                                                 \
  extern "C" __global__ void __launch_bounds__(64 * WAVES, PER_CU) KH_TYPED8(attention8_##D)(KhAttention8Params p) { \
    __shared__ __attribute__((aligned(16))) char lds[WAVES * Ring<D>::lds];                                          \
    narrow_even<D, WAVES>(p, (int)blockIdx.x, lds);                                                                  \
  }
KH_ATTENTION8(64, 4, 2)
KH_ATTENTION8(128, 4, 2)
KH_ATTENTION8(256, 2, 1)
#define KH_ATTENTION8_ODD(D, PER_CU)                                                                               \
  extern "C" __global__ void __launch_bounds__(256, PER_CU) KH_TYPED8(attention8_odd_##D)(KhAttention8Params p) { \
    __shared__ __attribute__((aligned(16))) float lds[kWaves * kRows * 2 + kRows * 2 + kWaves * kRows * (D + 4)]; \
    narrow<D>(p, (int)blockIdx.x, lds);                                                                    \
  }
KH_ATTENTION8_ODD(64, 2)
KH_ATTENTION8_ODD(128, 2)
KH_ATTENTION8_ODD(256, 1)
// Steps with sequences of many rows or shared entries: their workgroups first. fp32
// rows of 128, three parts of each, leave registers for one workgroup to a CU: two
// chunks of 1024 at 4096 entries, 16 heads on 4, 224 us; for two, which spill, 247.
#define KH_ATTENTION8_WIDE(D, PER_CU)                                                                              \
  extern "C" __global__ void __launch_bounds__(256, PER_CU) KH_TYPED8(attention8_wide_##D)(KhAttention8Params p) { \
    constexpr int kFew = kWaves * Ring<D>::lds;                                                                    \
    __shared__ __attribute__((aligned(16))) char lds[Many<D>::lds > kFew ? Many<D>::lds : kFew];                   \
    settle_shared(p);                                                                                              \
    const int block = (int)blockIdx.x, wide_end = p.shared_blocks + p.wide_blocks;                                 \
    if (block < wide_end)                                                                                          \
      wide<D>(p, block < p.shared_blocks ? block : block - p.shared_blocks, block < p.shared_blocks, lds);         \
    else if (p.even)                                                                                               \
      narrow_even<D, kWaves>(p, block - wide_end, lds);                                                            \
    else                                                                                                           \
      narrow<D>(p, block - wide_end, reinterpret_cast<float *>(lds));                                              \
  }
KH_ATTENTION8_WIDE(64, 2)
KH_ATTENTION8_WIDE(128, kParts == 3 ? 1 : 2)
KH_ATTENTION8_WIDE(256, 1)
#define KH_ATTENTION8_JOIN(D)                                                                                   \
  extern "C" __global__ void __launch_bounds__(256) KH_TYPED8(attention8_join_##D)(KhAttention8Params p) {      \
    __shared__ JoinLds lds;                                                                                     \
    settle_shared(p);                                                                                           \
    join_told<D>(p, lds);                                                                                       \
  }                                                                                                             \
  extern "C" __global__ void __launch_bounds__(256) KH_TYPED8(attention8_combine_##D)(KhAttention8Params p) { \
    settle_shared(p);                                                                                           \
    combine<D>(p);                                                                                              \
  }
KH_ATTENTION8_JOIN(64)
KH_ATTENTION8_JOIN(128)
KH_ATTENTION8_JOIN(256)
