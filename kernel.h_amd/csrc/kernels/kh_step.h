// What attention over a paged cache does apart from reading it: how a step is
// shared out over the workgroups, and how parts of rows that several of them
// worked on are joined. Parameters P are KhAttentionParams or go on from them,
// with kh_units_of and kh_span_of of their own.
#pragma once

#include "kh_cache.h"

namespace kh {

constexpr int kRows = KH_TILE_ROWS;
constexpr int kWaves = 4;          // waves of a workgroup; they take blocks of entries in turn
constexpr float kSeed = -3.402823466e38f;  // of the running maximum: no finite score lies below it, and max - max is never NaN
constexpr float kFine = 4194304.0f;        // 2^22, see coarse()

constexpr int kWideRows = 32;                  // of a wave
constexpr int kWideTile = kWaves * kWideRows;  // of a workgroup

// h, worked out where it is used: on a path that is hardly ever taken, what
// follows from it is not to be kept in registers across the loop round it.
__device__ __forceinline__ int apart(int h) {
  asm volatile("" : "+v"(h));
  return h;
}

// 2^x takes scores times a factor less the row's maximum m (in powers of two; in fp16
// paged_attention more its kLift): one multiply-add, exact but for its last rounding,
// while m itself was rounded.
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

template <class P>
__device__ __forceinline__ KhSeq sequence(const P &p, int seq) {
  return kh_seq(p.table.lens[seq], p.q_starts[seq], p.q_starts[seq + 1], p.table.capacity, p.tokens);
}

// The step's blocks, and of the first 64 sequences, one to a lane, what they
// are and how many blocks they have.
struct Line {
  KhSeq s;
  int own, upto, all;
};

// Blocks of the lane's sequence, or units where `wide`; 0 past the last.
template <class P>
__device__ __forceinline__ int work_of(const P &p, int seq, bool wide, KhSeq &s) {
  s = KhSeq{0, 0, 0};
  if (seq < p.table.seqs) s = sequence(p, seq);
  const bool is_wide = s.m * p.group > p.narrow_rows;
  if (is_wide != wide) return 0;
  return wide ? kh_wide_tiles(s, p.group) * p.cache.kv_heads
              : kh_work(kh_units_of(p, s), kh_groups_of(p));
}

template <class P>
__device__ __forceinline__ Line line_of(const P &p, bool wide) {
  const int lane = lane_id();
  Line l;
  l.own = work_of(p, lane, wide, l.s);
  l.upto = up_to(l.own);
  l.all = __builtin_amdgcn_readlane(l.upto, kWave - 1);
  for (int s0 = kWave; s0 < p.table.seqs; s0 += kWave) {
    KhSeq s;
    l.all += __builtin_amdgcn_readlane(up_to(work_of(p, s0 + lane, wide, s)), kWave - 1);
  }
  return l;
}

// The sequence that block x (less than all) is of, and the blocks before that
// sequence. -1 if there is none: starts that do not ascend can make the counts
// wrap, and every walk over the sequences ends at the last one all the same.
template <class P>
__device__ __forceinline__ int sequence_at(const P &p, const Line &l, int x, bool wide, KhSeq &s, int &before) {
  const int lane = lane_id();
  int own = l.own, upto = l.upto;
  KhSeq mine = l.s;
  for (int s0 = 0; s0 < p.table.seqs; s0 += kWave) {
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > x);
    if (past != 0) {
      const int first = __builtin_ctzll(past);
      before = __builtin_amdgcn_readlane(upto - own, first);
      s.n = __builtin_amdgcn_readlane(mine.n, first);
      s.m = __builtin_amdgcn_readlane(mine.m, first);
      s.start = __builtin_amdgcn_readlane(mine.start, first);
      return s0 + first;
    }
    const int sum = __builtin_amdgcn_readlane(upto, kWave - 1);
    own = work_of(p, s0 + kWave + lane, wide, mine);
    upto = sum + up_to(own);
  }
  return -1;
}

// Behind a launch's wide workgroups one to a CU cannot be had: where the idle ones
// of them leave first, two of the others come to lie on one CU beside empty ones.
template <class P>
__device__ __forceinline__ KhShares shares_of(const P &p, const Line &line) {
  return kh_shares(line.all, kh_most_of(p, line.all));
}

// A wide unit: its rows and all entries that any of them sees. A sequence's units
// go from its last tile on: with causal rows the longest first.
struct WideUnit {
  int head, tile0, tile_end, first, end;
};

template <class P>
__device__ __forceinline__ WideUnit wide_unit(const P &p, const KhSeq &s, int in_seq) {
  const int rows = s.m * p.group, turn = in_seq / p.cache.kv_heads;
  WideUnit u;
  u.head = in_seq - turn * p.cache.kv_heads;
  u.tile0 = (kh_wide_tiles(s, p.group) - 1 - turn) * kWideTile;
  u.tile_end = u.tile0 + kWideTile < rows ? u.tile0 + kWideTile : rows;
  u.first = kh_span_of(p, s, (int)kh_div(u.tile0, p.by_group)).first & ~15;
  u.end = kh_span_of(p, s, (int)kh_div(u.tile_end - 1, p.by_group)).end;
  return u;
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
  const KhUnits units = kh_units_of(p, s);
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

template <class P>
__device__ __forceinline__ bool wide_parts(const P &p, int unit, int row0, KhSeq &s, Parts &parts) {
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
template <int D, class Done>
__device__ __forceinline__ void join(const KhAttentionParams &p, float *lds, Done &&done) {
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
      lds_barrier();
      if (live) {
        float top = m;
        for (int k = 0; k < here; ++k) top = fmaxf(top, lds[2 * (k * kRows + row)]);
        const float fade = exp2_hw(m - top);
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
              const float w = exp2_hw(lds[2 * (k * kRows + row)] - top);
              total += lds[2 * (k * kRows + row) + 1] * w;
              o += x[j] * w;
            }
          }
        }
      }
      lds_barrier();
    }
    // The shares' sums, in their order.
    if (shares > 1) {
      float *sum = lds + 5 * tid;
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = o[e];
      sum[4] = total;
      lds_barrier();
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
    done(s.start + i, hq, col, o, m, total);
  }
}

}  // namespace kh
