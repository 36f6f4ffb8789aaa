// The attention that each entry of a paged cache received from a step's new
// tokens, added to what it had received before:
//   w[j] = (entry j is one of the new tokens ? 0 : w_in[j])
//        + sum over the kv head's query heads and the new tokens i that see j
//          of exp(scale q_i . k_j - lse_i)
// with lse_i from the attention of the same tokens. A row with lse = -inf saw
// nothing and adds nothing.
//
// As in paged_attention.hip the heads of a group are rows of one product, row R
// being token R / group, head R % group. Here S = Q K^T has entries in columns
// and rows in registers, so that the sum over rows stays in a lane until the
// end: every weight is written by one lane, its rows added in order, and a
// repeated call gives the same bits. What a key is seen by is a range of rows,
// [first, end): no row's token is worked out in the loops.
//
// Sequences of few rows: bound by reading K. A wave has all the rows' queries in
// registers and goes through blocks of 32 entries, the next block in flight: 32
// sequences of 1025 to 8192 entries (bf16, 32 heads on 8 of 128) 67 to 72 us, 4.4 to
// 4.7 TB/s.
// Sequences of many: a wave has 32 entries in registers and the workgroup brings
// tiles of 64 rows through LDS, one ahead. 32 x 32 scores of heads of 128 are eight
// product instructions of 32 cycles and 16 exponentials of 16 cycles for 64
// values: 256 cycles each, which a wave spends one after the other, with the masks
// and sums behind them.
#include "kh_cache.h"

namespace {

using namespace kh;

constexpr int kWaves = 4;
constexpr int kFewRows = 32;                  // a sequence of more is for wide()
constexpr int kWideKeys = 32 * kWaves;        // entries of a workgroup there

// Rows that see an entry: [first, end).
struct Seers {
  int first, end;
};

__device__ __forceinline__ Seers seers_of(const KhSeq &s, int key, int group, int window) {
  const int64_t own = (int64_t)key - (s.n - s.m);  // the token whose entry it is; below 0 an older one's
  const int64_t end = window > 0 && own + window < s.m ? own + window : s.m;
  Seers r;
  r.first = own > 0 ? (int)own * group : 0;
  r.end = end > 0 ? (int)end * group : 0;
  return r;
}

// Bit n: row R0 + n is one of them, n < 32.
__device__ __forceinline__ uint32_t rows_of(const Seers &s, int R0) {
  const int from = kh_clamp(s.first - R0, 0, 32), to = kh_clamp(s.end - R0, 0, 32);
  return from >= to ? 0u : (~0u >> (32 - to)) & (~0u << from);
}

// lse as it is subtracted from scores in powers of two; of a row that saw nothing
// (or is none) infinity. Such a row adds nothing whatever its scores are: those of
// infinities and NaN would not become 2^-inf, so it is masked like one that
// does not see the entry.
__device__ __forceinline__ float taken(float lse, bool real) {
  return real && lse != -__builtin_inff() ? lse * kLog2e : __builtin_inff();
}
__device__ __forceinline__ bool adds(float taken) { return taken != __builtin_inff(); }

struct Job {
  KhSeq s;
  int seq, head, rows;
  int64_t row;  // of weights
  const int32_t *table;
  const char *kbase;
};

// What was there before, from an address that is there in any case: read as
// bits, and kept by kept(). A choice between the loaded value and zero would
// become a branch round the load, with a wait for all loads in flight.
__device__ __forceinline__ uint32_t before(const KhWeightsParams &p, const Job &j, int key) {
  const float *in = p.weights_in != nullptr ? p.weights_in : p.weights;
  return __float_as_uint(in[j.row + (key < j.s.n ? key : j.s.n - 1)]);
}
__device__ __forceinline__ float kept(const KhWeightsParams &p, const Job &j, int key, uint32_t old) {
  return __uint_as_float(old & (p.weights_in != nullptr && key < j.s.n - j.s.m ? ~0u : 0u));
}

// The rows' queries and what their scores are taken from, for 1 to 32 rows.
template <int D>
struct Queries {
  u32x4 q[kFewRows / 16][Form<D>::steps];
  float lse[kFewRows / 16][4];
  uint32_t some;  // bit 16 t + e: the lane's row e of tile t is one that saw something
  bool two;       // more than 16 rows
};

template <int D>
__device__ __forceinline__ Queries<D> queries(const KhWeightsParams &p, const Job &j, int r, int h) {
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);
  Queries<D> y;
  y.two = j.rows > 16;
  y.some = 0;
#pragma unroll
  for (int t = 0; t < kFewRows / 16; ++t) {
    const KhQuery row = kh_query(j.s, p.group, p.by_group, 16 * t + r);
    const char *qp = static_cast<const char *>(p.q) +
                     ((int64_t)row.token * p.q_stride + (int64_t)(j.head * p.group + row.head) * d) * (int)sizeof(elem);
#pragma unroll
    for (int c = 0; c < Form<D>::steps; ++c) {
      const u32x4 x = *reinterpret_cast<const u32x4 *>(qp + within(64 * c + 16 * h, row_bytes));
      y.q[t][c] = 64 * c + 16 * h < row_bytes ? x : u32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int R = 16 * t + 4 * h + e;
      const KhQuery at = kh_query(j.s, p.group, p.by_group, R);
      y.lse[t][e] = taken(p.lse[(int64_t)at.token * p.q_heads + j.head * p.group + at.head], R < j.rows);
      y.some |= adds(y.lse[t][e]) ? 1u << (16 * t + e) : 0u;
    }
  }
  return y;
}

// What entry `key` of the lane's column receives, of scores x.
template <int D>
__device__ __forceinline__ float received(const KhWeightsParams &p, const Job &j, const Queries<D> &y, const f32x4 (&x)[kFewRows / 16],
                                          int key, bool there, int h) {
  const uint32_t sees = there ? rows_of(seers_of(j.s, key, p.group, p.window), 0) >> 4 * h & y.some : 0;
  float sum = 0.0f;
#pragma unroll
  for (int t = 0; t < kFewRows / 16; ++t)
    if (t == 0 || y.two) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float w = exp2_hw(fmaf(x[t][e], p.scale_log2, -y.lse[t][e]));
        sum += (sees >> (16 * t + e) & 1) != 0 ? w : 0.0f;
      }
    }
  return over_rows(sum, false);
}

// Few rows, pages of a multiple of 16 entries. K goes to LDS that the wave alone
// uses, whole rows to 16 lanes (as operands its loads would take 64 separate
// pieces of as many rows), and with it what the entries had received before; two
// blocks are in flight. Nothing in the loop is a load that the compiler sees:
// its wait for one would be a wait for all.
template <int D>
struct Ring {
  using F = Form<D>;
  static constexpr int pieces = Rows<D>::pieces, rows = Rows<D>::per_wave;  // that an instruction brings
  static constexpr int loads = F::keys / rows, old_at = F::keys * F::bytes, buffer = old_at + 256;
  static constexpr int lds = kWaves * 2 * buffer;
};

template <int D>
__device__ __forceinline__ uint32_t send(const KhWeightsParams &p, const Job &j, const Block<D, true> &b, const uint32_t (&lanes)[16 / Ring<D>::rows],
                                         u32x4 old, int key0, int end, const char *buffer, int lane) {
  using R = Ring<D>;
  const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>(buffer);
#pragma unroll
  for (int t = 0; t < Form<D>::tiles; ++t) {
    const uint64_t at = (uint64_t)reinterpret_cast<uintptr_t>(j.kbase) + kh_row(b.at[t], p.cache.k_page, p.cache.k_slot);
    const uint32_t real = (uint32_t)__builtin_popcount(b.present >> (16 * t) & 0xffffu);
    const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32), real * p.cache.k_slot, 0x00020000u};
#pragma unroll
    for (int i = 0; i < 16 / R::rows; ++i) dma16(rsrc, lanes[i], lds + (uint32_t)((16 * t + i * R::rows) * Form<D>::bytes));
  }
  // Entries key0 .. of the row of weights: the resource starts at `first`.
  dma4(old, key0 + lane < end && lane < Form<D>::keys ? (uint32_t)(key0 + lane) * 4u : kOutside, lds + (uint32_t)R::old_at);
  return b.present;
}

template <int D>
__device__ __forceinline__ void few_even(const KhWeightsParams &p, const Job &j, int first, int end, char *lds) {
  using F = Form<D>;
  using G = Ring<D>;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, h = lane >> 4;
  const int row_bytes = p.cache.head_dim * (int)sizeof(elem);
  constexpr int kStep = kWaves * F::keys;
  int key0 = first + wave * F::keys;
  if (key0 >= end) return;
  char *ring = lds + wave * 2 * G::buffer;
  uint32_t lanes[16 / G::rows];
#pragma unroll
  for (int i = 0; i < 16 / G::rows; ++i) {
    const int row = i * G::rows + lane / G::pieces, c = 16 * (lane % G::pieces ^ k_turn<D>(row));
    lanes[i] = c < row_bytes ? (uint32_t)row * p.cache.k_slot + (uint32_t)c : kOutside;
  }
  // The weights of the chunk's older entries; of the new tokens' own, and without weights_in, zeros.
  const uint64_t in = (uint64_t)reinterpret_cast<uintptr_t>(p.weights_in + j.row + first);
  const uint32_t older = p.weights_in == nullptr ? 0u : (uint32_t)kh_older(j.s, first, end);
  const u32x4 old = {(uint32_t)in, (uint32_t)(in >> 32), older * 4u, 0x00020000u};
  Block<D, true> b;
  uint32_t now, next;
  find<D, true>(b, p, j.table, key0, end, r);
  const Queries<D> y = queries<D>(p, j, r, h);
  settle<D, true>(b, p, key0, end, r);
  now = send<D>(p, j, b, lanes, old, key0 - first, end - first, ring, lane);
  find<D, true>(b, p, j.table, key0 + kStep, end, r);
  settle<D, true>(b, p, key0 + kStep, end, r);
  next = send<D>(p, j, b, lanes, old, key0 + kStep - first, end - first, ring + G::buffer, lane);
  find<D, true>(b, p, j.table, key0 + 2 * kStep, end, r);
  for (int cur = 0; key0 < end; key0 += kStep, cur ^= 1) {
    char *buffer = ring + cur * G::buffer;
    const uint32_t present = now;
    arrived<G::loads + 1>();  // all but the next block
    f32x4 x[F::tiles][kFewRows / 16];
    u32x4 k[F::tiles][F::steps];
    float before[F::tiles];
#pragma unroll
    for (int t = 0; t < F::tiles; ++t) {
      before[t] = *reinterpret_cast<const float *>(buffer + G::old_at + 4 * (16 * t + r));
#pragma unroll
      for (int c = 0; c < F::steps; ++c)
        k[t][c] = *reinterpret_cast<const u32x4 *>(buffer + (16 * t + r) * F::bytes + 16 * ((4 * c | h) ^ k_turn<D>(r)));
    }
#pragma unroll
    for (int t = 0; t < F::tiles; ++t)
#pragma unroll
      for (int n = 0; n < kFewRows / 16; ++n)
        if (n == 0 || y.two) {
          x[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < F::steps; ++c) x[t][n] = mma16(y.q[n][c], k[t][c], x[t][n]);
        }
    // The block has been read: the one after the next takes its place.
    now = next;
    settle<D, true>(b, p, key0 + 2 * kStep, end, r);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    next = send<D>(p, j, b, lanes, old, key0 + 2 * kStep - first, end - first, buffer, lane);
    find<D, true>(b, p, j.table, key0 + 3 * kStep, end, r);
#pragma unroll
    for (int t = 0; t < F::tiles; ++t) {
      const int key = key0 + 16 * t + r;
      const float sum = received<D>(p, j, y, x[t], key, (present >> (16 * t + r) & 1) != 0, h);
      if (h == t && key < end) p.weights[j.row + key] = before[t] + sum;
    }
  }
  vm_wait<0>();  // nothing is on its way to LDS that the workgroup may give back
}

// Few rows, other pages: K in registers, a block ahead.
template <int D>
__device__ __forceinline__ void few(const KhWeightsParams &p, const Job &j, int first, int end) {
  using F = Form<D>;
  const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);
  constexpr int kStep = kWaves * F::keys;
  int key0 = first + wave * F::keys;
  if (key0 >= end) return;
  u32x4 k[F::tiles][F::steps];
  Block<D, false> now, next;
  find<D, false>(now, p, j.table, key0, end, r);
  find<D, false>(next, p, j.table, key0 + kStep, end, r);
  const Queries<D> y = queries<D>(p, j, r, h);
  settle<D, false>(now, p, key0, end, r);
  __builtin_amdgcn_sched_barrier(0);
  load_k<D, false>(k, now, p, j.kbase, row_bytes, r, h);
  __builtin_amdgcn_sched_barrier(0);
  for (; key0 < end; key0 += kStep) {
    const uint32_t present = now.present;
    uint32_t old[F::tiles];
#pragma unroll
    for (int b = 0; b < F::tiles; ++b) old[b] = before(p, j, key0 + 16 * b + r);
    if (d != D) {
#pragma unroll
      for (int c = 0; c < F::steps; ++c)
        if (64 * c + 16 * h >= row_bytes) {
#pragma unroll
          for (int b = 0; b < F::tiles; ++b) k[b][c] = u32x4{0, 0, 0, 0};
        }
    }
    f32x4 x[F::tiles][kFewRows / 16];
#pragma unroll
    for (int b = 0; b < F::tiles; ++b)
#pragma unroll
      for (int t = 0; t < kFewRows / 16; ++t)
        if (t == 0 || y.two) {
          x[b][t] = f32x4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < F::steps; ++c) x[b][t] = mma16(y.q[t][c], k[b][c], x[b][t]);
        }
    now = next;
    settle<D, false>(now, p, key0 + kStep, end, r);
    load_k<D, false>(k, now, p, j.kbase, row_bytes, r, h);
    find<D, false>(next, p, j.table, key0 + 2 * kStep, end, r);
#pragma unroll
    for (int b = 0; b < F::tiles; ++b) {
      const int key = key0 + 16 * b + r;
      const float sum = received<D>(p, j, y, x[b], key, (present >> (16 * b + r) & 1) != 0, h);
      if (h == b && key < end) p.weights[j.row + key] = kept(p, j, key, old[b]) + sum;
    }
  }
}

// Where a lane's pieces of a tile of rows of q lie, past the tile's first token.
// `steady` (the tile holds whole tokens, and no two share bytes): the same for
// every tile, and the resource's end keeps out rows past the last; otherwise
// they are kept out here.
template <int D>
__device__ __forceinline__ void pieces_of(const KhWeightsParams &p, const Job &j, int R0, uint32_t (&off)[Rows<D>::passes], int lane, int wave) {
  using W = Rows<D>;
  const int row_bytes = p.cache.head_dim * (int)sizeof(elem), i0 = (int)kh_div(R0, p.by_group);
#pragma unroll
  for (int i = 0; i < W::passes; ++i) {
    const int row = wave * W::share + i * W::per_wave + lane / W::pieces, R = R0 + row;
    const int t = (int)kh_div(R, p.by_group), c = 16 * (lane % W::pieces ^ k_turn<D>(row));
    off[i] = (uint32_t)(t - i0) * (uint32_t)(p.q_stride * (int)sizeof(elem)) + (uint32_t)((R - t * p.group) * row_bytes + c);
    if (c >= row_bytes || (!p.steady && R >= j.rows)) off[i] = kOutside;
  }
}

// Sends a tile of rows of q to LDS.
template <int D>
__device__ __forceinline__ void send(const KhWeightsParams &p, const Job &j, int R0, const uint32_t (&off)[Rows<D>::passes],
                                     const char *buffer, int wave) {
  using W = Rows<D>;
  const int i0 = (int)kh_div(R0, p.by_group), left = j.s.m > i0 ? j.s.m - i0 : 0;
  const uint64_t at = (uint64_t)reinterpret_cast<uintptr_t>(p.q) +
                      (uint64_t)((int64_t)(j.s.start + i0) * p.q_stride + (int64_t)j.head * p.group * p.cache.head_dim) * sizeof(elem);
  const uint64_t bytes = (uint64_t)left * (uint64_t)p.q_stride * sizeof(elem);
  const u32x4 rsrc = {(uint32_t)at, (uint32_t)(at >> 32), p.steady && bytes < kOutside ? (uint32_t)bytes : kOutside, 0x00020000u};
#pragma unroll
  for (int i = 0; i < W::passes; ++i)
    dma16(rsrc, off[i], (uint32_t)reinterpret_cast<uintptr_t>(buffer) + (uint32_t)((wave * W::share + i * W::per_wave) * W::bytes));
}

// Two tiles of rows, what is taken of each row's scores, and which rows add something.
template <int D>
constexpr int kWideLdsOf = 2 * (Rows<D>::tile * (Rows<D>::bytes + 4) + 8);

template <int D>
__device__ __forceinline__ void wide(const KhWeightsParams &p, const Job &j, int key0, char *lds) {
  using W = Rows<D>;
  constexpr int kSteps = W::bytes / 32, kBuffer = W::tile * W::bytes;
  float *stats = reinterpret_cast<float *>(lds + 2 * kBuffer);  // [2][tile]
  uint32_t *some = reinterpret_cast<uint32_t *>(stats + 2 * W::tile);  // [2][2], bit n: row n of 32 adds something
  const int tid = threadIdx.x, lane = lane_id(), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 31, h = lane >> 5;
  const int row_bytes = p.cache.head_dim * (int)sizeof(elem);
  const int mine0 = key0 + 32 * wave, key = mine0 + r, last = mine0 + 31 < j.s.n ? mine0 + 31 : j.s.n - 1;
  const Seers own = seers_of(j.s, key, p.group, p.window);
  // Rows that see all of the wave's entries, and any of them; any of the workgroup's.
  const Seers wave_first = seers_of(j.s, mine0, p.group, p.window), wave_last = seers_of(j.s, last, p.group, p.window);
  const int group_last = key0 + kWideKeys <= j.s.n ? key0 + kWideKeys - 1 : j.s.n - 1;
  const int R_begin = seers_of(j.s, key0, p.group, p.window).first / W::tile * W::tile;
  const int R_end = seers_of(j.s, group_last, p.group, p.window).end;

  const uint32_t old = before(p, j, key);
  KhSlot at = look_up<false>(p, j.table, key, j.s.n);
  const bool there = key < j.s.n && (uint32_t)at.page < (uint32_t)p.cache.pages;
  if (!there) at = KhSlot{0, 0};
  u32x4 k[kSteps];
  const char *kp = j.kbase + kh_row(at, p.cache.k_page, p.cache.k_slot);
#pragma unroll
  for (int c = 0; c < kSteps; ++c) {
    const u32x4 x = *reinterpret_cast<const u32x4 *>(kp + within(32 * c + 16 * h, row_bytes));
    k[c] = there && 32 * c + 16 * h < row_bytes ? x : u32x4{0, 0, 0, 0};
  }
  float sum = 0.0f;
  if (R_begin < R_end) {
    // The tile's lse: a thread's row, a tile ahead as the rows are.
    auto lse_at = [&](int R0) {
      if (wave >= (W::tile + kWave - 1) / kWave) return 0.0f;
      const int R = R0 + tid % W::tile, real = R < j.rows ? R : 0, i = (int)kh_div(real, p.by_group);
      return p.lse[(int64_t)(j.s.start + i) * p.q_heads + j.head * p.group + real - i * p.group];
    };
    float ahead = lse_at(R_begin);
    uint32_t off[W::passes];
    pieces_of<D>(p, j, R_begin, off, lane, wave);
    send<D>(p, j, R_begin, off, lds, wave);
    int cur = 0;
    for (int R0 = R_begin; R0 < R_end; R0 += W::tile, cur ^= 1) {
      const char *buffer = lds + cur * kBuffer;
      float *lse = stats + cur * W::tile;
      vm_wait<0>();
      if (wave == 0) {  // a tile has no more rows than a wave lanes
        const float y = taken(ahead, R0 + tid < j.rows);
        const uint64_t all = __builtin_amdgcn_ballot_w64(adds(y));
        if (tid < W::tile) lse[tid] = y;
        if (tid < 2) some[2 * cur + tid] = (uint32_t)(all >> 32 * tid);
      }
      lds_barrier();
      uint32_t added[2];
#pragma unroll
      for (int t = 0; t < W::tile / 32; ++t) added[t] = __builtin_amdgcn_readfirstlane(some[2 * cur + t]);
      ahead = lse_at(R0 + W::tile);
      if (!p.steady) pieces_of<D>(p, j, R0 + W::tile, off, lane, wave);
      send<D>(p, j, R0 + W::tile, off, lds + (cur ^ 1) * kBuffer, wave);
#pragma unroll
      for (int t = 0; t < W::tile / 32; ++t) {
        const int R1 = R0 + 32 * t;
        if (mine0 >= j.s.n || R1 >= wave_last.end || R1 + 32 <= wave_first.first) continue;
        f32x16 x = {};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) x = mma32(k_rows<D>(buffer, t, c, lane), k[c], x);
        const bool whole = R1 >= wave_last.first && R1 + 32 <= wave_first.end && added[t] == ~0u;
        const uint32_t sees = whole ? ~0u : (rows_of(own, R1) & added[t]) >> 4 * h;
        float part = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 y = *reinterpret_cast<const f32x4 *>(lse + 32 * t + 8 * g + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * g + e] = exp2_hw(fmaf(x[4 * g + e], p.scale_log2, -y[e]));
        }
        if (!whole) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = (sees >> (8 * (i / 4) + i % 4) & 1) != 0 ? x[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) part += x[i];
        sum += part;
      }
    }
  }
  vm_wait<0>();  // nothing is on its way to LDS that the workgroup may give back
  sum = over_halves(sum, false);
  if (h == 0 && key < j.s.n) p.weights[j.row + key] = kept(p, j, key, old) + (there ? sum : 0.0f);
}

// No new tokens: what was there before, or zeros. Neither q nor lse is read.
__device__ __forceinline__ void copy(const KhWeightsParams &p, const Job &j, int first, int end) {
  for (int key = first + (int)threadIdx.x; key < end; key += kWaves * kWave)
    p.weights[j.row + key] = p.weights_in != nullptr ? p.weights_in[j.row + key] : 0.0f;
}

// RING: there is LDS for few_even().
template <int D, bool RING>
__device__ __forceinline__ void weights(const KhWeightsParams &p, char *lds) {
  Job j;
  const int pairs = p.table.seqs * p.cache.kv_heads, chunk = (int)blockIdx.x / pairs, pair = (int)blockIdx.x - chunk * pairs;
  j.seq = pair / p.cache.kv_heads, j.head = pair - j.seq * p.cache.kv_heads;
  j.s = kh_seq(p.table.lens[j.seq], p.q_starts[j.seq], p.q_starts[j.seq + 1], p.table.capacity, p.tokens);
  j.rows = j.s.m * p.group;
  j.row = j.seq * p.seq_stride + j.head * p.head_stride;
  j.table = p.table.pages + j.seq * p.table.row_stride;
  j.kbase = p.cache.k + (uint64_t)j.head * p.cache.k_head;
  // Chunks past those that the launch was sized for fall to its workgroups in turn.
  for (int64_t first = (int64_t)chunk * p.chunk_keys; first < j.s.n; first += (int64_t)p.chunks * p.chunk_keys) {
    const int end = first + p.chunk_keys < j.s.n ? (int)first + p.chunk_keys : j.s.n;
    if (j.rows == 0) {
      copy(p, j, (int)first, end);
    } else if (j.rows <= kFewRows) {
      if constexpr (RING)
        few_even<D>(p, j, (int)first, end, lds);
      else
        few<D>(p, j, (int)first, end);
    } else {
      for (int key0 = (int)first; key0 < end; key0 += kWideKeys) {
        wide<D>(p, j, key0, lds);
        lds_barrier();  // before the next takes the same LDS
      }
    }
  }
}

}  // namespace

// Steps of single tokens, and of few: with the ring, two workgroups to a CU.
#define KH_WEIGHTS(D)                                                                                      \
  extern "C" __global__ void __launch_bounds__(256, D > 128 ? 1 : 2) KH_TYPED(paged_weights_##D)(const KhWeightsParams p) { \
    constexpr int kWideLds = kWideLdsOf<D>;                                                                 \
    __shared__ __attribute__((aligned(16))) char lds[kWideLds > Ring<D>::lds ? kWideLds : Ring<D>::lds];    \
    if (p.even)                                                                                             \
      weights<D, true>(p, lds);                                                                             \
    else                                                                                                    \
      weights<D, false>(p, lds);                                                                            \
  }
KH_WEIGHTS(64)
KH_WEIGHTS(128)
KH_WEIGHTS(256)
// Steps with chunks: without it, three. Two sequences of up to 1024 new tokens
// and 6000 entries (bf16, 32 heads on 8 of 128): 116 to 120 us, 645 to 665 TFLOP/s.
// With the ring's LDS, two workgroups to a CU, such a step took half as long again.
// In 32 bits heads of 128 take 66 KB: two.
#define KH_WEIGHTS_WIDE(D)                                                                                 \
  extern "C" __global__ void __launch_bounds__(256, D > 128 ? 1 : kWide && D > 64 ? 2 : 3) KH_TYPED(paged_weights_wide_##D)(const KhWeightsParams p) { \
    __shared__ __attribute__((aligned(16))) char lds[kWideLdsOf<D>];                                        \
    weights<D, false>(p, lds);                                                                              \
  }
KH_WEIGHTS_WIDE(64)
KH_WEIGHTS_WIDE(128)
KH_WEIGHTS_WIDE(256)
