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
// Rows of V that no row of the tile sees (past the sequence's end, in pages
// that do not exist) are not read and count as zeros. Where some rows of the
// tile see an entry and others do not, 0 x V must be 0 also for infinities and
// NaN in V: see poison().
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

using kh::elem;
using kh::f32x4;
using kh::u32x2;
using kh::u32x4;

constexpr int kRows = 16;          // rows of a tile
constexpr int kKeys = 32;          // entries of a block
constexpr int kWaves = 4;          // waves of a workgroup; they take blocks in turn
constexpr float kNegBig = -1e30f;  // seed of the running maximum: finite, so that max - max is never NaN

// Elements of V that a lane loads in one piece, and how many pieces.
template <int D>
struct Cols {
  static constexpr int piece = kh::kWide ? 4 : D / 16 < 8 ? D / 16 : 8;
  static constexpr int span = 16 * piece;  // columns that 16 lanes cover
  static constexpr int count = D / span;
  static constexpr int words = piece * (int)sizeof(elem) / 4;
};

template <int D>
struct Tile {
  f32x4 o[Cols<D>::count][Cols<D>::piece];
  float m, l;  // of row l % 16; l of this lane's entries alone
};

// The eight rows of V of a lane, one piece of columns.
template <int D>
struct Piece {
  uint32_t w[8][Cols<D>::words];
};

// A operand for element e of the piece: entry j's element, j = 0..7 in order.
#if KH_ELEM != 0
template <int D>
__device__ __forceinline__ u32x4 across(const Piece<D> &v, int e) {
  u32x4 a;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    a[j] = __builtin_amdgcn_perm(v.w[2 * j + 1][e / 2], v.w[2 * j][e / 2], (e & 1) != 0 ? 0x07060302u : 0x05040100u);
  return a;
}
#endif

// o += (this piece's element e of V)^T P^T, p[j] for the lane's entry j.
template <int D>
__device__ __forceinline__ f32x4 pv(const Piece<D> &v, int e, const float (&p)[8], f32x4 o) {
#if KH_ELEM == 0
#pragma unroll
  for (int j = 0; j < 8; ++j) o = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v.w[j][e]), p[j], o, 0, 0, 0);
  return o;
#else
  u32x4 b;
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = kh::pack2(p[2 * j], p[2 * j + 1]);
  return kh::mma16(across<D>(v, e), b, o);
#endif
}

// Entries with infinities or NaN in V where rows differ in what they see: takes
// those elements out of v (as zeros) and adds to o what they give the rows
// that do see them. Products of 0/1 marks say which rows meet a NaN, +inf or
// -inf in which column; they are exact, and only blocks at a row's limit with
// such a value come here.
template <int D>
__device__ __forceinline__ void poison(Piece<D> &v, const float (&seen)[8], f32x4 (&o)[Cols<D>::piece]) {
  constexpr int kPerWord = 4 / (int)sizeof(elem);
#pragma nounroll
  for (int kind = 0; kind < 3; ++kind) {
    Piece<D> mark;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int w = 0; w < Cols<D>::words; ++w) {
        uint32_t r = 0;
#pragma unroll
        for (int b = 0; b < kPerWord; ++b) {
#if KH_ELEM == 0
          const uint32_t x = v.w[j][w], magnitude = x & 0x7fffffffu, inf = 0x7f800000u, sign = x >> 31, one = 0x3f800000u;
#else
          const uint32_t x = v.w[j][w] >> (16 * b) & 0xffffu, magnitude = x & 0x7fffu,
                         inf = KH_ELEM == 1 ? 0x7c00u : 0x7f80u, sign = x >> 15, one = KH_ELEM == 1 ? 0x3c00u : 0x3f80u;
#endif
          const bool hit = kind == 0 ? magnitude > inf : magnitude == inf && sign == (uint32_t)(kind - 1);
          r |= hit ? one << (16 * b) : 0u;
        }
        mark.w[j][w] = r;
      }
    const float add = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
    for (int e = 0; e < Cols<D>::piece; ++e) {
      const f32x4 met = pv<D>(mark, e, seen, f32x4{0, 0, 0, 0});
#pragma unroll
      for (int i = 0; i < 4; ++i) o[e][i] = met[i] > 0.0f ? o[e][i] + add : o[e][i];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int w = 0; w < Cols<D>::words; ++w) {
      uint32_t x = v.w[j][w];
#if KH_ELEM == 0
      x = kh::not_finite(x) ? 0u : x;
#else
      x = kh::not_finite(x & 0xffffu) ? x & 0xffff0000u : x;
      x = kh::not_finite(x & 0xffff0000u) ? x & 0xffffu : x;
#endif
      v.w[j][w] = x;
    }
}

// Natural log of a sum of exponentials held as its binary maximum and the
// sum relative to it.
__device__ __forceinline__ float lse_of(float top, float total) {
  return total == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * 0.69314718055994530942f;
}

template <int D>
__device__ __forceinline__ void attention(const KhAttentionParams &p, float *lds) {
  constexpr int kBytes = D * (int)sizeof(elem);
  constexpr int kSteps = kBytes / 64;
  using C = Cols<D>;
  const int lane = kh::lane_id(), wave = threadIdx.x / kh::kWave;
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);

  uint32_t id = blockIdx.x;
  const int head = (int)(id % (uint32_t)p.cache.kv_heads);
  id /= (uint32_t)p.cache.kv_heads;
  const int split = (int)(id % (uint32_t)p.splits), seq = (int)(id / (uint32_t)p.splits);
  const KhSeq s = kh_seq(p.table.lens[seq], p.q_starts[seq], p.q_starts[seq + 1], p.table.capacity, p.tokens);
  const KhSplit sp = kh_split(s, p.window, p.splits, p.split_keys, split);
  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const elem *kbase = static_cast<const elem *>(p.cache.k) + head * p.cache.k_head;
  const elem *vbase = static_cast<const elem *>(p.cache.v) + head * p.cache.v_head;
  const int rows = s.m * p.group;  // < 2^31: tokens x q_heads is
  const bool alone = sp.used == 1;
  // The join area: each wave's maxima and sums of its rows, what each row's
  // sum is multiplied by, and each wave's part of O.
  float *ml = lds, *inv = lds + kWaves * kRows * 2, *part = inv + kRows;
  constexpr int kPitch = D + 4;
  if (split >= sp.used) {
    // Nothing left for this workgroup: an empty part where the rows are joined.
    if (!alone) {
      for (int R = blockIdx.y * (int)blockDim.x + (int)threadIdx.x; R < rows; R += (int)(gridDim.y * blockDim.x)) {
        const int i = (int)kh_div(R, p.by_group);
        const int64_t row = (int64_t)(s.start + i) * p.q_heads + head * p.group + (R - i * p.group);
        float *to = p.part_ml + ((int64_t)split * p.tokens * p.q_heads + row) * 2;
        to[0] = kNegBig;
        to[1] = 0.0f;
      }
    }
    return;
  }

  for (int row0 = blockIdx.y * kRows; row0 < rows; row0 += gridDim.y * kRows) {
    const int R = row0 + r;
    const bool mine = R < rows;
    const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
    const int i_first = (int)kh_div(row0, p.by_group);
    const int i_last = (int)kh_div(row0 + kRows < rows ? row0 + kRows - 1 : rows - 1, p.by_group);
    const KhSpan seen = kh_seen(s, i, p.window);
    const KhSpan low = kh_seen(s, i_first, p.window), high = kh_seen(s, i_last, p.window);
    const int key_first = low.first > sp.first ? low.first : sp.first;
    const int key_end = high.end < sp.end ? high.end : sp.end;

    u32x4 q[kSteps];
    const elem *qp = static_cast<const elem *>(p.q) + (int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      q[c] = u32x4{0, 0, 0, 0};
      if (mine && 64 * c + 16 * h < row_bytes) q[c] = *reinterpret_cast<const u32x4 *>(qp + (64 * c + 16 * h) / (int)sizeof(elem));
    }

    Tile<D> t;
    t.m = kNegBig;
    t.l = 0.0f;
#pragma unroll
    for (int a = 0; a < C::count; ++a)
#pragma unroll
      for (int e = 0; e < C::piece; ++e) t.o[a][e] = f32x4{0, 0, 0, 0};

    for (int key0 = key_first + wave * kKeys; key0 < key_end; key0 += kWaves * kKeys) {
      // Rows of K: entries r and 16 + r of the block.
      KhSlot at[2];
      f32x4 x[2];
      bool there[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int key = key0 + 16 * b + r;
        at[b] = KhSlot{-1, 0};
        if (key < key_end) at[b] = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)key);
        there[b] = at[b].page >= 0;
        const elem *kp = kbase + at[b].page * p.cache.k_page + at[b].slot * p.cache.k_slot;
        x[b] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          u32x4 k = {0, 0, 0, 0};
          if (there[b] && 64 * c + 16 * h < row_bytes) k = *reinterpret_cast<const u32x4 *>(kp + (64 * c + 16 * h) / (int)sizeof(elem));
          x[b] = kh::mma16(k, q[c], x[b]);
        }
      }
      const uint32_t present = ((uint32_t)__builtin_amdgcn_ballot_w64(there[0]) & 0xffffu) |
                               ((uint32_t)__builtin_amdgcn_ballot_w64(there[1]) << 16);
      // Rows of V: the lane's eight entries, in the order of its scores.
      Piece<D> v[C::count];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = 16 * (j / 4) + 4 * h + j % 4;
        const int page = __shfl(at[j / 4].page, key & 15, kh::kWave), slot = __shfl(at[j / 4].slot, key & 15, kh::kWave);
        const elem *vp = vbase + page * p.cache.v_page + slot * p.cache.v_slot + C::piece * r;
#pragma unroll
        for (int a = 0; a < C::count; ++a) {
#pragma unroll
          for (int w = 0; w < C::words; ++w) v[a].w[j][w] = 0;
          if (page >= 0 && a * C::span + C::piece * r < d) {
            if constexpr (C::words == 4) {
              const u32x4 g = *reinterpret_cast<const u32x4 *>(vp + a * C::span);
              v[a].w[j][0] = g.x, v[a].w[j][1] = g.y, v[a].w[j][2] = g.z, v[a].w[j][3] = g.w;
            } else {
              const u32x2 g = *reinterpret_cast<const u32x2 *>(vp + a * C::span);
              v[a].w[j][0] = g.x, v[a].w[j][1] = g.y;
            }
          }
        }
      }

      float y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[j / 4][j % 4] * p.scale_log2;
      // Every row sees every entry of the block: no mask.
      const bool whole = present == 0xffffffffu && key0 + kKeys <= low.end && key0 >= high.first;
      float on[8];
      bool odd = false;
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = 16 * (j / 4) + 4 * h + j % 4, key = key0 + k;
          const bool sees = mine && key >= seen.first && key < seen.end && (present >> k & 1) != 0;
          on[j] = sees ? 1.0f : 0.0f;
          y[j] = sees ? y[j] : -__builtin_inff();
#pragma unroll
          for (int a = 0; a < C::count; ++a)
#pragma unroll
            for (int w = 0; w < C::words; ++w) odd |= kh::not_finite(v[a].w[j][w]);
        }
      }
      float top = t.m;
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, y[j]);
      top = fmaxf(top, __shfl_xor(top, 16, kh::kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kh::kWave));
      float fade = kh::exp2_hw(t.m - top);
      t.m = top;
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[j] = kh::exp2_hw(y[j] - top);
        sum += y[j];
      }
      t.l = t.l * fade + sum;
      if (__builtin_amdgcn_ballot_w64(odd) != 0) {
        // After the fading: an infinity does not survive a factor of zero.
#pragma unroll
        for (int a = 0; a < C::count; ++a) {
#pragma unroll
          for (int e = 0; e < C::piece; ++e) t.o[a][e] *= fade;
          poison<D>(v[a], on, t.o[a]);
        }
        fade = 1.0f;
      }
#pragma unroll
      for (int a = 0; a < C::count; ++a)
#pragma unroll
        for (int e = 0; e < C::piece; ++e) t.o[a][e] = pv<D>(v[a], e, y, t.o[a][e] * fade);
    }

    // Join the waves: rescale to the rows' common maximum, add in wave order.
    float l = t.l + __shfl_xor(t.l, 16, kh::kWave);
    l += __shfl_xor(l, 32, kh::kWave);
    if (h == 0) {
      ml[(wave * kRows + r) * 2] = t.m;
      ml[(wave * kRows + r) * 2 + 1] = l;
    }
    kh::lds_barrier();
    float top = kNegBig;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[(w * kRows + r) * 2]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += ml[(w * kRows + r) * 2 + 1] * kh::exp2_hw(ml[(w * kRows + r) * 2] - top);
    const float fade = kh::exp2_hw(t.m - top);
#pragma unroll
    for (int a = 0; a < C::count; ++a)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4)
#pragma unroll
        for (int e = 0; e < C::piece; ++e)
          part[(wave * kRows + r) * kPitch + a * C::span + C::piece * (4 * h + i4) + e] = t.o[a][e][i4] * fade;
    const int64_t row_of = (int64_t)(s.start + i) * p.q_heads + hq;  // this lane's row
    if (wave == 0 && h == 0) {
      inv[r] = alone ? (total == 0.0f ? 0.0f : 1.0f / total) : 1.0f;
      if (mine && alone) {
        if (p.lse != nullptr) p.lse[row_of] = lse_of(top, total);
        if (p.splits > 1) p.part_ml[row_of * 2 + 1] = -1.0f;  // finished here
      } else if (mine) {
        float *to = p.part_ml + ((int64_t)split * p.tokens * p.q_heads + row_of) * 2;
        to[0] = top;
        to[1] = total;
      }
    }
    kh::lds_barrier();
    for (int at = threadIdx.x; at < kRows * (D / 4); at += kWaves * kh::kWave) {
      const int row = at / (D / 4), col = at % (D / 4) * 4, RR = row0 + row;
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
        const int64_t at_row = (int64_t)split * p.tokens * p.q_heads + (int64_t)(s.start + ii) * p.q_heads + hh;
        *reinterpret_cast<f32x4 *>(p.part_o + at_row * d + col) = f32x4{y[0], y[1], y[2], y[3]};
      }
    }
    kh::lds_barrier();  // before the next tile writes the join area
  }
}

// Joins the parts of rows that several workgroups worked on, a wave per row.
__device__ __forceinline__ void join(const KhAttentionParams &p) {
  const int lane = kh::lane_id();
  const int64_t all = (int64_t)p.tokens * p.q_heads;
  const int64_t row = (int64_t)blockIdx.x * kWaves + threadIdx.x / kh::kWave;
  const int token = (int)(row / p.q_heads), hq = (int)(row - (int64_t)token * p.q_heads);
  // Tokens before the first and behind the last sequence have no parts.
  if (row >= all || token < p.q_starts[0] || token >= p.q_starts[p.table.seqs]) return;
  if (p.part_ml[row * 2 + 1] < 0.0f) return;  // finished by the one workgroup that had entries
  float top = kNegBig;
  for (int s0 = lane; s0 < p.splits; s0 += kh::kWave) top = fmaxf(top, p.part_ml[(s0 * all + row) * 2]);
  top = kh::wave_max(top);
  const int d = p.cache.head_dim;
  float o[4] = {}, total = 0.0f;
  for (int s0 = 0; s0 < p.splits; ++s0) {
    const float m = p.part_ml[(s0 * all + row) * 2], l = p.part_ml[(s0 * all + row) * 2 + 1];
    if (l == 0.0f) continue;
    const float w = kh::exp2_hw(m - top);
    total += l * w;
#pragma unroll
    for (int a = 0; a < 4; ++a)
      if (a * 64 + lane < d) o[a] += p.part_o[(s0 * all + row) * d + a * 64 + lane] * w;
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
  for (int a = 0; a < 4; ++a)
    if (a * 64 + lane < d)
      static_cast<elem *>(p.out)[(int64_t)token * p.out_stride + (int64_t)hq * d + a * 64 + lane] = static_cast<elem>(o[a] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[row] = lse_of(top, total);
}

}  // namespace

#define KH_ATTENTION(D)                                                                                     \
  extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_attention_##D)(const KhAttentionParams p) { \
    __shared__ float lds[kWaves * kRows * 2 + kRows + kWaves * kRows * (D + 4)];                             \
    attention<D>(p, lds);                                                                                    \
  }
KH_ATTENTION(64)
KH_ATTENTION(128)
KH_ATTENTION(256)
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_attention_join)(const KhAttentionParams p) { join(p); }
