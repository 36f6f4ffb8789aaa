// The attention that each entry of a paged cache received from a step's new
// tokens, added to what it had received before:
//   w[j] = (entry j is one of the new tokens ? 0 : w_in[j])
//        + sum over the kv head's query heads and the new tokens i that see j
//          of exp(scale q_i . k_j - lse_i)
// with lse_i from the attention of the same tokens. A row with lse = -inf saw
// nothing and adds nothing.
//
// Per wave: 32 entries, held as the B operand of S = Q K^T for the whole
// kernel, against all rows (tokens x heads of the group) 16 at a time. The
// result's lane l holds entry l % 16 and rows 4 (l / 16) + i: the sum over rows
// is the lane's own until the end. Each weight is written by one lane and its
// rows are added in order, so a repeated call gives the same bits.
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

using kh::elem;
using kh::f32x4;
using kh::u32x4;

constexpr int kKeys = 32;  // entries of a wave
constexpr int kWaves = 4;

template <int D>
__device__ __forceinline__ void weights(const KhWeightsParams &p) {
  constexpr int kSteps = D * (int)sizeof(elem) / 64;
  const int lane = kh::lane_id(), wave = threadIdx.x / kh::kWave;
  const int r = lane & 15, h = lane >> 4;
  const int d = p.cache.head_dim, row_bytes = d * (int)sizeof(elem);
  const int head = (int)(blockIdx.x % (uint32_t)p.cache.kv_heads), seq = (int)(blockIdx.x / (uint32_t)p.cache.kv_heads);
  const KhSeq s = kh_seq(p.table.lens[seq], p.q_starts[seq], p.q_starts[seq + 1], p.table.capacity, p.tokens);
  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const char *kbase = p.cache.k + (uint64_t)head * p.cache.k_head;
  const int64_t row = seq * p.seq_stride + head * p.head_stride;
  const int rows = s.m * p.group;

  for (int64_t key0 = ((int64_t)blockIdx.y * kWaves + wave) * kKeys; key0 < s.n; key0 += (int64_t)gridDim.y * kWaves * kKeys) {
    u32x4 k[2][kSteps];
    bool there[2];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int key = (int)key0 + 16 * b + r;
      KhSlot at{-1, 0};
      if (key < s.n) at = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)key);
      there[b] = at.page >= 0;
      const char *kp = kbase + kh_row(at, p.cache.k_page, p.cache.k_slot);
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        k[b][c] = u32x4{0, 0, 0, 0};
        if (there[b] && 64 * c + 16 * h < row_bytes)
          k[b][c] = *reinterpret_cast<const u32x4 *>(kp + 64 * c + 16 * h);
      }
    }
    // The first token that sees any of these entries is the one whose own
    // entry is the first of them.
    const int i0 = (int)key0 - (s.n - s.m);
    const int from = i0 > 0 ? i0 * p.group / 16 * 16 : 0;
    for (int row0 = from; row0 < rows; row0 += 16) {
      const int R = row0 + r;
      const bool mine = R < rows;
      const int i = mine ? (int)kh_div(R, p.by_group) : 0, hq = head * p.group + (mine ? R - i * p.group : 0);
      // With a window: past the last token that sees any of the entries.
      if (p.window > 0 && kh_seen(s, (int)kh_div(row0, p.by_group), p.window).first >= key0 + kKeys) break;
      const elem *qp = static_cast<const elem *>(p.q) + (int64_t)(s.start + i) * p.q_stride + (int64_t)hq * d;
      f32x4 x[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        u32x4 q = {0, 0, 0, 0};
        if (mine && 64 * c + 16 * h < row_bytes) q = *reinterpret_cast<const u32x4 *>(qp + (64 * c + 16 * h) / (int)sizeof(elem));
#pragma unroll
        for (int b = 0; b < 2; ++b) x[b] = kh::mma16(q, k[b][c], x[b]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int RR = row0 + 4 * h + j;
        const bool real = RR < rows;
        const int ii = real ? (int)kh_div(RR, p.by_group) : 0;
        const float lse = real ? p.lse[(int64_t)(s.start + ii) * p.q_heads + head * p.group + RR - ii * p.group] : 0.0f;
        const KhSpan seen = kh_seen(s, ii, p.window);
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int key = (int)key0 + 16 * b + r;
          const bool sees = real && there[b] && key >= seen.first && key < seen.end && lse != -__builtin_inff();
          const float w = kh::exp2_hw(x[b][j] * p.scale_log2 - lse * kh::kLog2e);
          sum[b] += sees ? w : 0.0f;
        }
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      sum[b] += __shfl_xor(sum[b], 16, kh::kWave);
      sum[b] += __shfl_xor(sum[b], 32, kh::kWave);
      const int key = (int)key0 + 16 * b + r;
      if (h == b && key < s.n) {
        const float before = p.weights_in != nullptr && key < s.n - s.m ? p.weights_in[row + key] : 0.0f;
        p.weights[row + key] = before + sum[b];
      }
    }
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_weights_64)(const KhWeightsParams p) { weights<64>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_weights_128)(const KhWeightsParams p) { weights<128>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(paged_weights_256)(const KhWeightsParams p) { weights<256>(p); }
