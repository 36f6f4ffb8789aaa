// Norms of queries and keys for each head, with the position rotation and
// the write of the new keys and values to a paged cache in the same pass.
//
// For token t and head h, a row x of head_dim elements:
//   y = x / sqrt(mean(x^2) + eps) gamma         (norm != 0; y = x otherwise)
//   (a, b) -> (a cos w - b sin w, b cos w + a sin w),  w = positions[t] inv_freq[i]
// over the pairs (a, b) = (y[i], y[i + r/2]), or (y[2i], y[2i + 1]) where
// interleaved, i < r/2, r = rotary_dim; elements past r are not rotated.
// Rows of v are copied.
//
// Bound by memory: a row is read once and written once. A row takes L lanes,
// a power of two with L x 8 >= head_dim, each with two groups of four
// elements: the two ends of four pairs, so that no rotation crosses lanes
// (half-split pairs lie r/2 apart, interleaved ones next to each other). A
// wave runs through the heads of one token, 64 / L at a time, and computes the
// lane's four angles once for all of them.
//
// The angle is formed in 64 bits: at position 2e6 a 32-bit product is off by
// up to 0.06 rad. Its part past whole quarter turns, below pi/4, goes through
// the Taylor series of sine and cosine in 32 bits (first terms left out
// 2e-9 and 2e-10).
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

__device__ __forceinline__ void turn(double angle, float &c, float &s) {
  const double quarters = angle * 0.63661977236758134308;  // 2 / pi
  const double whole = __builtin_rint(quarters);
  const float x = static_cast<float>((quarters - whole) * 1.57079632679489661923);
  const int q = static_cast<int>(static_cast<int64_t>(whole)) & 3;
  const float z = x * x;
  const float si = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float co = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const float a = (q & 1) != 0 ? si : co, b = (q & 1) != 0 ? co : si;
  c = q == 1 || q == 2 ? -a : a;
  s = q >= 2 ? -b : b;
}

// Sum over the L lanes of a row.
template <int L>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int i = L / 2; i > 0; i /= 2) v += __shfl_xor(v, i, kh::kWave);
  return v;
}

template <int L>
__device__ __forceinline__ void rope(const KhRopeParams &p) {
  using kh::elem;
  const int lane = kh::lane_id();
  // A job is one part of one token's heads; a wave takes one.
  const int64_t job = (int64_t)blockIdx.x * (256 / kh::kWave) + threadIdx.x / kh::kWave;
  const int64_t t = job / p.parts;
  const int part = (int)(job - t * p.parts);
  if (t >= p.tokens) return;
  const int u = lane % L, d = p.head_dim, r = p.rotary;
  const bool live = u * 8 < d;
  const bool turned = u * 8 < r;
  const int a0 = turned && !p.interleaved ? 4 * u : 8 * u, a1 = turned && !p.interleaved ? r / 2 + 4 * u : 8 * u + 4;

  const int64_t slot = p.k_cache != nullptr ? p.slots[t] : -1;
  const bool cached = slot >= 0 && slot < p.rows;
  const int64_t page = cached ? slot / p.page_size : 0, in_page = cached ? slot - page * p.page_size : 0;

  float c[4], s[4], gq[2][4], gk[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = 1.0f, s[i] = 0.0f;
  if (turned) {
    const double pos = static_cast<double>(p.positions[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) turn(pos * static_cast<double>(p.inv_freq[4 * u + i]), c[i], s[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) gq[0][i] = gq[1][i] = gk[0][i] = gk[1][i] = 1.0f;
  if (live && p.norm && p.q_gamma != nullptr) {
    kh::load4(gq[0], static_cast<const elem *>(p.q_gamma) + a0);
    kh::load4(gq[1], static_cast<const elem *>(p.q_gamma) + a1);
  }
  if (live && p.norm && p.k_gamma != nullptr) {
    kh::load4(gk[0], static_cast<const elem *>(p.k_gamma) + a0);
    kh::load4(gk[1], static_cast<const elem *>(p.k_gamma) + a1);
  }

  const int heads = p.q_heads + p.kv_heads + (cached ? p.kv_heads : 0);
  constexpr int kRows = kh::kWave / L;
  for (int h0 = part * kRows; h0 < heads; h0 += p.parts * kRows) {
    // Every lane takes part in its row's sum, those without elements too.
    const int h = h0 + lane / L;
    const bool on = live && h < heads;
    const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
    const int hk = is_q ? h : is_v ? h - p.q_heads - p.kv_heads : h - p.q_heads;
    const elem *src = is_q   ? static_cast<const elem *>(p.q) + t * p.q_stride
                      : is_v ? static_cast<const elem *>(p.v) + t * p.v_stride
                             : static_cast<const elem *>(p.k) + t * p.k_stride;
    src += (int64_t)hk * d;
    float x[2][4] = {};
    if (on) {
      kh::load4(x[0], src + a0);
      kh::load4(x[1], src + a1);
    }
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sq += x[0][i] * x[0][i] + x[1][i] * x[1][i];
    sq = row_sum<L>(sq);
    if (!is_v) {
      const float scale = p.norm ? 1.0f / __builtin_sqrtf(sq / (float)d + p.eps) : 1.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[0][i] *= scale * (is_q ? gq[0][i] : gk[0][i]);
        x[1][i] *= scale * (is_q ? gq[1][i] : gk[1][i]);
      }
      if (turned && !p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = x[0][i], b = x[1][i];
          x[0][i] = a * c[i] - b * s[i];
          x[1][i] = b * c[i] + a * s[i];
        }
      } else if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float &a = x[i / 2][2 * (i % 2)], &b = x[i / 2][2 * (i % 2) + 1];
          const float y = a * c[i] - b * s[i];
          b = b * c[i] + a * s[i];
          a = y;
        }
      }
    }
    if (on && (is_q || (!is_v && p.k_out != nullptr))) {
      elem *dst = is_q ? static_cast<elem *>(p.q_out) + t * p.q_out_stride : static_cast<elem *>(p.k_out) + t * p.k_out_stride;
      dst += (int64_t)hk * d;
      kh::store4(dst + a0, x[0]);
      kh::store4(dst + a1, x[1]);
    }
    if (on && !is_q && cached) {
      elem *dst = is_v ? static_cast<elem *>(p.v_cache) + page * p.v_page + in_page * p.v_slot + hk * p.v_head
                       : static_cast<elem *>(p.k_cache) + page * p.k_page + in_page * p.k_slot + hk * p.k_head;
      kh::store4(dst + a0, x[0]);
      kh::store4(dst + a1, x[1]);
    }
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_8)(const KhRopeParams p) { rope<8>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_16)(const KhRopeParams p) { rope<16>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_32)(const KhRopeParams p) { rope<32>(p); }
