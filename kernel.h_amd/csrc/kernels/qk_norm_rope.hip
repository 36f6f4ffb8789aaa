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
// wave runs through the heads of one token, 64 / L at a time, the next ones'
// rows on their way, and computes the lane's four angles once for all of them,
// while the first rows come. 8192 tokens of 32 + 8 + 8 heads of 128, bf16: 42 us,
// 4.8 TB/s; with outputs that stay in the caches 47.
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

template <int CONTROL>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CONTROL, 0xf, 0xf, false));
}

// Sum over the L lanes of a row.
template <int L>
__device__ __forceinline__ float row_sum(float v) {
  v += moved<0xb1>(v);   // lane ^ 1
  v += moved<0x4e>(v);   // lane ^ 2
  v += moved<0x141>(v);  // 7 - lane of each eight: the other four, which all hold the same
  if constexpr (L >= 16) v += moved<0x140>(v);  // 15 - lane of each sixteen: the other eight
  if constexpr (L >= 32) v += __shfl_xor(v, 16, kh::kWave);
  return v;
}

// 1 / sqrt(x), x >= 0, to a unit in the last place: v_rsq_f32, which takes no
// denormal numbers (and gives what the formula gives for 0, infinities, NaN).
__device__ __forceinline__ float inverse_root(float x) {
  const bool tiny = x < 0x1p-100f;
  const float y = __builtin_amdgcn_rsqf(tiny ? x * 0x1p64f : x);
  return tiny ? y * 0x1p32f : y;
}

#if KH_ELEM == 0
typedef kh::f32x4 Four;  // elements as they lie in memory
#else
typedef kh::u32x2 Four;
#endif

__device__ __forceinline__ void unpack(float (&x)[4], Four v) {
#if KH_ELEM == 0
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
#else
  x[0] = kh::low_of(v.x), x[1] = kh::high_of(v.x), x[2] = kh::low_of(v.y), x[3] = kh::high_of(v.y);
#endif
}

// Past the caches: what a long chunk writes is more than they hold, and what a
// step of single tokens writes is little for its readers to fetch.
__device__ __forceinline__ void store_past(kh::elem *p, const float (&x)[4]) {
#if KH_ELEM == 0
  __builtin_nontemporal_store(kh::f32x4{x[0], x[1], x[2], x[3]}, reinterpret_cast<kh::f32x4 *>(p));
#else
  __builtin_nontemporal_store(kh::u32x2{kh::pack2(x[0], x[1]), kh::pack2(x[2], x[3])}, reinterpret_cast<kh::u32x2 *>(p));
#endif
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

  // Steps: those of q's heads, then k's, then v's, kRows heads each.
  constexpr int kRows = kh::kWave / L;
  const int of_q = (p.q_heads + kRows - 1) / kRows, of_k = (p.kv_heads + kRows - 1) / kRows;
  // A lane without elements or without a head reads some other's.
  const int l0 = live ? a0 : 0, l1 = live ? a1 : 4;
  const int q_heads = p.q_heads, kv_heads = p.kv_heads, parts = p.parts;
  const elem *const of_t[3] = {static_cast<const elem *>(p.q) + t * p.q_stride, static_cast<const elem *>(p.k) + t * p.k_stride,
                               static_cast<const elem *>(p.v) + t * p.v_stride};
  Four ahead[2];
  auto load = [&](int step) {
    const bool is_q = step < of_q, is_v = step >= of_q + of_k;
    const elem *src = is_q ? of_t[0] : is_v ? of_t[2] : of_t[1];
    const int n = is_q ? q_heads : kv_heads, h = (step - (is_q ? 0 : is_v ? of_q + of_k : of_q)) * kRows + lane / L;
    src += (int64_t)(h < n ? h : n - 1) * d;
    ahead[0] = *reinterpret_cast<const Four *>(src + l0);
    ahead[1] = *reinterpret_cast<const Four *>(src + l1);
  };
  // The first rows come while the angles are worked out.
  load(p.k_cache != nullptr || part < of_q + of_k ? part : 0);
  Four gamma[2][2];
  const bool q_gamma = p.norm && p.q_gamma != nullptr, k_gamma = p.norm && p.k_gamma != nullptr;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = i == 0 ? l0 : l1;
    if (q_gamma) gamma[0][i] = *reinterpret_cast<const Four *>(static_cast<const elem *>(p.q_gamma) + at);
    if (k_gamma) gamma[1][i] = *reinterpret_cast<const Four *>(static_cast<const elem *>(p.k_gamma) + at);
  }
  const int64_t slot = p.k_cache != nullptr ? p.slots[t] : -1;
  const bool cached = slot >= 0 && slot < p.rows;
  const int64_t page = cached ? slot / p.page_size : 0, in_page = cached ? slot - page * p.page_size : 0;
  const int steps = of_q + of_k + (cached ? of_k : 0);
  const float inverse_d = 1.0f / (float)d;

  float c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = 1.0f, s[i] = 0.0f;
  if (turned) {
    const double pos = static_cast<double>(p.positions[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) turn(pos * static_cast<double>(p.inv_freq[4 * u + i]), c[i], s[i]);
  }
  for (int step = part; step < steps; step += parts) {
    const bool is_q = step < of_q, is_v = step >= of_q + of_k;
    const Four raw[2] = {ahead[0], ahead[1]};
    // The next step's rows while this one's are worked on (in place, they are
    // nobody else's); behind the last, this one's once more.
    load(step + parts < steps ? step + parts : step);
    const int n = is_q ? q_heads : kv_heads, h = (step - (is_q ? 0 : is_v ? of_q + of_k : of_q)) * kRows + lane / L;
    const bool on = live && h < n;
    if (is_v) {
      if (on) {
        elem *dst = static_cast<elem *>(p.v_cache) + page * p.v_page + in_page * p.v_slot + h * p.v_head;
        __builtin_nontemporal_store(raw[0], reinterpret_cast<Four *>(dst + a0));
        __builtin_nontemporal_store(raw[1], reinterpret_cast<Four *>(dst + a1));
      }
      continue;
    }
    float x[2][4];
    unpack(x[0], raw[0]);
    unpack(x[1], raw[1]);
    if (p.norm) {
      float sq = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sq += x[0][i] * x[0][i] + x[1][i] * x[1][i];
      const float scale = inverse_root(row_sum<L>(live ? sq : 0.0f) * inverse_d + p.eps);
      const bool weighted = is_q ? q_gamma : k_gamma;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (weighted) unpack(g, is_q ? gamma[0][half] : gamma[1][half]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[half][i] *= scale * g[i];
      }
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
    if (on && (is_q || p.k_out != nullptr)) {
      elem *dst = is_q ? static_cast<elem *>(p.q_out) + t * p.q_out_stride : static_cast<elem *>(p.k_out) + t * p.k_out_stride;
      dst += (int64_t)h * d;
      store_past(dst + a0, x[0]);
      store_past(dst + a1, x[1]);
    }
    if (on && !is_q && cached) {
      elem *dst = static_cast<elem *>(p.k_cache) + page * p.k_page + in_page * p.k_slot + h * p.k_head;
      store_past(dst + a0, x[0]);
      store_past(dst + a1, x[1]);
    }
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_8)(const KhRopeParams p) { rope<8>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_16)(const KhRopeParams p) { rope<16>(p); }
extern "C" __global__ void __launch_bounds__(256) KH_TYPED(qk_norm_rope_32)(const KhRopeParams p) { rope<32>(p); }
