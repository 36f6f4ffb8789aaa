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
//
// Built with KH_CACHE8 the cache is one in 8 bits (rope8_*): pair i is rotated by
// the position of its own axis, and a row of k or v becomes e4m3 numbers times the
// least power of two 2^e, e >= -117, with which the row's largest is at most 448:
// the type's relative step is the same under any scale, so that a power of two loses
// nothing by it, and what is read back is exact. Rows of k are worked out in 64 bits,
// the angles' series too, and rounded once: between two numbers of four bits there are
// ties, which 32 bits take either way (17 of 8 million numbers). Infinities and NaN
// become NaN; a row's power is that of its finite elements. A wave's token, part and
// page are the same in all lanes, and are kept so. The 8192 tokens take 41-44 us, 4.2-4.5
// TB/s: fewer bytes, but as many rows to work through, each with a maximum across its
// lanes (in 32 bits 42). 5 fp32 tokens of 16 heads of 64 7 us, a launch and one row's way
// through (6.3 in 32 bits).
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

#ifdef KH_CACHE8
// The series in 64 bits too (first terms left out 7e-12 and 4e-13).
__device__ __forceinline__ void turn(double angle, double &c, double &s) {
  const double quarters = angle * 0.63661977236758134308;  // 2 / pi
  const double whole = __builtin_rint(quarters);
  const double x = (quarters - whole) * 1.57079632679489661923;
  const int q = static_cast<int>(static_cast<int64_t>(whole)) & 3;
  const double z = x * x;
  const double si = x + x * z * (-1.0 / 6 + z * (1.0 / 120 + z * (-1.0 / 5040 + z * (1.0 / 362880 + z * (-1.0 / 39916800)))));
  const double co =
      1.0 + z * (-0.5 + z * (1.0 / 24 + z * (-1.0 / 720 + z * (1.0 / 40320 + z * (-1.0 / 3628800 + z * (1.0 / 479001600))))));
  const double a = (q & 1) != 0 ? si : co, b = (q & 1) != 0 ? co : si;
  c = q == 1 || q == 2 ? -a : a;
  s = q >= 2 ? -b : b;
}
#else
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
#endif

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

#ifdef KH_CACHE8
template <int CONTROL>
__device__ __forceinline__ double moved(double v) {
  const uint64_t w = __builtin_bit_cast(uint64_t, v);
  const uint32_t low = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)w, CONTROL, 0xf, 0xf, false);
  const uint32_t high = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(w >> 32), CONTROL, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)high << 32 | low);
}

template <int L>
__device__ __forceinline__ double row_sum(double v) {
  v += moved<0xb1>(v);
  v += moved<0x4e>(v);
  v += moved<0x141>(v);
  if constexpr (L >= 16) v += moved<0x140>(v);
  if constexpr (L >= 32) v += __shfl_xor(v, 16, kh::kWave);
  return v;
}

// In 64 bits: the instruction's 2^-25 or so, and a Newton step.
__device__ __forceinline__ double inverse_root(double x) {
  const double y = __builtin_amdgcn_rsq(x);
  const double z = y * (1.5 - 0.5 * x * y * y);
  return x > 0.0 && x < __builtin_inf() ? z : y;
}

// y in 21 bits, the last of them set where that is not all of it: rounded further to
// nearest, it becomes what y does.
__device__ __forceinline__ float leading(double y) {
  const uint64_t w = __builtin_bit_cast(uint64_t, y);
  const uint32_t high = (uint32_t)(w >> 32) | ((uint32_t)w != 0 ? 1u : 0u);
  return static_cast<float>(__builtin_bit_cast(double, (uint64_t)high << 32));
}
#endif

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

#ifdef KH_CACHE8
using Params = KhRope8Params;

struct Turn {
  double c, s;
};

// The largest over the L lanes of a row.
template <int L>
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, moved<0xb1>(v));  // as row_sum
  v = fmaxf(v, moved<0x4e>(v));
  v = fmaxf(v, moved<0x141>(v));
  if constexpr (L >= 16) v = fmaxf(v, moved<0x140>(v));
  if constexpr (L >= 32) v = fmaxf(v, __shfl_xor(v, 16, kh::kWave));
  return v;
}

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7fffffffu) < 0x7f800000u; }

// The byte of the least power of two 2^e with 448 2^e = 1.75 2^(e + 8) >= top.
__device__ __forceinline__ uint32_t scale_of(float top) {
  const uint32_t w = __float_as_uint(top);
  const int byte = (int)(w >> 23) - 8 + ((w & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)(byte < KH_SCALE_LEAST ? KH_SCALE_LEAST : byte < KH_SCALE_MOST ? byte : KH_SCALE_MOST);
}

// Four numbers times a power of two as e4m3, rounded to nearest even; past 448,
// as only the largest scale leaves some, they are 448.
__device__ __forceinline__ uint32_t narrowed(const float (&x)[4], float power) {
  float y[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = is_finite(x[i]) ? fminf(fmaxf(x[i] * power, -448.0f), 448.0f) : __builtin_nanf("");
  const uint32_t low = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], (int)low, true);
}

// A lane's eight elements of a row to the cache, the row's scale by its first lane.
template <int L>
__device__ __forceinline__ void store8(const float (&x)[2][4], bool live, bool on, uint8_t *row, int a0, int a1, uint8_t *scale, int u) {
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = x[i / 4][i % 4];
    top = fmaxf(top, is_finite(y) ? fabsf(y) : 0.0f);
  }
  const uint32_t byte = scale_of(row_max<L>(live ? top : 0.0f));
  if (!on) return;
  const float power = __uint_as_float((254 - byte) << 23);  // 2^(127 - byte), byte in [10, 246]
  __builtin_nontemporal_store(narrowed(x[0], power), reinterpret_cast<uint32_t *>(row + a0));
  __builtin_nontemporal_store(narrowed(x[1], power), reinterpret_cast<uint32_t *>(row + a1));
  if (u == 0) *scale = (uint8_t)byte;
}
#else
using Params = KhRopeParams;
#endif

template <int L>
__device__ __forceinline__ void rope(const Params &p) {
  using kh::elem;
  const int lane = kh::lane_id();
  // A job is one part of one token's heads; a wave takes one.
#ifdef KH_CACHE8
  // Fewer than 2^31 jobs: the launcher sees to it.
  const uint32_t job = blockIdx.x * (256 / kh::kWave) + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x / kh::kWave);
  const int64_t t = kh_div(job, p.by_parts);
  const int part = (int)(job - (uint32_t)t * p.by_parts.by);
#else
  const int64_t job = (int64_t)blockIdx.x * (256 / kh::kWave) + threadIdx.x / kh::kWave;
  const int64_t t = job / p.parts;
  const int part = (int)(job - t * p.parts);
#endif
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
#ifdef KH_CACHE8
    const uint32_t row = (uint32_t)(h < n ? h : n - 1) * (uint32_t)d;  // below 2^24
    ahead[0] = *reinterpret_cast<const Four *>(src + (row + (uint32_t)l0));
    ahead[1] = *reinterpret_cast<const Four *>(src + (row + (uint32_t)l1));
    return;
#endif
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
#ifdef KH_CACHE8
  // A division in 64 bits takes 125 instructions; few caches have 2^31 slots.
  const bool near = slot < int64_t(1) << 31;
  const int64_t page = !cached ? 0 : near ? (int64_t)kh_div((uint32_t)slot, p.by_page) : slot / p.page_size;
  const int64_t in_page = cached ? slot - page * p.page_size : 0;
#else
  const int64_t page = cached ? slot / p.page_size : 0, in_page = cached ? slot - page * p.page_size : 0;
#endif
  const int steps = of_q + of_k + (cached ? of_k : 0);
  const float inverse_d = 1.0f / (float)d;

  float c[4], s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = 1.0f, s[i] = 0.0f;
#ifdef KH_CACHE8
  __shared__ Turn of_waves[256 / kh::kWave][4][L];
  Turn(*const turns)[L] = of_waves[threadIdx.x / kh::kWave];
#endif
  if (turned) {
#ifdef KH_CACHE8
    // A lane works out kOwn of its row's four angles, and gets the others by way of LDS
    // from the lanes with the same elements of the other rows of the wave.
    constexpr int kOwn = L == 32 ? 2 : 1;
    const int own = 4 * u + (lane / L * kOwn) % 4;
    int axis[kOwn];
    float freq[kOwn];
    double co[kOwn], si[kOwn];
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      axis[i] = p.pair_axis != nullptr ? p.pair_axis[own + i] : 0;
      freq[i] = p.inv_freq[own + i];
    }
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      turn(static_cast<double>(p.positions[kh_clamp(axis[i], 0, p.axes - 1) * p.axis_stride + t]) * static_cast<double>(freq[i]), co[i], si[i]);
    // The wave's own part of LDS: nobody else waits for it.
#pragma unroll
    for (int i = 0; i < kOwn; ++i) turns[(lane / L * kOwn + i) % 4][u] = Turn{co[i], si[i]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const Turn at = turns[i][u];
      c[i] = static_cast<float>(at.c), s[i] = static_cast<float>(at.s);
    }
#else
    const double pos = static_cast<double>(p.positions[t]);
#pragma unroll
    for (int i = 0; i < 4; ++i) turn(pos * static_cast<double>(p.inv_freq[4 * u + i]), c[i], s[i]);
#endif
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
#ifdef KH_CACHE8
      float y[2][4];
      unpack(y[0], raw[0]);
      unpack(y[1], raw[1]);
      const int64_t at = page * p.v_page + in_page * p.v_slot + h * p.v_head;
      store8<L>(y, live, on, static_cast<uint8_t *>(p.v_cache) + at, a0, a1,
                p.v_scale + (page * p.scale_page + h * p.scale_head + in_page), u);
#else
      if (on) {
        elem *dst = static_cast<elem *>(p.v_cache) + page * p.v_page + in_page * p.v_slot + h * p.v_head;
        __builtin_nontemporal_store(raw[0], reinterpret_cast<Four *>(dst + a0));
        __builtin_nontemporal_store(raw[1], reinterpret_cast<Four *>(dst + a1));
      }
#endif
      continue;
    }
    float x[2][4];
    unpack(x[0], raw[0]);
    unpack(x[1], raw[1]);
#ifdef KH_CACHE8
    if (!is_q) {
      // In 64 bits: a row is rounded once, to four bits a number. In 32, ties between
      // two of them go either way: of 8192 tokens' 8 heads of 128 17 numbers.
      double scale = 1.0;
      if (p.norm) {
        double sq = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += static_cast<double>(x[i / 4][i % 4]) * static_cast<double>(x[i / 4][i % 4]);
        scale = inverse_root(row_sum<L>(live ? sq : 0.0) * p.inverse_d + static_cast<double>(p.eps));
      }
      float g[2][4];
      unpack(g[0], gamma[1][0]);
      unpack(g[1], gamma[1][1]);
      auto weighted = [&](int half, int i) {
        if (!k_gamma) return static_cast<double>(x[half][i]);
        // Exact in 16 bits' types.
        return KH_ELEM == 0 ? static_cast<double>(x[half][i]) * static_cast<double>(g[half][i]) : static_cast<double>(x[half][i] * g[half][i]);
      };
      elem *const k_out = static_cast<elem *>(p.k_out) + t * p.k_out_stride;
      float exact[2][4];  // fp32's own rounding, for k_out
      auto pair = [&](int ha, int ia, int hb, int ib, int i) {
        double y = weighted(ha, ia), z = weighted(hb, ib);
        if (turned) {
          const Turn at = turns[i][u];
          const double first = y * at.c - z * at.s;
          z = z * at.c + y * at.s;
          y = first;
        }
        y *= scale, z *= scale;
        if (KH_ELEM == 0) exact[ha][ia] = static_cast<float>(y), exact[hb][ib] = static_cast<float>(z);
        x[ha][ia] = leading(y), x[hb][ib] = leading(z);
      };
      if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) pair(i / 2, 2 * (i % 2), i / 2, 2 * (i % 2) + 1, i);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) pair(0, i, 1, i, i);
      }
      if (on && p.k_out != nullptr) {
        const uint32_t row = (uint32_t)h * (uint32_t)d;
        store_past(k_out + (row + (uint32_t)a0), KH_ELEM == 0 ? exact[0] : x[0]);
        store_past(k_out + (row + (uint32_t)a1), KH_ELEM == 0 ? exact[1] : x[1]);
      }
      if (cached) {
        const int64_t at = page * p.k_page + in_page * p.k_slot + h * p.k_head;
        store8<L>(x, live, on, static_cast<uint8_t *>(p.k_cache) + at, a0, a1,
                  p.k_scale + (page * p.scale_page + h * p.scale_head + in_page), u);
      }
      continue;
    }
#endif
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
#ifdef KH_CACHE8
    if (on) {
      elem *const dst = static_cast<elem *>(p.q_out) + t * p.q_out_stride;
      const uint32_t row = (uint32_t)h * (uint32_t)d;
      store_past(dst + (row + (uint32_t)a0), x[0]);
      store_past(dst + (row + (uint32_t)a1), x[1]);
    }
#else
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
#endif
  }
}

}  // namespace

#ifdef KH_CACHE8
// Six waves to a SIMD where the elements leave registers for it: 1999 fp16 tokens of 24
// heads of 96 17.4 us, 18.8 with five; fp32 would spill 37 and has four.
#define KH_ROPE(name) __launch_bounds__(256, KH_ELEM == 0 ? 1 : 6) KH_TYPED(rope8_##name)
#else
#define KH_ROPE(name) __launch_bounds__(256) KH_TYPED(qk_norm_rope_##name)
#endif
extern "C" __global__ void KH_ROPE(8)(const Params p) { rope<8>(p); }
extern "C" __global__ void KH_ROPE(16)(const Params p) { rope<16>(p); }
extern "C" __global__ void KH_ROPE(32)(const Params p) { rope<32>(p); }
