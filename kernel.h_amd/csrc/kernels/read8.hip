// Rows of a paged cache in 8 bits, read back in fp32, fp16 or bf16: for each token
// the rows of all kv heads in its slot, each number its e4m3 value times its row's
// power of two (exact but in fp16, where it is rounded once and may be infinite).
//
// Bound by memory, the writes more than the reads. A workgroup takes the K or the V
// of a few tokens: their places are worked out once, a token to a thread, and the
// rows of a token's heads, which follow each other in the output, are written 16
// bytes a lane, several of them on their way at once.
#include "kh_elem.h"
#include "kh_paged.h"

namespace {

using kh::elem;
using kh::f32x2;
using kh::kPer16;
using kh::u32x4;

constexpr int kThreads = 256, kAhead = 4;

// `kPer16` numbers, a byte each, times a power of two, in the elements' type.
__device__ __forceinline__ u32x4 widen(const uint32_t (&w)[kPer16 / 4], float power) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < kPer16 / 4; ++i) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
#if KH_ELEM == 0
    out = u32x4{__float_as_uint(a.x * power), __float_as_uint(a.y * power), __float_as_uint(b.x * power), __float_as_uint(b.y * power)};
#else
    out[2 * i] = kh::pack2(a.x * power, a.y * power);
    out[2 * i + 1] = kh::pack2(b.x * power, b.y * power);
#endif
  }
  return out;
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) KH_TYPED(read8)(const KhRead8Params p) {
  __shared__ uint64_t rows[kThreads], scales[kThreads];
  __shared__ int there[kThreads];
  const bool is_v = blockIdx.y != 0;
  const char *base = reinterpret_cast<const char *>(is_v ? p.v : p.k);
  const uint8_t *scale_base = is_v ? p.v_scale : p.k_scale;
  const uint32_t page_stride = is_v ? p.v_page : p.k_page, slot_stride = is_v ? p.v_slot : p.k_slot, head_stride = is_v ? p.v_head : p.k_head;
  elem *out = static_cast<elem *>(is_v ? p.v_out : p.k_out);
  if (out == nullptr) return;
  const int64_t out_stride = is_v ? p.v_out_stride : p.k_out_stride;
  const int64_t t0 = (int64_t)blockIdx.x * p.each;
  const int tokens = p.tokens - t0 < p.each ? (int)(p.tokens - t0) : p.each;  // each <= kThreads
  if ((int)threadIdx.x < tokens) {
    const int64_t slot = p.slots[t0 + threadIdx.x];
    const bool cached = slot >= 0 && slot < p.rows;
    const uint64_t page = cached ? (uint64_t)slot / (uint32_t)p.page_size : 0;
    const uint32_t in_page = cached ? (uint32_t)((uint64_t)slot - page * (uint32_t)p.page_size) : 0;
    rows[threadIdx.x] = page * page_stride + (uint64_t)in_page * slot_stride;
    scales[threadIdx.x] = page * p.scale_page + in_page;
    there[threadIdx.x] = cached;
  }
  kh::lds_barrier();
  const uint32_t items = (uint32_t)tokens * p.by_token.by;  // below 2^31: one token's pieces are, and more have few
  for (uint32_t x0 = threadIdx.x; x0 < items; x0 += kThreads * kAhead) {
    uint32_t w[kAhead][kPer16 / 4];
    float power[kAhead];
    elem *to[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const uint32_t x = x0 + j * kThreads < items ? x0 + j * kThreads : x0;
      const uint32_t t = kh_div(x, p.by_token), in = x - t * p.by_token.by;
      const uint32_t head = kh_div(in, p.by_row), col = (in - head * p.by_row.by) * kPer16;
      const char *from = base + rows[t] + (uint64_t)head * head_stride + col;
      if constexpr (kPer16 == 8) {
        const kh::u32x2 g = __builtin_nontemporal_load(reinterpret_cast<const kh::u32x2 *>(from));
        w[j][0] = g.x, w[j][kPer16 / 4 - 1] = g.y;
      } else {
        w[j][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(from));
      }
      const uint32_t byte = scale_base[scales[t] + (uint64_t)head * p.scale_head];
      const uint32_t up = byte > KH_SCALE_LEAST ? byte : KH_SCALE_LEAST;
      power[j] = __uint_as_float((up < KH_SCALE_MOST ? up : KH_SCALE_MOST) << 23);
      to[j] = there[t] != 0 ? out + (t0 + t) * out_stride + (int64_t)in * kPer16 : nullptr;
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (x0 + j * kThreads < items && to[j] != nullptr)
        __builtin_nontemporal_store(widen(w[j], power[j]), reinterpret_cast<u32x4 *>(to[j]));
  }
}
