// Element types of the sequence-cache kernels: storage, conversions and the
// matrix instructions that take them. A code object is built per type, with
// KH_ELEM 0 (fp32), 1 (fp16) or 2 (bf16).
#pragma once

#include "kh_device.h"

namespace kh {

#if KH_ELEM == 0
using elem = float;
#elif KH_ELEM == 1
using elem = _Float16;
#else
using elem = __bf16;
#endif

constexpr bool kWide = KH_ELEM == 0;        // 32-bit elements
constexpr int kPer16 = 16 / sizeof(elem);   // elements in 16 bytes

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
#if KH_ELEM != 0
typedef elem half2 __attribute__((ext_vector_type(2)));
typedef elem half8 __attribute__((ext_vector_type(8)));
#endif

// Two floats rounded to nearest even and packed (16-bit types).
#if KH_ELEM != 0
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const half2 h = {static_cast<elem>(a), static_cast<elem>(b)};
  return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ float low_of(uint32_t w) {
#if KH_ELEM == 2
  return __uint_as_float(w << 16);
#else
  return static_cast<float>(__builtin_bit_cast(half2, w).x);
#endif
}
__device__ __forceinline__ float high_of(uint32_t w) {
#if KH_ELEM == 2
  return __uint_as_float(w & 0xffff0000u);
#else
  return static_cast<float>(__builtin_bit_cast(half2, w).y);
#endif
}
#endif

// Four consecutive elements as floats, and back.
__device__ __forceinline__ void load4(float (&x)[4], const elem *p) {
#if KH_ELEM == 0
  const f32x4 v = *reinterpret_cast<const f32x4 *>(p);
  x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
#else
  const u32x2 v = *reinterpret_cast<const u32x2 *>(p);
  x[0] = low_of(v.x), x[1] = high_of(v.x), x[2] = low_of(v.y), x[3] = high_of(v.y);
#endif
}
__device__ __forceinline__ void store4(elem *p, const float (&x)[4]) {
#if KH_ELEM == 0
  *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
#else
  *reinterpret_cast<u32x2 *>(p) = u32x2{pack2(x[0], x[1]), pack2(x[2], x[3])};
#endif
}

// Whether any of the elements packed in w is an infinity or a NaN.
__device__ __forceinline__ bool not_finite(uint32_t w) {
#if KH_ELEM == 0
  return (w & 0x7fffffffu) >= 0x7f800000u;
#else
  constexpr uint32_t top = KH_ELEM == 1 ? 0x7c00u : 0x7f80u;
  return (w & 0x7fffu) >= top || (w & 0x7fff0000u) >= top << 16;
#endif
}

// acc += A B over 64 bytes of each row (16 rows of A, 16 columns of B): lane
// l holds bytes 16 (l / 16) .. + 15 of row, respectively column, l % 16. The
// result's column is l % 16, its rows 4 (l / 16) + i.
__device__ __forceinline__ f32x4 mma16(u32x4 a, u32x4 b, f32x4 acc) {
#if KH_ELEM == 0
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
  return acc;
#elif KH_ELEM == 1
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0, 0, 0);
#else
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0, 0, 0);
#endif
}

// The same over 32 bytes of 32 rows and 32 columns: lane l holds bytes
// 16 (l / 32) .. + 15 of row, respectively column, l % 32. The result's column is
// l % 32, its rows 8 (i / 4) + 4 (l / 32) + i % 4.
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 acc) {
#if KH_ELEM == 0
#pragma unroll
  for (int i = 0; i < 4; ++i)
    acc = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i]), __uint_as_float(b[i]), acc, 0, 0, 0);
  return acc;
#elif KH_ELEM == 1
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0, 0, 0);
#else
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0, 0, 0);
#endif
}

// One wave's load straight to LDS: lane l's 16 bytes at byte voff of the resource
// land at LDS byte address lds + 16 l. Inline assembly on purpose: the compiler
// cannot prove the places disjoint from those it reads, and would wait for its
// own form of this load before every later LDS read. The caller waits
// (vm_wait) before the barrier that hands the bytes over. The resource and `lds`
// are the same in all lanes. M0 carries the LDS address; it is saved and restored.
// A vector instruction's write of a scalar register (the resource's words may
// come straight from v_readfirstlane) needs five wait states before a load reads
// it, a write of M0 one: the compiler does not look into the assembly, so they are
// counted here, two moves and three more.
#define KH_DMA(load)                        \
  uint32_t saved;                           \
  asm volatile(                             \
      "s_mov_b32 %0, m0\n\t"                \
      "s_mov_b32 m0, %1\n\t"                \
      "s_nop 2\n\t" load                    \
      " %2, %3, 0 offen lds\n\t"            \
      "s_mov_b32 m0, %0"                    \
      : "=&s"(saved)                        \
      : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(rsrc) \
      : "memory")
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t voff, uint32_t lds) {
#pragma unroll
  for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
  KH_DMA("buffer_load_dwordx4");
}

// The same for 4 bytes a lane.
__device__ __forceinline__ void dma4(u32x4 rsrc, uint32_t voff, uint32_t lds) {
#pragma unroll
  for (int i = 0; i < 4; ++i) rsrc[i] = __builtin_amdgcn_readfirstlane(rsrc[i]);
  KH_DMA("buffer_load_dword");
}
#undef KH_DMA

// For LDS that the wave alone uses: all but the last N vector-memory operations
// are done, and what they brought is read after this.
template <int N>
__device__ __forceinline__ void arrived() {
  vm_wait<N>();
  asm volatile("" ::: "memory");
}

#if KH_ELEM != 0
// Of 4 x 16 elements in LDS that the 16 lanes of a row point at (lane 4 r + c:
// row r, columns 4 c ..), lane i receives column i, its four rows in order
// (ds_read_b64_tr_b16).
__device__ __forceinline__ u32x2 read_across(const char *p) {
  typedef short s16x4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4 *)const_cast<char *>(p)));
}
#endif

}  // namespace kh

#define KH_PASTE2(a, b) a##_##b
#define KH_PASTE(a, b) KH_PASTE2(a, b)
#if KH_ELEM == 0
#define KH_TYPED(name) KH_PASTE(name, f32)
#elif KH_ELEM == 1
#define KH_TYPED(name) KH_PASTE(name, f16)
#else
#define KH_TYPED(name) KH_PASTE(name, bf16)
#endif
