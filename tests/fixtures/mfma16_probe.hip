// Test-only code object: the 16-bit matrix instructions and the transposing
// LDS read one at a time, so that a GPU test can check the lane layouts the
// sequence-cache kernels rely on. Operands are 16-bit patterns (fp16 for the
// products), written and read unchanged. One wavefront.
#include "kh_device.h"

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

extern "C" __global__ void __launch_bounds__(64)
probe_mfma_16x16x32_f16(const _Float16 *__restrict__ a, const _Float16 *__restrict__ b, float *__restrict__ out) {
  const int l = threadIdx.x;
  h8 x, y;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = a[l * 8 + i], y[i] = b[l * 8 + i];
  v4f acc = {};
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 4; ++r) out[l * 4 + r] = acc[r];
}

extern "C" __global__ void __launch_bounds__(64)
probe_mfma_32x32x16_f16(const _Float16 *__restrict__ a, const _Float16 *__restrict__ b, float *__restrict__ out) {
  const int l = threadIdx.x;
  h8 x, y;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = a[l * 8 + i], y[i] = b[l * 8 + i];
  v16f acc = {};
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, acc, 0, 0, 0);
#pragma unroll
  for (int r = 0; r < 16; ++r) out[l * 16 + r] = acc[r];
}

// ds_read_b64_tr_b16: each lane gives the address of four 16-bit values (at
// index 4 l here) and receives four of its 16 lanes' 64.
extern "C" __global__ void __launch_bounds__(64)
probe_read_tr16(const short *__restrict__ a, const short *__restrict__ unused, short *__restrict__ out) {
  __shared__ short lds[256];
  const int l = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) lds[l * 4 + i] = a[l * 4 + i];
  __syncthreads();
  const s4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4 *)(lds + l * 4));
#pragma unroll
  for (int i = 0; i < 4; ++i) out[l * 4 + i] = r[i];
}
