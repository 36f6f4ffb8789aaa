// Eviction from a paged cache by accumulated attention weight, for each kv
// head of each sequence on its own: of n entries the `recent` newest stay, and
// of the others the budget - recent of largest weight, of equal weights those
// of lowest index. Entries keep their order and go to the pages of another
// table; a sequence of no more than budget entries is copied whole.
//
// Two kernels. paged_evict_choose, a workgroup per (sequence, head), finds the
// smallest kept weight a byte at a time (four histograms of the weights' bits,
// made to order like unsigned integers) and then lists the kept entries in
// order, with their weights. paged_evict_move_* copies the rows, 16 bytes to a
// lane: bound by memory, every kept row is read once and written once.
//
// Weights are sums of exponentials, but any 32 bits are ordered: -0 counts as
// 0, a NaN as larger than all else.
#include "kh_device.h"
#include "kh_paged.h"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kh::kWave;

__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 + 0 = 0
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return (u >> 31) != 0 ? ~u : u | 0x80000000u;
}

// Lanes of the wave below this one for which `on` holds.
__device__ __forceinline__ int below(uint64_t on) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(on >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)on, 0));
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads) paged_evict_choose(const KhEvictParams p) {
  __shared__ uint32_t histogram[256];
  __shared__ uint32_t found[2];      // the byte's value, how many are still wanted
  __shared__ uint32_t counts[2][kWaves];
  const int tid = threadIdx.x, lane = kh::lane_id(), wave = tid / kh::kWave;
  const int head = (int)(blockIdx.x % (uint32_t)p.cache.kv_heads), seq = (int)(blockIdx.x / (uint32_t)p.cache.kv_heads);
  const int n = kh_clamp(p.table.lens[seq], 0, p.table.capacity);
  const int kept = n < p.budget ? n : p.budget;
  const float *in = p.weights_in + seq * p.in_seq_stride + head * p.in_head_stride;
  float *out = p.weights + seq * p.seq_stride + head * p.head_stride;
  int32_t *chosen = p.chosen + (int64_t)blockIdx.x * p.budget;
  if (head == 0 && tid == 0) p.kept_lens[seq] = kept;
  if (kept == n) {
    for (int j = tid; j < n; j += kThreads) {
      chosen[j] = j;
      out[j] = in[j];
    }
    return;
  }
  // n > budget >= recent.
  const int old = n - p.recent;
  uint32_t wanted = (uint32_t)(p.budget - p.recent), limit = 0;  // of limit the bytes found so far
  if (wanted > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) histogram[tid] = 0;
      __syncthreads();
      const uint32_t known = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int j = tid; j < old; j += kThreads) {
        const uint32_t o = order_of(in[j]);
        if ((o & known) == limit) atomicAdd(&histogram[o >> shift & 255u], 1u);
      }
      __syncthreads();
      // From the largest byte down, where the count first reaches `wanted`.
      if (wave == 0) {
        uint32_t c[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += c[i] = histogram[255 - 4 * lane - i];
        uint32_t upto = mine;
#pragma unroll
        for (int i = 1; i < kh::kWave; i *= 2) {
          const uint32_t x = __shfl_up(upto, i, kh::kWave);
          if (lane >= i) upto += x;
        }
        uint32_t before = upto - mine;
        if (before < wanted && upto >= wanted) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (before < wanted && before + c[i] >= wanted) {
              found[0] = 255u - 4 * lane - i;
              found[1] = wanted - before;
            }
            before += c[i];
          }
        }
      }
      __syncthreads();
      limit |= found[0] << shift;
      wanted = found[1];
      __syncthreads();
    }
  }
  // All weights above the limit are kept, and the first `wanted` at it.
  const bool none = p.budget == p.recent;
  uint32_t to = 0, ties = 0;
  for (int j0 = 0; j0 < n; j0 += kThreads) {
    const int j = j0 + tid;
    const float w = j < n ? in[j] : 0.0f;
    const uint32_t o = order_of(w);
    const bool inside = j < old && !none;
    const bool tie = inside && o == limit;
    const uint64_t tied = __builtin_amdgcn_ballot_w64(tie);
    if (lane == 0) counts[0][wave] = (uint32_t)__popcll(tied);
    __syncthreads();
    uint32_t ties_before = ties, all_ties = ties;
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) ties_before += counts[0][i];
      all_ties += counts[0][i];
    }
    const bool keep = (j < n && j >= old) || (inside && o > limit) || (tie && ties_before + below(tied) < wanted);
    const uint64_t kept_here = __builtin_amdgcn_ballot_w64(keep);
    if (lane == 0) counts[1][wave] = (uint32_t)__popcll(kept_here);
    __syncthreads();
    uint32_t at = to;
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) at += counts[1][i];
      to += counts[1][i];
    }
    at += below(kept_here);
    if (keep && at < (uint32_t)kept) {
      chosen[at] = j;
      out[at] = w;
    }
    ties = all_ties;
  }
}

// Rows of the chosen entries, a piece of 16 bytes to a lane and step.
extern "C" __global__ void __launch_bounds__(256) paged_evict_move(const KhEvictParams p) {
  const int head = (int)(blockIdx.x % (uint32_t)p.cache.kv_heads), seq = (int)(blockIdx.x / (uint32_t)p.cache.kv_heads);
  const int n = kh_clamp(p.table.lens[seq], 0, p.table.capacity);
  const int kept = n < p.budget ? n : p.budget;
  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const int32_t *kept_table = p.kept_pages + seq * p.kept_row_stride;
  const int32_t *chosen = p.chosen + (int64_t)blockIdx.x * p.budget;
  const char *k = p.cache.k + (uint64_t)head * p.cache.k_head, *v = p.cache.v + (uint64_t)head * p.cache.v_head;
  const int pieces = p.cache.head_dim * p.element / 16;
  const int64_t all = (int64_t)kept * pieces;
  for (int64_t at = (int64_t)blockIdx.y * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.y * 256) {
    const int row = (int)(at / pieces), piece = (int)(at - (int64_t)row * pieces);
    const KhSlot a = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)chosen[row]);
    const KhSlot b = kh_slot(kept_table, p.kept_width, p.cache.pages, p.cache.by_page, (uint32_t)row);
    if (a.page < 0 || b.page < 0) continue;
    const float4 x = *reinterpret_cast<const float4 *>(k + kh_row(a, p.cache.k_page, p.cache.k_slot) + 16 * piece);
    const float4 y = *reinterpret_cast<const float4 *>(v + kh_row(a, p.cache.v_page, p.cache.v_slot) + 16 * piece);
    *reinterpret_cast<float4 *>(const_cast<char *>(k) + kh_row(b, p.cache.k_page, p.cache.k_slot) + 16 * piece) = x;
    *reinterpret_cast<float4 *>(const_cast<char *>(v) + kh_row(b, p.cache.v_page, p.cache.v_slot) + 16 * piece) = y;
  }
}
