// Eviction from a paged cache by accumulated attention weight, for each kv
// head of each sequence on its own: of n entries the `recent` newest stay, and
// of the others the budget - recent of largest weight, of equal weights those
// of lowest index. Entries keep their order and go to the pages of another
// table; a sequence of no more than budget entries is copied whole.
//
// Two kernels. paged_evict_choose, a workgroup per (sequence, head), finds the
// smallest kept weight a byte at a time (four histograms of the weights' bits,
// made to order like unsigned integers) and then lists the kept entries in
// order, with their weights. Up to 16384 entries it holds them in registers,
// consecutive ones to a thread, so that one sum over the workgroup places them
// all; longer rows are read again for each step. paged_evict_move copies the
// rows, 16 bytes to a lane: bound by memory, every kept row is read once and
// written once, with stores that pass the caches by. 16 sequences of 8 heads of
// 128 (bf16), 4096 entries kept of 4200 to 4352: 14 us and 97 to 108 us (5.0 to
// 5.5 TB/s).
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

// Of the 256 counts, from the largest value down: the first at which they reach
// `wanted`, and how many of that value are wanted. By one wave, into found.
__device__ __forceinline__ void pick(const uint32_t (&histogram)[256], uint32_t wanted, uint32_t (&found)[2], int lane) {
  uint32_t c[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) mine += c[i] = histogram[255 - 4 * lane - i];
  const uint32_t upto = kh::up_to(mine);
  uint32_t before = upto - mine;
  if (before >= wanted || upto < wanted) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (before < wanted && before + c[i] >= wanted) {
      found[0] = 255u - 4 * lane - i;
      found[1] = wanted - before;
    }
    before += c[i];
  }
}

struct Shared {
  uint32_t histogram[256];
  uint32_t found[2];
  uint32_t counts[2][kWaves];
};

// The smallest kept weight's order in `limit`, and how many of that order are
// kept. each(count) calls count(order) for the thread's share of the old entries.
template <class Each>
__device__ __forceinline__ uint32_t smallest_kept(Shared &sh, uint32_t wanted, uint32_t &limit, int tid, int lane, Each &&each) {
  limit = 0;
  if (wanted == 0) return 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) sh.histogram[tid] = 0;
    __syncthreads();
    const uint32_t known = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    each([&](uint32_t o) {
      if ((o & known) == limit) atomicAdd(&sh.histogram[o >> shift & 255u], 1u);
    });
    __syncthreads();
    if (tid < kh::kWave) pick(sh.histogram, wanted, sh.found, lane);
    __syncthreads();
    limit |= sh.found[0] << shift;
    wanted = sh.found[1];
  }
  return wanted;
}

// Sum over the threads before this one, and over all.
__device__ __forceinline__ uint32_t before_me(uint32_t v, uint32_t (&counts)[kWaves], int lane, int wave, uint32_t &all) {
  const uint32_t upto = kh::up_to(v);
  if (lane == kh::kWave - 1) counts[wave] = upto;
  __syncthreads();
  uint32_t before = 0;
  all = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    if (i < wave) before += counts[i];
    all += counts[i];
  }
  return before + upto - v;
}

// Up to E x 1024 entries, E consecutive ones to a thread.
template <int E>
__device__ __forceinline__ void choose_held(const float *in, float *out, int32_t *chosen, int n, int kept, int old, uint32_t wanted,
                                            Shared &sh, int tid, int lane, int wave) {
  float w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = in[E * tid + e < n ? E * tid + e : n - 1];
  uint32_t limit;
  const bool some = wanted > 0;
  wanted = smallest_kept(sh, wanted, limit, tid, lane, [&](auto &&count) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (E * tid + e < old) count(order_of(w[e]));
  });
  uint32_t ties = 0, all;
#pragma unroll
  for (int e = 0; e < E; ++e) ties += some && E * tid + e < old && order_of(w[e]) == limit ? 1 : 0;
  uint32_t tie = before_me(ties, sh.counts[0], lane, wave, all), bits = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int j = E * tid + e;
    const uint32_t o = order_of(w[e]);
    const bool inside = some && j < old, same = inside && o == limit;
    if ((j < n && j >= old) || (inside && o > limit) || (same && tie < wanted)) bits |= 1u << e;
    tie += same ? 1 : 0;
  }
  uint32_t at = before_me((uint32_t)__popc(bits), sh.counts[1], lane, wave, all);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if ((bits >> e & 1) != 0 && at < (uint32_t)kept) {
      chosen[at] = E * tid + e;
      out[at] = w[e];
      ++at;
    }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(kThreads) paged_evict_choose(const KhEvictParams p) {
  __shared__ Shared sh;
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
  uint32_t wanted = (uint32_t)(p.budget - p.recent), limit;
  if (n <= 4 * kThreads) return choose_held<4>(in, out, chosen, n, kept, old, wanted, sh, tid, lane, wave);
  if (n <= 8 * kThreads) return choose_held<8>(in, out, chosen, n, kept, old, wanted, sh, tid, lane, wave);
  if (n <= 16 * kThreads) return choose_held<16>(in, out, chosen, n, kept, old, wanted, sh, tid, lane, wave);

  const bool some = wanted > 0;
  wanted = smallest_kept(sh, wanted, limit, tid, lane, [&](auto &&count) {
    for (int j = tid; j < old; j += kThreads) count(order_of(in[j]));
  });
  // All weights above the limit are kept, and the first `wanted` at it.
  uint32_t to = 0, ties = 0;
  for (int64_t j0 = 0; j0 < n; j0 += kThreads) {
    const int64_t j = j0 + tid;
    const float w = j < n ? in[j] : 0.0f;
    const uint32_t o = order_of(w);
    const bool inside = some && j < old, tie = inside && o == limit;
    const uint64_t tied = __builtin_amdgcn_ballot_w64(tie);
    if (lane == 0) sh.counts[0][wave] = (uint32_t)__popcll(tied);
    __syncthreads();
    uint32_t ties_before = ties, all_ties = ties;
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) ties_before += sh.counts[0][i];
      all_ties += sh.counts[0][i];
    }
    const bool keep = (j < n && j >= old) || (inside && o > limit) || (tie && ties_before + below(tied) < wanted);
    const uint64_t kept_here = __builtin_amdgcn_ballot_w64(keep);
    if (lane == 0) sh.counts[1][wave] = (uint32_t)__popcll(kept_here);
    __syncthreads();
    uint32_t at = to;
    for (int i = 0; i < kWaves; ++i) {
      if (i < wave) at += sh.counts[1][i];
      to += sh.counts[1][i];
    }
    at += below(kept_here);
    if (keep && at < (uint32_t)kept) {
      chosen[at] = (int32_t)j;
      out[at] = w;
    }
    ties = all_ties;
  }
}

// Rows of the chosen entries, `lanes` lanes to a row (a power of two) and
// kMoveRows rows of a lane in flight. A sequence's rows are taken in the order in
// which they will lie: of all heads of an entry one after another where slots
// hold all heads, else of a head's entries.
constexpr int kMoveRows = 4;
extern "C" __global__ void __launch_bounds__(256) paged_evict_move(const KhEvictParams p) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  const int seq = (int)(blockIdx.x / (uint32_t)p.chunks), chunk = (int)(blockIdx.x - (uint32_t)seq * (uint32_t)p.chunks);
  const int n = kh_clamp(p.table.lens[seq], 0, p.table.capacity);
  const int kept = n < p.budget ? n : p.budget, heads = p.cache.kv_heads;
  const int32_t *table = p.table.pages + seq * p.table.row_stride;
  const int32_t *kept_table = p.kept_pages + seq * p.kept_row_stride;
  const int32_t *chosen = p.chosen + (int64_t)seq * heads * p.budget;
  const int piece = (int)threadIdx.x % p.lanes, first = (int)threadIdx.x / p.lanes, step = 256 / p.lanes;
  if (16 * piece >= p.cache.head_dim * p.element) return;
  const int64_t all = (int64_t)kept * heads;
  for (int64_t at = (int64_t)chunk * step * kMoveRows; at < all; at += (int64_t)p.chunks * step * kMoveRows) {
    int row[kMoveRows], head[kMoveRows], entry[kMoveRows];
    u32x4 x[kMoveRows], y[kMoveRows];
    KhSlot to[kMoveRows];
    bool real[kMoveRows];
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      const int64_t item = at + i * step + first;
      real[i] = item < all;
      const uint32_t it = real[i] ? (uint32_t)item : 0;  // below 2^31: the launcher sees to it
      if (p.heads_inner) {
        row[i] = (int)kh_div(it, p.by_heads), head[i] = (int)(it - (uint32_t)row[i] * (uint32_t)heads);
      } else {
        head[i] = (int)(it / (uint32_t)kept), row[i] = (int)(it - (uint32_t)head[i] * (uint32_t)kept);
      }
      entry[i] = chosen[(int64_t)head[i] * p.budget + row[i]];
    }
    // Rows that there are none of are read from the cache's first page.
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i) {
      KhSlot from = kh_slot(table, p.table.width, p.cache.pages, p.cache.by_page, (uint32_t)entry[i]);
      to[i] = kh_slot(kept_table, p.kept_width, p.cache.pages, p.cache.by_page, (uint32_t)row[i]);
      real[i] = real[i] && from.page >= 0 && to[i].page >= 0;
      if (from.page < 0) from = KhSlot{0, 0};
      x[i] = *reinterpret_cast<const u32x4 *>(p.cache.k + kh_row(from, p.cache.k_page, p.cache.k_slot) +
                                              (uint64_t)head[i] * p.cache.k_head + 16 * piece);
      y[i] = *reinterpret_cast<const u32x4 *>(p.cache.v + kh_row(from, p.cache.v_page, p.cache.v_slot) +
                                              (uint64_t)head[i] * p.cache.v_head + 16 * piece);
    }
#pragma unroll
    for (int i = 0; i < kMoveRows; ++i)
      if (real[i]) {
        char *k = const_cast<char *>(p.cache.k) + kh_row(to[i], p.cache.k_page, p.cache.k_slot) + (uint64_t)head[i] * p.cache.k_head;
        char *v = const_cast<char *>(p.cache.v) + kh_row(to[i], p.cache.v_page, p.cache.v_slot) + (uint64_t)head[i] * p.cache.v_head;
        __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4 *>(k + 16 * piece));
        __builtin_nontemporal_store(y[i], reinterpret_cast<u32x4 *>(v + 16 * piece));
      }
  }
}
