// The pages that a query is to attend: those whose summaries allow the largest scores.
//
// The score of a page for the heads of a KV head is the largest sum of their
// products that the page's extremes allow,
//   sum_h sum_d max(q_hd lo_d, q_hd hi_d) = sum_d (lo_d sum_h min(q_hd, 0) + hi_d sum_h max(q_hd, 0)),
// one product of length 2D a page however many heads share it. It is summed in 64
// bits: scores of neighbouring ranks differ by far more than its rounding, so the
// choice does not depend on the order of the sums. NaN in q counts as 0 and an
// infinity as the largest fp32 number, so every score is finite.
//
// A cluster of CTAs scores the pages of a (query, KV head); its first CTA then picks
// from their scores in its shared memory. fp16 and bf16 become doubles by moving
// bits: a half's bits, shifted, are the double's but for a power of two, which is in
// the weights. The pick: a histogram of the keys (scores as ordered integers) over
// 2048 equal parts of their range finds the part that the last chosen key lies in; the
// few keys of that part are ranked against each other. Where it has more than 512, it
// is the next range. Equal keys go to the lowest page.
#pragma once
#include <type_traits>

#include "kv4_rows.cuh"
#include "paged.cuh"

namespace vg {

struct PagedSelectParams {
  PagedView c;
  const void *q;
  int64_t q_query, q_head;   // strides
  PagedQueries which;
  int32_t *chosen;           // [queries][kv_heads][budget]
  uint32_t group, budget, sinks, recent;
};

constexpr uint32_t kSelectThreads = 512;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kSelectBins = 2048;
constexpr uint32_t kSelectPages = 24576;   // keys that the first CTA has room for
constexpr uint32_t kSelectRanked = 512;    // keys that are ranked against each other
static_assert(kSelectRanked * 12 <= kSelectBins * 4 && kSelectPages / 32 <= 2 * kSelectThreads, "");

// Doubles whose order as unsigned integers is the numbers'.
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);   // -0 becomes 0
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// A value of type C, in bits 16 to 31 of h, times a power of two.
template <typename C>
constexpr int kMantissa = std::is_same<C, __half>::value ? 10 : 7;
// The factor that makes up for the bias (2^1008 and 2^896) would take large weights past the largest double; with this
// one every score is off by the same power of two, and neither the largest q nor the smallest overflows or vanishes.
constexpr double kWeightScale = 0x1p880;
template <typename C>
__device__ __forceinline__ double widened(uint32_t h) {
  // C's sign, exponent and mantissa as a double's, the exponent's bias left as it is
  return __hiloint2double((int)((h & 0x80000000u) | (h & 0x7FFF0000u) >> (kMantissa<C> - 4)), 0);
}

template <int D, typename T, typename C>
__global__ void __launch_bounds__(kSelectThreads, 2) paged_select_kernel(const PagedSelectParams p) {
  extern __shared__ __align__(16) uint64_t keys[];   // [candidates], of the first CTA
  __shared__ __align__(16) double weights[2][D];     // of the smallest, of the largest
  __shared__ __align__(16) uint32_t bins[kSelectBins];
  __shared__ uint32_t taken[kSelectPages / 32], same[kSelectPages / 32];   // a bit a key
  __shared__ unsigned long long reach[8 * kSelectWarps];   // upper halves of the greatest and the least key of the cluster's warps
  __shared__ uint32_t w_sum[kSelectWarps];
  __shared__ uint32_t found_bin, found_above, found_count, listed;
  const PagedTable &t = p.c.t;
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t ctas = cluster_size(), rank = cluster_rank(), item = blockIdx.x / ctas;
  const uint32_t query = item / p.c.kv_heads, head = item - query * p.c.kv_heads;
  pdl_launch_dependents();
  pdl_wait();
  const PagedSeen who = paged_seen(t, p.which, query);
  const uint32_t count = (who.seen + t.page_rows() - 1) >> t.shift;
  int32_t *out = p.chosen + (size_t)item * p.budget;
  if (count <= p.budget) {   // all of them; the whole cluster leaves
    if (rank == 0)
      for (uint32_t i = tid; i < p.budget; i += kSelectThreads) out[i] = i < count ? (int32_t)i : -1;
    return;
  }
  const uint32_t n = count - p.sinks - p.recent, want = p.budget - p.sinks - p.recent;   // candidates: more than wanted
  if (want == 0) {   // likewise
    if (rank == 0) {
      for (uint32_t i = tid; i < p.sinks; i += kSelectThreads) out[i] = (int32_t)i;
      for (uint32_t i = tid; i < p.recent; i += kSelectThreads) out[p.sinks + i] = (int32_t)(count - p.recent + i);
    }
    return;
  }
  // ---- weights ----
  for (uint32_t d = tid; d < D; d += kSelectThreads) {
    const T *q = (const T *)p.q + (int64_t)query * p.q_query + (int64_t)head * p.group * p.q_head + d;
    double up = 0, down = 0;
    for (uint32_t h = 0; h < p.group; ++h) {
      float x = (float)q[(int64_t)h * p.q_head];
      x = x != x ? 0.f : fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
      if (x > 0) up += x;
      else down += x;
    }
    weights[0][d] = down * kWeightScale, weights[1][d] = up * kWeightScale;
  }
  cluster_sync();   // the weights are there, and so is the CTA that the keys go to
  // ---- scores: a warp takes 8 pages at a time, a lane 16 bytes of a summary ----
  {
    constexpr uint32_t L = 2 * D / 8, kPer = 32 / L;   // lanes of a summary, summaries of a warp's load
    constexpr uint32_t kBatch = 8;                     // loads in flight
    const uint32_t part = lane % L, sub = lane / L;
    double w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = ((const double *)weights)[part * 8 + i];
    const int32_t *table = t.table + (size_t)who.seq * t.seq_pages + p.sinks;
    const uint32_t step = kBatch * kPer, stride = ctas * kSelectWarps * step;
    const uint32_t there = remote_smem(keys, 0);
    uint32_t low = ~0u, high = 0;   // upper halves of the least and the greatest key
    const auto pages_at = [&](uint32_t base) {
      return lane < step && base + lane < n ? (uint32_t)table[base + lane] : ~0u;
    };
    uint32_t base = (rank * kSelectWarps + warp) * step, ahead = pages_at(base);
    for (; base < n; base += stride) {
      const uint32_t page = ahead;
      ahead = pages_at(base + stride);
      uint4 x[kBatch];
#pragma unroll
      for (uint32_t i = 0; i < kBatch; ++i) {
        const uint32_t pg = __shfl_sync(~0u, page, i * kPer + sub);
        x[i] = make_uint4(0, 0, 0, 0);
        if (pg < t.pages) x[i] = __ldg((const uint4 *)((const C *)p.c.summaries + ((size_t)pg * p.c.kv_heads + head) * 2 * D) + part);
      }
      double s[kBatch];
#pragma unroll
      for (uint32_t i = 0; i < kBatch; ++i) {
        const uint32_t y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        double a = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          a = fma(widened<C>(y[j] << 16), w[2 * j], a);
          a = fma(widened<C>(y[j]), w[2 * j + 1], a);
        }
        s[i] = a;
      }
      // 8 sums over the L lanes: every exchange halves the sums that a lane still carries
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const bool up = lane & 1;
        const double give = up ? s[i] : s[i + 4], keep = up ? s[i + 4] : s[i];
        s[i] = keep + __shfl_xor_sync(~0u, give, 1);
      }
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) {
        const bool up = lane & 2;
        const double give = up ? s[i] : s[i + 2], keep = up ? s[i + 2] : s[i];
        s[i] = keep + __shfl_xor_sync(~0u, give, 2);
      }
      {
        const bool up = lane & 4;
        const double give = up ? s[0] : s[1], keep = up ? s[1] : s[0];
        s[0] = keep + __shfl_xor_sync(~0u, give, 4);
      }
#pragma unroll
      for (uint32_t o = 8; o < L; o <<= 1) s[0] += __shfl_xor_sync(~0u, s[0], o);
      // this lane's sum is of batch (lane & 1) * 4 + (lane & 2) + (lane & 4) / 4
      const uint32_t i = base + ((lane & 1) * 4 + (lane & 2) + (lane & 4) / 4) * kPer + sub;
      if (part < 8 && i < n) {
        const unsigned long long k = ordered(s[0]);
        st_remote(there + i * 8, k);
        low = min(low, (uint32_t)(k >> 32)), high = max(high, (uint32_t)(k >> 32));
      }
    }
    low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high);
    if (lane == 0) st_remote(remote_smem(&reach[rank * kSelectWarps + warp], 0), (uint64_t)high << 32 | low);
  }
  cluster_sync();
  if (rank) return;
  // ---- the part of the range that the last chosen key lies in ----
  uint32_t low_half = ~0u, high_half = 0;
  for (uint32_t i = lane; i < ctas * kSelectWarps; i += 32) {
    low_half = min(low_half, (uint32_t)reach[i]);
    high_half = max(high_half, (uint32_t)(reach[i] >> 32));
  }
  unsigned long long low = (unsigned long long)__reduce_min_sync(~0u, low_half) << 32;
  unsigned long long high = (unsigned long long)__reduce_max_sync(~0u, high_half) << 32 | 0xFFFFFFFFu;
  uint32_t left = want;   // of the keys in [low, high]; want < n, so some are left out
  uint32_t count_in;
  for (;;) {
    const unsigned long long span = high - low;
    const int bits = 64 - __clzll((long long)span), shift = max(bits - 11, 0);
    *(uint4 *)(bins + 4 * tid) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kSelectThreads) {
      const unsigned long long k = keys[i];
      if (k >= low && k <= high) atomicAdd(&bins[(uint32_t)((k - low) >> shift)], 1u);
    }
    __syncthreads();
    // from the top, four parts a thread
    const uint4 four = *(const uint4 *)(bins + kSelectBins - 4 - 4 * tid);
    const uint32_t b[4] = {four.w, four.z, four.y, four.x}, mine = b[0] + b[1] + b[2] + b[3];
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    if (lane == 31) w_sum[warp] = sum;
    __syncthreads();
    const uint32_t others = lane < warp ? w_sum[lane] : 0;   // 16 warps
    uint32_t above = sum - mine + __reduce_add_sync(~0u, others);
    if (above < left && above + mine >= left) {
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        if (above < left && above + b[i] >= left)
          found_bin = kSelectBins - 1 - (4 * tid + i), found_above = above, found_count = b[i];
        above += b[i];
      }
    }
    __syncthreads();
    low += (unsigned long long)found_bin << shift;
    left -= found_above;
    count_in = found_count;
    const unsigned long long end = low + ((1ull << shift) - 1);
    high = end < high ? end : high;
    if (count_in <= kSelectRanked || shift == 0) break;
  }
  // ---- keys past the part are taken; those in it are listed, or marked where all are equal or all are taken ----
  const bool rank_them = count_in > left && count_in <= kSelectRanked;
  unsigned long long *list_keys = (unsigned long long *)bins;
  uint32_t *list_at = bins + 2 * kSelectRanked;
  if (tid == 0) listed = 0;
  __syncthreads();
  for (uint32_t i = tid; i < (n + 31) / 32 * 32; i += kSelectThreads) {
    const unsigned long long k = i < n ? keys[i] : 0;   // 0 is below every key
    const bool in = k >= low && k <= high;
    const uint32_t more = __ballot_sync(~0u, k > high), equal = __ballot_sync(~0u, in);
    if (lane == 0) taken[i / 32] = more, same[i / 32] = rank_them ? 0 : equal;
    if (rank_them && in) {
      const uint32_t at = atomicAdd(&listed, 1u);
      list_keys[at] = k, list_at[at] = i;
    }
  }
  __syncthreads();
  if (rank_them && tid < count_in) {
    const unsigned long long k = list_keys[tid];
    const uint32_t at = list_at[tid];
    uint32_t before = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < count_in; ++i) before += list_keys[i] > k || (list_keys[i] == k && list_at[i] < at);
    if (before < left) atomicOr(&taken[at / 32], 1u << at % 32);
  }
  __syncthreads();
  // ---- the chosen ones in order: a thread has the keys of two words ----
  const uint32_t words = (n + 31) / 32;
  const auto sums_before32 = [&](uint32_t mine) {   // of the threads before this one
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    if (lane == 31) w_sum[warp] = sum;
    __syncthreads();
    const uint32_t others = lane < warp ? w_sum[lane] : 0;
    sum += __reduce_add_sync(~0u, others) - mine;
    __syncthreads();
    return sum;
  };
  uint32_t two[2];
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) two[i] = 2 * tid + i < words ? taken[2 * tid + i] : 0;
  if (!rank_them) {   // the first `left` of the marked ones
    uint32_t marked[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) marked[i] = 2 * tid + i < words ? same[2 * tid + i] : 0;
    uint32_t before = sums_before32(__popc(marked[0]) + __popc(marked[1]));
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      for (; marked[i] && before < left; ++before) {
        const uint32_t bit = marked[i] & -marked[i];
        two[i] |= bit;
        marked[i] ^= bit;
      }
      before += __popc(marked[i]);
    }
  }
  uint32_t at = sums_before32(__popc(two[0]) + __popc(two[1]));
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    for (uint32_t w = two[i]; w; w &= w - 1) out[p.sinks + at++] = (int32_t)(p.sinks + (2 * tid + i) * 32 + __ffs(w) - 1);
  }
  for (uint32_t i = tid; i < p.sinks; i += kSelectThreads) out[i] = (int32_t)i;
  for (uint32_t i = tid; i < p.recent; i += kSelectThreads) out[p.sinks + want + i] = (int32_t)(count - p.recent + i);
}

}  // namespace vg
