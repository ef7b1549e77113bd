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
// the weights. The pick narrows a range of keys (scores as ordered integers): a
// histogram of 2048 equal parts, then the part that the last chosen key lies in,
// until its keys are all taken or all equal; two or three rounds unless scores
// crowd together. Equal keys go to the lowest page.
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
constexpr uint32_t kSelectChunks = kSelectPages / kSelectThreads;

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
__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const PagedSelectParams p) {
  extern __shared__ __align__(16) uint64_t keys[];   // [candidates], of the first CTA
  __shared__ __align__(16) double weights[2][D];     // of the smallest, of the largest
  __shared__ uint32_t bins[kSelectBins];
  __shared__ uint32_t counts[kSelectChunks * kSelectWarps];   // greater | equal << 16 of 32 keys
  __shared__ uint64_t w_low[kSelectWarps], w_high[kSelectWarps];
  __shared__ uint32_t w_sum[kSelectWarps];
  __shared__ uint32_t found_bin, found_above, found_count;
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
    const uint32_t step = kBatch * kPer;
    const uint32_t there = remote_smem(keys, 0);
    for (uint32_t base = (rank * kSelectWarps + warp) * step; base < n; base += ctas * kSelectWarps * step) {
      const uint32_t mine = base + lane;
      const uint32_t page = lane < step && mine < n ? (uint32_t)table[mine] : ~0u;
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
      if (part < 8 && i < n) st_remote(there + i * 8, ordered(s[0]));
    }
  }
  cluster_sync();
  if (rank) return;
  // ---- the range of the keys ----
  uint64_t low = ~0ull, high = 0;
  const auto widen = [&](uint64_t a, uint64_t b) { low = a < low ? a : low, high = b > high ? b : high; };
  for (uint32_t i = tid; i < n; i += kSelectThreads) widen(keys[i], keys[i]);
#pragma unroll
  for (int o = 16; o; o >>= 1) widen(__shfl_xor_sync(~0u, low, o), __shfl_xor_sync(~0u, high, o));
  if (lane == 0) w_low[warp] = low, w_high[warp] = high;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kSelectWarps; ++i) widen(w_low[i], w_high[i]);
  // ---- keys from `low` on are taken, but for `equal` == true: of those equal to it only the first `left` ----
  uint32_t left = want;   // of the keys in [low, high]; want < n, so some are left out
  bool equal = false;
  for (;;) {
    const uint64_t span = high - low;
    const int bits = 64 - __clzll((long long)span), shift = span ? max(bits - 11, 0) : 0;
    for (uint32_t i = tid; i < kSelectBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kSelectThreads) {
      const uint64_t k = keys[i];
      if (k >= low && k <= high) atomicAdd(&bins[(uint32_t)((k - low) >> shift)], 1u);
    }
    __syncthreads();
    // from the top: the bin in which the `left`-th key lies; a thread has 4 bins
    constexpr uint32_t kEach = kSelectBins / kSelectThreads;
    uint32_t b[kEach], mine = 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) b[i] = bins[kSelectBins - 1 - (tid * kEach + i)], mine += b[i];
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    if (lane == 31) w_sum[warp] = sum;
    __syncthreads();
    uint32_t above = sum - mine;
#pragma unroll
    for (uint32_t i = 0; i < kSelectWarps; ++i) above += i < warp ? w_sum[i] : 0;
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
      if (above < left && above + b[i] >= left)
        found_bin = kSelectBins - 1 - (tid * kEach + i), found_above = above, found_count = b[i];
      above += b[i];
    }
    __syncthreads();
    low += (uint64_t)found_bin << shift;
    left -= found_above;
    if (found_count == left) break;      // all of this part
    if (shift == 0) {                    // one key, met more often than it is wanted
      equal = true;
      break;
    }
    const uint64_t end = low + ((1ull << shift) - 1);
    high = end < high ? end : high;
  }
  // ---- the chosen ones in order ----
  const uint32_t chunks = (n + kSelectThreads - 1) / kSelectThreads;
  for (uint32_t c = 0; c < chunks; ++c) {
    const uint32_t i = c * kSelectThreads + tid;
    const uint64_t k = i < n ? keys[i] : 0;   // 0 is below every key
    const uint32_t more = __ballot_sync(~0u, equal ? k > low : k >= low), same = __ballot_sync(~0u, equal && k == low);
    if (lane == 0) counts[c * kSelectWarps + warp] = __popc(more) | __popc(same) << 16;
  }
  __syncthreads();
  // sums before each 32 keys: up to 24576 greater ones and as many equal ones, in 16 bits each
  if (warp == 0) {
    uint32_t before = 0;
    for (uint32_t base = 0; base < chunks * kSelectWarps; base += 32) {
      const uint32_t i = base + lane, x = i < chunks * kSelectWarps ? counts[i] : 0;
      uint32_t sum = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, sum, o);
        if (lane >= (uint32_t)o) sum += up;
      }
      if (i < chunks * kSelectWarps) counts[i] = before + sum - x;
      before += __shfl_sync(~0u, sum, 31);
    }
  }
  __syncthreads();
  for (uint32_t c = 0; c < chunks; ++c) {
    const uint32_t i = c * kSelectThreads + tid;
    const uint64_t k = i < n ? keys[i] : 0;
    const bool is_more = equal ? k > low : k >= low, is_same = equal && k == low;
    const uint32_t more = __ballot_sync(~0u, is_more), same = __ballot_sync(~0u, is_same), below = (1u << lane) - 1;
    const uint32_t before = counts[c * kSelectWarps + warp];
    const uint32_t a = (before & 0xFFFF) + __popc(more & below), e = (before >> 16) + __popc(same & below);
    if (is_more || (is_same && e < left)) out[p.sinks + a + min(e, equal ? left : 0u)] = (int32_t)(p.sinks + i);
  }
  for (uint32_t i = tid; i < p.sinks; i += kSelectThreads) out[i] = (int32_t)i;
  for (uint32_t i = tid; i < p.recent; i += kSelectThreads) out[p.sinks + want + i] = (int32_t)(count - p.recent + i);
}

}  // namespace vg
