// The pages that a query is to attend: those whose summaries allow the largest scores.
//
// The score of a page for the heads of a KV head is the largest sum of their
// products that the page's extremes allow,
//   sum_h sum_d max(q_hd lo_d, q_hd hi_d) = sum_d (lo_d sum_h min(q_hd, 0) + hi_d sum_h max(q_hd, 0)),
// one product of length 2D a page however many heads share it. The choice is that of
// the scores in 64 bits: those of neighbouring ranks differ by far more than their
// rounding, so it does not depend on the order of sums. NaN in q counts as 0 and an
// infinity as the largest fp32 number, so every score is finite.
//
// Most pages need no 64 bits. A cluster of CTAs scores them all on the tensor cores:
// 16 summaries are the rows of an m16n8k16 MMA's A, straight from global memory (the
// order of channels within a contraction is free), three terms of the weights are
// columns of B, and a fourth column times |A| is the sum of magnitudes that bounds the
// error. The cluster's first CTA finds the border by a histogram over 2048 equal parts
// of the scores' range. Pages above the border's part by more than the error are taken,
// those below it by more are not, and the few in between are listed and ranked; where
// one of them is nearer to the last taken one than the error, in 64 bits (fp16 and bf16
// become doubles by moving bits: a half's bits, shifted, are the double's but for a power
// of two). Where more than 512 are in between (ties, scores that overflow 32 bits), all
// pages are scored in 64 bits. Equal scores go to the lowest
// page. Measured: 8192 pages for 32 heads (134 MB of summaries): 34 us, 49 in 64 bits
// alone; 2048 pages for one query: 7.5 us, bound by steps that depend on each other and
// by code that runs once.
#pragma once
#include <type_traits>

#include "kv4_rows_attention.cuh"
#include "paged.cuh"
#include "paged_mma.cuh"

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
static_assert(kSelectPages / 32 <= 2 * kSelectThreads && kSelectRanked <= kSelectThreads, "");

// Numbers whose order as unsigned integers is the numbers'; -0 becomes 0.
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k); }
// The factor that makes up for the bias (2^1008 and 2^896) would take large weights past the largest double; with this
// one every score is off by the same power of two, and neither the largest q nor the smallest overflows or vanishes.
constexpr double kWeightScale = 0x1p880;
template <typename C>
constexpr int kMantissa = std::is_same<C, __half>::value ? 10 : 7;
// A value of type C, in bits 16 to 31 of h, times a power of two.
template <typename C>
__device__ __forceinline__ double widened(uint32_t h) {
  // C's sign, exponent and mantissa as a double's, the exponent's bias left as it is
  return __hiloint2double((int)((h & 0x80000000u) | (h & 0x7FFF0000u) >> (kMantissa<C> - 4)), 0);
}
// A score of terms whose magnitudes add up to S is off by at most S times this: 16 MMAs, each off by at most 2^-22 of what
// it has summed (its 17 terms are aligned to the largest and cut), the weights' third terms and the last sums of three.
constexpr float kScoreError = 0x1p-17f;
// What the weights' magnitudes are raised by: with it, S covers what is left of a weight after three terms (2^-25 where
// the largest weight is 2^14 or more).
constexpr float kScoreLeast = 0x1p-6f;

struct Words {
  uint32_t w[8];
};
__device__ __forceinline__ Words load32(const void *p) {
  Words x;
  asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3]), "=r"(x.w[4]), "=r"(x.w[5]), "=r"(x.w[6]), "=r"(x.w[7])
      : "l"(p));
  return x;
}

template <int D, typename T, typename C>
__global__ void __launch_bounds__(kSelectThreads, 1) paged_select_kernel(const PagedSelectParams p) {
  constexpr int kSteps = 2 * D / 16;
  extern __shared__ __align__(16) uint32_t select_smem[];   // 8 bytes a candidate
  uint32_t *keys = select_smem;                             // scores in 32 bits, of the first CTA
  __shared__ __align__(16) double weights[2][D];            // of the smallest, of the largest
  __shared__ __align__(8) uint32_t frag[kSteps][32][2];     // B fragments: three terms and the magnitudes, columns of 0
  __shared__ __align__(16) uint32_t bins[kSelectBins];
  __shared__ uint32_t taken[kSelectPages / 32], same[kSelectPages / 32];   // a bit a key
  __shared__ unsigned long long reach[8 * kSelectWarps], size[8 * kSelectWarps];   // of the cluster's warps: keys, magnitudes
  __shared__ unsigned long long list_keys[kSelectRanked];
  __shared__ uint32_t list_at[kSelectRanked];
  __shared__ uint32_t w_sum[kSelectWarps];
  __shared__ uint32_t found_bin, found_above, found_count, listed, top_weight, border;
  const PagedTable &t = p.c.t;
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t ctas = cluster_size(), rank = cluster_rank(), item = blockIdx.x / ctas;
  const uint32_t query = item / p.c.kv_heads, head = item - query * p.c.kv_heads;
  if (tid == 0) top_weight = 0;
  __syncthreads();
  cluster_arrive();   // waited for where the first CTA's shared memory is first written
  pdl_launch_dependents();
  pdl_wait();
  // ---- weights ----
  if (tid < D) {
    const T *q = (const T *)p.q + (int64_t)query * p.q_query + (int64_t)head * p.group * p.q_head + tid;
    double up = 0, down = 0;
#pragma unroll 8
    for (uint32_t h = 0; h < p.group; ++h) {
      float x = (float)q[(int64_t)h * p.q_head];
      x = x != x ? 0.f : fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
      up += x > 0 ? x : 0.f, down += x > 0 ? 0.f : x;
    }
    weights[0][tid] = down, weights[1][tid] = up;
    const float most = fmaxf((float)up, (float)-down);   // infinity: scores in 64 bits alone
    const uint32_t top = __reduce_max_sync(~0u, __float_as_uint(most));
    if (lane == 0) atomicMax(&top_weight, top);
  }
  const PagedSeen who = paged_seen(t, p.which, query);
  const uint32_t count = (who.seen + t.page_rows() - 1) >> t.shift;
  int32_t *out = p.chosen + (size_t)item * p.budget;
  if (count <= p.budget) {   // all of them; the whole cluster leaves
    cluster_wait();
    if (rank == 0)
      for (uint32_t i = tid; i < p.budget; i += kSelectThreads) out[i] = i < count ? (int32_t)i : -1;
    return;
  }
  const uint32_t n = count - p.sinks - p.recent, want = p.budget - p.sinks - p.recent;   // candidates: more than wanted
  if (want == 0) {   // likewise
    cluster_wait();
    if (rank == 0) {
      for (uint32_t i = tid; i < p.sinks; i += kSelectThreads) out[i] = (int32_t)i;
      for (uint32_t i = tid; i < p.recent; i += kSelectThreads) out[p.sinks + i] = (int32_t)(count - p.recent + i);
    }
    return;
  }
  // the first pages that this warp scores, asked for early
  const int32_t *table = t.table + (size_t)who.seq * t.seq_pages + p.sinks;
  const uint32_t stride = ctas * kSelectWarps * 16;
  const auto pages_at = [&](uint32_t base) { return lane < 16 && base + lane < n ? (uint32_t)table[base + lane] : ~0u; };
  uint32_t base = (rank * kSelectWarps + warp) * 16, ahead = pages_at(base);
  __syncthreads();
  float inverse;
  const float power = row_power(__uint_as_float(top_weight), inverse);   // brings the largest weight to [2^14, 2^15)
  if (tid < D) {   // two weights a thread: channels c and c + 1 of the summary
    const uint32_t c = 2 * tid, in = c % 64 / 16, at = c / 64 * 4 + c % 16 / 4;
    const double *w = (const double *)weights + c;
    float x = (float)(w[0] * power), y = (float)(w[1] * power);
    const float ax = fabsf(x) + kScoreLeast, ay = fabsf(y) + kScoreLeast;
#pragma unroll
    for (int k = 0; k < 3; ++k) frag[at][k * 4 + in][c % 4 / 2] = take_pair(x, y, C{});
    float bx = ax * (1.f + 0x1p-6f), by = ay * (1.f + 0x1p-6f);   // rounded, they are no smaller than before
    frag[at][12 + in][c % 4 / 2] = take_pair(bx, by, C{});
#pragma unroll
    for (int k = 4; k < 8; ++k) frag[at][k * 4 + in][c % 4 / 2] = 0;
  }
  __syncthreads();
  // ---- scores in 32 bits: 16 pages a warp ----
  const uint32_t g = lane / 4, t4 = lane % 4;
  {
    const uint32_t there = remote_smem(keys, 0);
    uint32_t low = ~0u, high = 0, most = 0;
    cluster_wait();   // the CTA that the keys go to has started
    for (; base < n; base += stride) {
      const uint32_t page = ahead;
      ahead = pages_at(base + stride);
      Words x[2][D / 32];   // a lane has 32 of a row's 128 bytes: with less, L2 moves lines twice
      uint32_t pg[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        pg[y] = __shfl_sync(~0u, page, g + 8 * y);
        const C *src = (const C *)p.c.summaries + ((size_t)(pg[y] < t.pages ? pg[y] : 0) * p.c.kv_heads + head) * 2 * D + 16 * t4;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) x[y][j] = load32(src + 64 * j);
      }
      float c[4] = {}, d[4] = {};
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const Words &x0 = x[0][k / 4], &x1 = x[1][k / 4];
        const uint32_t w[4] = {x0.w[k % 4 * 2], x1.w[k % 4 * 2], x0.w[k % 4 * 2 + 1], x1.w[k % 4 * 2 + 1]};
        const uint32_t m[4] = {w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu, w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu};
        const uint2 b = *(const uint2 *)frag[k][lane];
        const uint32_t bb[2] = {b.x, b.y};
        mma_16(c, w, bb, C{});
        mma_16(d, m, bb, C{});
      }
      // columns 0 and 1 are lane t4 = 0's, 2 and 3 lane t4 = 1's
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const float third = __shfl_down_sync(~0u, c[2 * y], 1);
        const uint32_t i = base + 8 * y + g;
        if (i < n && t4 == 0) {
          const uint32_t k = ordered(pg[y] < t.pages ? c[2 * y] + (c[2 * y + 1] + third) : 0.f);
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + i * 4), "r"(k) : "memory");
          low = min(low, k), high = max(high, k);
        }
        if (i < n && t4 == 1) most = max(most, __float_as_uint(d[2 * y + 1]) & 0x7FFFFFFFu);
      }
    }
    low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high), most = __reduce_max_sync(~0u, most);
    if (lane == 0) {
      st_remote(remote_smem(&reach[rank * kSelectWarps + warp], 0), (uint64_t)high << 32 | low);
      st_remote(remote_smem(&size[rank * kSelectWarps + warp], 0), most);
    }
  }
  cluster_sync();
  if (rank) return;
  uint32_t low = ~0u, high = 0, most = 0;
  for (uint32_t i = lane; i < ctas * kSelectWarps; i += 32) {
    low = min(low, (uint32_t)reach[i]), high = max(high, (uint32_t)(reach[i] >> 32));
    most = max(most, (uint32_t)size[i]);
  }
  low = __reduce_min_sync(~0u, low), high = __reduce_max_sync(~0u, high);
  const float error = __uint_as_float(__reduce_max_sync(~0u, most)) * kScoreError;
  if (tid == 0) listed = 0;

  // The part of [low, high], one of up to 2048, in which the left-th key from the top lies: [low, high] becomes the part's
  // range, `left` loses the keys above it; how many keys the part has.
  const auto narrow = [&](auto &low, auto &high, uint32_t &left, int shift, auto key) {
    *(uint4 *)(bins + 4 * tid) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    for (uint32_t i = tid; i < n; i += kSelectThreads) {
      const auto k = key(i);
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
    using K = typename std::remove_reference<decltype(low)>::type;
    low += (K)found_bin << shift;
    left -= found_above;
    const K end = low + (((K)1 << shift) - 1);
    high = end < high ? end : high;
    return found_count;
  };
  // Marks the keys above `to` in `taken`, and lists (or, without a list, marks in `same`) those from `from` to `to`.
  const auto part = [&](auto from, auto to, bool list, auto key) {
    for (uint32_t i = tid; i < (n + 31) / 32 * 32; i += kSelectThreads) {
      const auto k = i < n ? key(i) : 0;
      const bool in = i < n && k >= from && k <= to;
      const uint32_t more = __ballot_sync(~0u, i < n && k > to), marked = __ballot_sync(~0u, in);
      if (lane == 0) taken[i / 32] = more, same[i / 32] = list ? 0 : marked;
      if (list && in) {
        const uint32_t at = atomicAdd(&listed, 1u);
        if (at < kSelectRanked) list_at[at] = i, list_keys[at] = k;
      }
    }
    __syncthreads();
  };
  const auto sums_before = [&](uint32_t mine, uint32_t &all) {   // of the threads before this one
    uint32_t sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    __syncthreads();
    if (lane == 31) w_sum[warp] = sum;
    __syncthreads();
    const uint32_t each = lane < kSelectWarps ? w_sum[lane] : 0;
    all = __reduce_add_sync(~0u, each);
    return sum + __reduce_add_sync(~0u, lane < warp ? each : 0) - mine;
  };

  // ---- the border in 32 bits, and the keys within twice the error of it ----
  bool exact = !(error < 0x1p100f);   // a score or its error overflows
  uint32_t left = want;
  if (!exact) {
    const auto key = [&](uint32_t i) { return keys[i]; };
    for (;;) {
      const int shift = max(32 - __clz(high - low) - 11, 0);
      const uint32_t in = narrow(low, high, left, shift, key);
      if (in <= kSelectRanked / 4 || shift == 0) break;
    }
    const uint32_t from = ordered(__fsub_rd(unordered(low), 2 * error)), to = ordered(__fadd_ru(unordered(high), 2 * error));
    part(from, to, true, key);
    exact = listed > kSelectRanked;
  }
  // Scores in 64 bits, of `count` pages, listed or the first: a warp takes 8 pages at a time, a lane 16 bytes of a summary.
  const auto score = [&](uint32_t count, const uint32_t *list, unsigned long long *dst) {
    __syncthreads();
    constexpr uint32_t L = 2 * D / 8, kPer = 32 / L;   // lanes of a summary, summaries of a warp's load
    constexpr uint32_t kBatch = 8, step = kBatch * kPer;
    const uint32_t piece = lane % L, sub = lane / L;
    for (uint32_t from = warp * step; from < count; from += kSelectWarps * step) {
      uint32_t page = ~0u;
      if (lane < step && from + lane < count) page = (uint32_t)table[list ? list[from + lane] : from + lane];
      double s[kBatch];
#pragma unroll
      for (uint32_t i = 0; i < kBatch; ++i) {
        const uint32_t pg = __shfl_sync(~0u, page, i * kPer + sub);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (pg < t.pages) x = __ldg((const uint4 *)((const C *)p.c.summaries + ((size_t)pg * p.c.kv_heads + head) * 2 * D) + piece);
        const uint32_t y[4] = {x.x, x.y, x.z, x.w};
        s[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const double2 w = *(const double2 *)((const double *)weights + piece * 8 + 2 * j);
          s[i] = fma(widened<C>(y[j] << 16), w.x * kWeightScale, s[i]);
          s[i] = fma(widened<C>(y[j]), w.y * kWeightScale, s[i]);
        }
      }
      // 8 sums over the L lanes: every exchange halves the sums that a lane still carries
#pragma unroll
      for (uint32_t o = 1, m = 4; o < 8; o <<= 1, m >>= 1) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          if (i >= m) continue;
          const bool up = lane & o;
          const double give = up ? s[i] : s[i + m], keep = up ? s[i + m] : s[i];
          s[i] = keep + __shfl_xor_sync(~0u, give, o);
        }
      }
#pragma unroll
      for (uint32_t o = 8; o < L; o <<= 1) s[0] += __shfl_xor_sync(~0u, s[0], o);
      // this lane's sum is of batch (lane & 1) * 4 + (lane & 2) + (lane & 4) / 4
      const uint32_t i = from + ((lane & 1) * 4 + (lane & 2) + (lane & 4) / 4) * kPer + sub;
      if (piece < 8 && i < count) dst[i] = ordered(s[0]);
    }
    __syncthreads();
  };
  // ---- without a list: the border in 64 bits ----
  if (exact) {
    unsigned long long *all_keys = (unsigned long long *)select_smem;
    score(n, nullptr, all_keys);
    const auto key = [&](uint32_t i) { return all_keys[i]; };
    unsigned long long from = 0, to = ~0ull;
    left = want;
    for (;;) {
      const int shift = max(64 - __clzll((long long)(to - from)) - 11, 0);
      const uint32_t in = narrow(from, to, left, shift, key);
      if (in <= kSelectRanked || shift == 0) break;
    }
    if (tid == 0) listed = 0;
    __syncthreads();
    part(from, to, found_count <= kSelectRanked, key);
  }
  const uint32_t listed_now = listed;
  // ---- how many of the listed or marked ones are taken ----
  const uint32_t words = (n + 31) / 32;   // two a thread
  uint32_t two[2], all;
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) two[i] = 2 * tid + i < words ? taken[2 * tid + i] : 0;
  sums_before(__popc(two[0]) + __popc(two[1]), all);
  left = want - all;
  // the listed ones are ranked by their scores in 32 bits; where one is nearer to the border than twice the error, in 64
  uint32_t before = 0;
  for (bool sure = exact;; sure = true) {
    const unsigned long long k = tid < listed_now ? list_keys[tid] : 0;
    const uint32_t at = tid < listed_now ? list_at[tid] : 0;
    before = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < listed_now; ++i) before += list_keys[i] > k || (list_keys[i] == k && list_at[i] < at);
    if (sure) break;
    const bool is_border = tid < listed_now && before == left - 1;
    if (is_border) border = (uint32_t)k;
    __syncthreads();
    const float away = fabsf(unordered((uint32_t)k) - unordered(border));
    if (!__syncthreads_or(tid < listed_now && !is_border && away <= 2.001f * error)) break;
    score(listed_now, list_at, list_keys);
  }
  if (tid < listed_now && before < left) atomicOr(&taken[list_at[tid] / 32], 1u << list_at[tid] % 32);
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) two[i] = 2 * tid + i < words ? taken[2 * tid + i] : 0;
  if (listed_now == 0) {   // the first `left` of the marked ones
    uint32_t marked[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) marked[i] = 2 * tid + i < words ? same[2 * tid + i] : 0;
    uint32_t before = sums_before(__popc(marked[0]) + __popc(marked[1]), all);
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
  // ---- the chosen ones in order ----
  uint32_t at = sums_before(__popc(two[0]) + __popc(two[1]), all);
#pragma unroll
  for (uint32_t i = 0; i < 2; ++i) {
    for (uint32_t w = two[i]; w; w &= w - 1) out[p.sinks + at++] = (int32_t)(p.sinks + (2 * tid + i) * 32 + __ffs(w) - 1);
  }
  for (uint32_t i = tid; i < p.sinks; i += kSelectThreads) out[i] = (int32_t)i;
  for (uint32_t i = tid; i < p.recent; i += kSelectThreads) out[p.sinks + want + i] = (int32_t)(count - p.recent + i);
}

}  // namespace vg
