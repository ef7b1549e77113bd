// Verification of drafted tokens against a model's probabilities.
#pragma once
#include <cooperative_groups.h>

#include <cstdint>

namespace vg {

struct VerifyParams {
  const int32_t *tokens;       // [seqs][drafted]
  const float *draft;          // [seqs][drafted][vocab]
  const float *target;         // [seqs][drafted + 1][vocab]
  const float *u_accept;       // [seqs][drafted]
  const float *u_sample;       // [seqs]
  const int32_t *counts;       // drafted tokens of each sequence, may be null
  int32_t *accepted, *next;    // [seqs]
  uint32_t drafted, vocab;
};

// A probability as a multiple of 2^-38. Sums of these are exact, so a total and
// a cumulative sum do not depend on the order they are taken in, and a sampled
// token does not depend on the launch shape. NaN and negative values count as
// 0, values above 1 as 1.
__device__ __forceinline__ uint64_t fixed_probability(float x) {
  return (uint64_t)(fminf(fmaxf(x, 0.f), 1.f) * 0x1p38f);
}

constexpr uint32_t kVerifyThreads = 1024;
constexpr uint32_t kVerifyCtas = 8;             // of a cluster: one sequence
constexpr uint32_t kVerifyVocab = 1u << 20;     // largest vocabulary
constexpr uint32_t kVerifyWarps = kVerifyThreads / 32;

// Sum over a warp of values up to 2^40 (four probabilities a lane), by integer reductions of the low 19 bits and of the 21
// above them: 32 of either stay below 2^32.
__device__ __forceinline__ uint64_t warp_sum(uint64_t x) {
  const uint32_t low = __reduce_add_sync(~0u, (uint32_t)x & 0x7FFFFu), high = __reduce_add_sync(~0u, (uint32_t)(x >> 19));
  return low + ((uint64_t)high << 19);
}

// Token t is accepted while u_t * q(x_t) < p(x_t); the first token that is not
// ends the run, and the next token is drawn from max(p - q, 0) there, or from p
// after the last drafted token (or where p <= q everywhere).
//
// Bound by the latency of three dependent reads: the tokens, their two
// probabilities, one row of each distribution. A cluster of 8 CTAs takes a
// sequence, so that one stream's row of 73448 probabilities is read by 8 SMs at
// once, each its own stretch; the stretches' exact sums meet through
// distributed shared memory, and the CTA whose stretch holds the drawn point
// finds it from the sums that its warps left, reading 32 or 128 values again. Four
// tokens of one stream at a vocabulary of 73448: 7.1 us (90 us with one block a
// sequence); 8 tokens of 32 streams: 12.4 us, 1.5 TB/s of the two rows each.
// VEC: rows start on 16-byte boundaries.
template <bool VEC>
__global__ void __cluster_dims__(kVerifyCtas, 1, 1) __launch_bounds__(kVerifyThreads, 2)
    verify_draft_kernel(const VerifyParams p) {
  constexpr uint32_t E = VEC ? 4 : 1;                  // values of a thread at a time
  constexpr uint32_t kTile = kVerifyThreads * E;
  constexpr uint32_t kTiles = kVerifyVocab / kVerifyCtas / kTile;
  __shared__ uint64_t sums[kTiles][kVerifyWarps], warp_total[kVerifyWarps], cta_total;
  __shared__ uint32_t run, positive;
  namespace cg = cooperative_groups;
  const cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = blockIdx.x % kVerifyCtas, seq = blockIdx.x / kVerifyCtas;
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t drafted = p.counts ? (uint32_t)min(max(p.counts[seq], 0), (int32_t)p.drafted) : p.drafted;
  const float u = p.u_sample[seq];
  if (warp == 0) {
    uint32_t n = drafted;
    for (uint32_t base = 0; base < drafted; base += 32) {
      const uint32_t t = base + lane;
      bool ok = true;
      if (t < drafted) {
        const size_t i = (size_t)seq * p.drafted + t;
        const int32_t x = p.tokens[i];
        const float ua = p.u_accept[i];
        ok = x >= 0 && (uint32_t)x < p.vocab &&
             ua * p.draft[i * p.vocab + x] < p.target[(i + seq) * p.vocab + x];   // target rows: drafted + 1 a sequence
      }
      const uint32_t no = __ballot_sync(~0u, !ok);
      if (no) {
        n = base + __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) run = n;
  }
  __syncthreads();
  const uint32_t n = run;
  const float *row = p.target + ((size_t)seq * (p.drafted + 1) + n) * p.vocab;
  const float *less = n < drafted ? p.draft + ((size_t)seq * p.drafted + n) * p.vocab : nullptr;
  const uint32_t stretch = (p.vocab + kVerifyCtas * E - 1) / (kVerifyCtas * E) * E;
  const uint32_t begin = min(p.vocab, rank * stretch), end = min(p.vocab, begin + stretch);
  auto value = [&](uint32_t i) { return row[i] - (less ? less[i] : 0.f); };
  uint64_t total = 0, before = 0;
  for (;;) {
    uint64_t mine = 0;
    bool any = false;
    if (tid == 0) positive = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t base = begin; base < end; base += kTile) {
      const uint32_t i = base + tid * E;
      uint64_t w = 0;
      if constexpr (VEC) {
        if (i < end) {   // the vocabulary and every stretch are multiples of 4
          float4 x = *(const float4 *)(row + i);
          if (less) {
            const float4 y = *(const float4 *)(less + i);
            x.x -= y.x, x.y -= y.y, x.z -= y.z, x.w -= y.w;
          }
          any |= x.x > 0.f || x.y > 0.f || x.z > 0.f || x.w > 0.f;
          w = fixed_probability(x.x) + fixed_probability(x.y) + fixed_probability(x.z) + fixed_probability(x.w);
        }
      } else if (i < end) {
        const float x = value(i);
        any |= x > 0.f;
        w = fixed_probability(x);
      }
      w = warp_sum(w);
      if (lane == 0) sums[(base - begin) / kTile][warp] = w;
      mine += w;
    }
    if (lane == 0) warp_total[warp] = mine;
    if (__any_sync(~0u, any) && lane == 0) positive = 1;
    __syncthreads();
    if (tid == 0) {
      uint64_t all = 0;
      for (uint32_t w = 0; w < kVerifyWarps; ++w) all += warp_total[w];
      cta_total = all;
    }
    cluster.sync();
    uint32_t some = 0;
    total = before = 0;
    for (uint32_t r = 0; r < kVerifyCtas; ++r) {
      const uint64_t x = *cluster.map_shared_rank(&cta_total, r);
      some |= *cluster.map_shared_rank(&positive, r);
      before += r < rank ? x : 0;
      total += x;
    }
    cluster.sync();   // the others have read this CTA's words: they may change, or the CTA end
    if (some || !less) break;
    less = nullptr;   // p <= q everywhere: draw from p
  }
  const uint64_t u24 = (uint64_t)(fminf(fmaxf(u, 0.f), 0x1.fffffep-1f) * 0x1p24f);
  const uint64_t point = (__umul64hi(u24, total) << 40) | (u24 * total >> 24);   // u24 / 2^24 of the total, rounded down
  if (rank == 0 && tid == 0) {
    p.accepted[seq] = (int32_t)n;
    if (total == 0) p.next[seq] = (int32_t)p.vocab - 1;
  }
  if (warp != 0 || point < before || point >= before + cta_total) return;
  // the chunk (tile, warp) that holds the point, then the value in it
  const uint32_t chunks = (end - begin + kTile - 1) / kTile * kVerifyWarps;
  uint64_t at = before;
  for (uint32_t base = 0; base < chunks; base += 32) {
    const uint64_t own = (&sums[0][0])[base + lane];
    uint64_t sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    const uint32_t past = __ballot_sync(~0u, at + sum > point);
    if (!past) {
      at += __shfl_sync(~0u, sum, 31);
      continue;
    }
    const int k = __ffs(past) - 1;
    at += __shfl_sync(~0u, sum - own, k);
    const uint32_t chunk = base + k, first = begin + chunk / kVerifyWarps * kTile + chunk % kVerifyWarps * 32 * E;
    for (uint32_t j = 0; j < E; ++j) {   // 32 values at a time
      const uint32_t i = first + j * 32 + lane;
      uint64_t w = i < end ? fixed_probability(value(i)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint64_t up = __shfl_up_sync(~0u, w, o);
        if (lane >= (uint32_t)o) w += up;
      }
      const uint32_t hit = __ballot_sync(~0u, at + w > point);
      if (hit) {
        if (lane == 0) p.next[seq] = (int32_t)(first + j * 32 + __ffs(hit) - 1);
        return;
      }
      at += __shfl_sync(~0u, w, 31);
    }
    return;
  }
}

}  // namespace vg
