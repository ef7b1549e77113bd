// Verification of drafted tokens against a model's probabilities.
#pragma once
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

constexpr uint32_t kVerifyThreads = 1024;

// A probability as a multiple of 2^-38. Sums of these are exact, so a total and
// a cumulative sum do not depend on the order they are taken in, and a sampled
// token does not depend on the launch shape. NaN and negative values count as
// 0, values above 1 as 1.
__device__ __forceinline__ uint64_t fixed_probability(float x) {
  return (uint64_t)(fminf(fmaxf(x, 0.f), 1.f) * 0x1p38f);
}

// Token t is accepted while u_t * q(x_t) < p(x_t); the first token that is not
// ends the run, and the next token is drawn from max(p - q, 0) there, or from p
// after the last drafted token (or where p <= q everywhere).
__global__ void __launch_bounds__(kVerifyThreads) verify_draft_kernel(const VerifyParams p) {
  __shared__ uint64_t sums[32];
  __shared__ uint32_t first_bad, found;
  const uint32_t seq = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t drafted = p.counts ? (uint32_t)min(max(p.counts[seq], 0), (int32_t)p.drafted) : p.drafted;
  if (tid == 0) first_bad = drafted, found = p.vocab;
  __syncthreads();
  for (uint32_t t = tid; t < drafted; t += kVerifyThreads) {
    const int32_t x = p.tokens[(size_t)seq * p.drafted + t];
    bool ok = false;
    if (x >= 0 && (uint32_t)x < p.vocab) {
      const float q = p.draft[((size_t)seq * p.drafted + t) * p.vocab + x];
      const float pr = p.target[((size_t)seq * (p.drafted + 1) + t) * p.vocab + x];
      ok = p.u_accept[(size_t)seq * p.drafted + t] * q < pr;
    }
    if (!ok) atomicMin(&first_bad, t);
  }
  __syncthreads();
  const uint32_t n = first_bad;
  const float *row = p.target + ((size_t)seq * (p.drafted + 1) + n) * p.vocab;
  const float *minus = n < drafted ? p.draft + ((size_t)seq * p.drafted + n) * p.vocab : nullptr;
  uint64_t total = 0;
  for (int attempt = 0; attempt < 2; ++attempt) {
    uint64_t mine = 0;
    bool any = false;
    for (uint32_t i = tid; i < p.vocab; i += kVerifyThreads) {
      const float x = row[i] - (minus ? minus[i] : 0.f);
      any |= x > 0.f;
      mine += fixed_probability(x);
    }
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
    __syncthreads();
    if (lane == 0) sums[warp] = mine;
    any = __syncthreads_or(any);
    total = 0;
    for (uint32_t i = 0; i < 32; ++i) total += sums[i];
    if (any || !minus) break;
    minus = nullptr;  // p <= q everywhere: draw from p
  }
  const float u = p.u_sample[seq];
  const uint64_t u24 = (uint64_t)(fminf(fmaxf(u, 0.f), 0x1.fffffep-1f) * 0x1p24f);
  const uint64_t point = (__umul64hi(u24, total) << 40) | (u24 * total >> 24);
  uint64_t before = 0;
  for (uint32_t base = 0; base < p.vocab; base += kVerifyThreads) {
    const uint32_t i = base + tid;
    uint64_t sum = i < p.vocab ? fixed_probability(row[i] - (minus ? minus[i] : 0.f)) : 0;
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    uint64_t all = 0;
    for (uint32_t k = 0; k < 32; ++k) {
      if (k < warp) sum += sums[k];
      all += sums[k];
    }
    if (i < p.vocab && before + sum > point) atomicMin(&found, i);
    before += all;
    if (before > point) break;
  }
  __syncthreads();
  if (tid == 0) {
    p.accepted[seq] = (int32_t)n;
    p.next[seq] = (int32_t)min(found, p.vocab - 1);
  }
}

}  // namespace vg
