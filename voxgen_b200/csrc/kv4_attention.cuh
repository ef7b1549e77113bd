// Attention over a 4-bit cache.
#pragma once
#include "kv4_rows.cuh"

namespace vg {

struct Kv4AttnParams {
  Kv4View c;
  const void *q;
  void *out;                // [seqs][tokens][heads][D]
  float *lse;               // [seqs][tokens][heads]: log2 of the softmax's denominator, when weights are tracked
  Strides qs;
  const int32_t *counts;    // new tokens of each sequence, may be null
  uint32_t tokens, heads, group;
  float scale;              // of the scores, times log2(e)
};

// Rows that query token t of a sequence sees; 0 for a token past its count.
__device__ __forceinline__ uint32_t kv4_seen(const Kv4AttnParams &p, uint32_t seq, uint32_t t) {
  const int32_t rows = min(max(p.c.state[seq].rows, 0), (int32_t)p.c.capacity);
  const int32_t count = p.counts ? min(max(p.counts[seq], 0), (int32_t)p.tokens) : (int32_t)p.tokens;
  const int32_t seen = rows - count + (int32_t)t + 1;
  return (int32_t)t < count && seen > 0 ? (uint32_t)seen : 0u;
}

constexpr uint32_t kAttnWarps = 8;

template <int D>
__device__ __forceinline__ void row_values(const uint8_t *run, uint32_t row, int v, uint32_t lane, float (&x)[D / 32]) {
  constexpr int N = D / 32;  // channels of a lane
  const uint8_t *b = run + Kv4<D>::codes(row, v) + lane * N / 2;
  uint32_t w = N == 4 ? *(const uint16_t *)b : *b;
  const float d = __half2float(*(const __half *)(run + Kv4<D>::scales(row, v) + lane * N / 32 * 2));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)((int)(w >> (4 * i) & 15) - 8) * d;
}

// One block per query row, one cache row per warp at a time.
template <int D, typename T>
__global__ void __launch_bounds__(kAttnWarps * 32) kv4_attention_kernel(const Kv4AttnParams p) {
  constexpr int N = D / 32;
  __shared__ float part[kAttnWarps][D], maxs[kAttnWarps], sums[kAttnWarps];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t head = blockIdx.x % p.heads, t = blockIdx.x / p.heads % p.tokens, seq = blockIdx.x / p.heads / p.tokens;
  const uint32_t seen = kv4_seen(p, seq, t);
  const T *q = (const T *)p.q + (int64_t)seq * p.qs.seq + (int64_t)t * p.qs.token + (int64_t)head * p.qs.head + lane * N;
  float x[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)q[i] * p.scale;
  const uint8_t *run = p.c.data + ((size_t)seq * p.c.kv_heads + head / p.group) * p.c.tiles * Kv4<D>::kTileBytes;
  for (uint32_t row = warp; row < seen; row += kAttnWarps) {
    float k[N], v[N], s = 0.f;
    row_values<D>(run, row, 0, lane, k);
    row_values<D>(run, row, 1, lane, v);
#pragma unroll
    for (int i = 0; i < N; ++i) s += x[i] * k[i];
#pragma unroll
    for (int b = 16; b; b >>= 1) s += __shfl_xor_sync(~0u, s, b);
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.f : exp2f(m - top), e = exp2f(s - top);
    m = top;
    l = l * old + e;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * old + e * v[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) part[warp][lane * N + i] = o[i];
  if (lane == 0) maxs[warp] = m, sums[warp] = l;
  __syncthreads();
  float top = -INFINITY, all = 0.f;
  for (uint32_t w = 0; w < kAttnWarps; ++w) top = fmaxf(top, maxs[w]);
  for (uint32_t w = 0; w < kAttnWarps; ++w) all += maxs[w] == -INFINITY ? 0.f : sums[w] * exp2f(maxs[w] - top);
  if (threadIdx.x < D) {
    float sum = 0.f;
    for (uint32_t w = 0; w < kAttnWarps; ++w)
      sum += maxs[w] == -INFINITY ? 0.f : part[w][threadIdx.x] * exp2f(maxs[w] - top);
    ((T *)p.out)[(size_t)blockIdx.x * D + threadIdx.x] = from_float<T>(seen ? sum / all : 0.f);
  }
  if (p.lse && threadIdx.x == 0) p.lse[blockIdx.x] = seen ? top + log2f(all) : INFINITY;
}

// weights[row] += the attention that the call's query rows gave to the row: one
// warp per cache row, recomputing its scores.
template <int D, typename T>
__global__ void __launch_bounds__(kAttnWarps * 32) kv4_weights_kernel(const Kv4AttnParams p) {
  constexpr int N = D / 32;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t blocks = (p.c.capacity + kAttnWarps - 1) / kAttnWarps;
  const uint32_t lane_row = blockIdx.x / blocks, seq = lane_row / p.c.kv_heads, kv = lane_row % p.c.kv_heads;
  const uint32_t row = blockIdx.x % blocks * kAttnWarps + warp;
  if (row >= p.c.capacity || row >= (uint32_t)max(p.c.state[seq].rows, 0)) return;
  float k[N], sum = 0.f;
  row_values<D>(p.c.data + (size_t)lane_row * p.c.tiles * Kv4<D>::kTileBytes, row, 0, lane, k);
  for (uint32_t t = 0; t < p.tokens; ++t) {
    if (row >= kv4_seen(p, seq, t)) continue;
    for (uint32_t g = 0; g < p.group; ++g) {
      const uint32_t head = kv * p.group + g;
      const T *q = (const T *)p.q + (int64_t)seq * p.qs.seq + (int64_t)t * p.qs.token + (int64_t)head * p.qs.head + lane * N;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += (float)q[i] * p.scale * k[i];
#pragma unroll
      for (int b = 16; b; b >>= 1) s += __shfl_xor_sync(~0u, s, b);
      sum += exp2f(s - p.lse[((size_t)seq * p.tokens + t) * p.heads + head]);
    }
  }
  if (lane == 0) p.c.weights[(size_t)lane_row * p.c.capacity + row] += sum;
}

}  // namespace vg
