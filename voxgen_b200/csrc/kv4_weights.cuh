// The attention that cache rows draw.
#pragma once
#include "kv4_rows_attention.cuh"

namespace vg {

constexpr uint32_t kWeightWarps = 8;

template <int D>
__device__ __forceinline__ void row_values(const uint8_t *run, uint32_t row, int v, uint32_t lane, float (&x)[D / 32]) {
  constexpr int N = D / 32;  // channels of a lane
  const uint8_t *b = run + Kv4<D>::codes(row, v) + lane * N / 2;
  uint32_t w = N == 4 ? *(const uint16_t *)b : *b;
  const float d = __half2float(*(const __half *)(run + Kv4<D>::scales(row, v) + lane * N / 32 * 2));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = (float)((int)(w >> (4 * i) & 15) - 8) * d;
}

// weights[row] += the attention that the call's query rows gave to the row: one
// warp per cache row, recomputing its scores.
template <int D, typename T>
__global__ void __launch_bounds__(kWeightWarps * 32) kv4_weights_kernel(const Kv4AttnParams p) {
  constexpr int N = D / 32;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t blocks = (p.c.capacity + kWeightWarps - 1) / kWeightWarps;
  const uint32_t lane_row = blockIdx.x / blocks, seq = lane_row / p.c.kv_heads, kv = lane_row % p.c.kv_heads;
  const uint32_t row = blockIdx.x % blocks * kWeightWarps + warp;
  if (row >= p.c.capacity || row >= kv4_held(p.c, seq)) return;
  const uint32_t held = kv4_held(p.c, seq);
  const int32_t count = kv4_count(p, seq);
  float k[N], sum = 0.f;
  row_values<D>(p.c.data + (size_t)lane_row * p.c.tiles * Kv4<D>::kTileBytes, row, 0, lane, k);
  for (uint32_t t = 0; t < p.tokens; ++t) {
    if ((int32_t)t >= count || (int64_t)row > (int64_t)held - count + t) continue;
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
