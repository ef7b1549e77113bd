// The attention that cache rows draw: weights[row] += the sum, over a call's query
// rows, of exp2(score - log2 of the row's softmax denominator).
//
// The denominators come from the attention kernel before it; the scores are
// computed again, which needs the K codes once more (72 bytes a row, from L2
// after a decode step) and no room for P. A warp unpacks 32 cache rows to MMA A
// operands that stay in its registers, and the query rows pass by as B fragments
// in shared memory, 64 at a time. With 5 tokens of 16 ragged streams it adds 6 us to
// the attention's 25 (one warp a cache row, scalar, took 200). Every row is summed by one warp in a fixed
// order and written by one lane.
#pragma once
#include "kv4_rows_attention.cuh"

namespace vg {

constexpr uint32_t kWeightWarps = 8, kWeightThreads = kWeightWarps * 32;
constexpr uint32_t kWeightRows = kWeightWarps * 32;   // cache rows of a block
constexpr uint32_t kWeightTiles = 8;                  // of 8 query rows, in shared memory at a time

template <int D, typename T>
constexpr uint32_t kWeightSmem = kWeightTiles * (D / 16) * 32 * 2 * 4 * (sizeof(T) == 4 ? 2 : 1);

template <int D, typename T>
__global__ void __launch_bounds__(kWeightThreads, 2) kv4_weights_kernel(const Kv4AttnParams p) {
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr int kSteps = D / 16;
  constexpr uint32_t kFrag = kSteps * 32 * 2 * (kSplit ? 2 : 1);   // words of a tile's fragments
  extern __shared__ __align__(16) uint32_t frags[];
  __shared__ float factors[kWeightTiles * 8], denominators[kWeightTiles * 8];
  __shared__ uint32_t seens[kWeightTiles * 8];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const uint32_t blocks = (p.c.capacity + kWeightRows - 1) / kWeightRows;
  const uint32_t lane_row = blockIdx.x / blocks, seq = lane_row / p.c.kv_heads, kv = lane_row - seq * p.c.kv_heads;
  const uint32_t held = kv4_held(p.c, seq), block_row = (blockIdx.x - lane_row * blocks) * kWeightRows;
  if (block_row >= held) {
    // One block at least waits for the attention, so that no kernel after this one starts before it is done. The other
    // idle ones make room.
    if (blockIdx.x == 0) pdl_wait();
    return;
  }
  const uint32_t row0 = block_row + warp * 32, rows = p.tokens * p.group;
  const uint8_t *run = p.c.data + (size_t)lane_row * p.c.tiles * Kv4<D>::kTileBytes;
  float old[4];   // only this kernel and append write them, and both of those before are done
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = row0 + 8 * i + g;
    old[i] = t == 0 && row < held ? p.c.weights[(size_t)lane_row * p.c.capacity + row] : 0.f;
  }
  // ---- K rows row0 + {g, 8 + g, 16 + g, 24 + g} as A fragments ----
  uint32_t a[2][kSteps][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t row = row0 + 8 * i + g;
    uint32_t w[kSteps / 2] = {};
    __half2 d = __half2half2(__half(0.f));
    if (row < held) {
      const uint8_t *b = run + Kv4<D>::codes(row, 0) + t * (D / 8);
      if constexpr (D == 128) {
        const uint4 v = *(const uint4 *)b;
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
        const uint2 v = *(const uint2 *)b;
        w[0] = v.x, w[1] = v.y;
      }
      d = __half2half2(*(const __half *)(run + Kv4<D>::scales(row, 0) + t * (D / 4) / 32 * 2));
    }
    const __half2 d72 = minus72(d);
#pragma unroll
    for (int k = 0; k < kSteps / 2; ++k) {
      __half2 h[4];
      unpack8(w[k], d, d72, h);
#pragma unroll
      for (int y = 0; y < 4; ++y) a[i / 2][2 * k + y / 2][y % 2 * 2 + i % 2] = half2_bits(h[y]);
    }
  }
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t base = 0; base < rows; base += kWeightTiles * 8) {
    __syncthreads();
    const uint32_t n = min(kWeightTiles * 8, rows - base), tiles = (n + 7) / 8;
    // a warp takes rows warp, warp + 8, ... (column `warp` of every tile), four loads in flight
#pragma unroll 1
    for (uint32_t j0 = 0; j0 < tiles; j0 += 4) {
      float x[4][D / 32];
      uint32_t seen[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) seen[j] = load_query<D, T>(p, seq, kv, base + (j0 + j) * 8 + warp, held, x[j]);
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        if (j0 + j >= tiles) break;
        const float factor = store_query<D, T>(p, x[j], warp, frags + (j0 + j) * kFrag);
        const uint32_t i = (j0 + j) * 8 + warp;
        if (lane == 0) factors[i] = factor, seens[i] = seen[j];
      }
    }
    if (base == 0) pdl_wait();   // what follows needs the attention's sums
    if (threadIdx.x < tiles * 8) {
      const uint32_t r = base + threadIdx.x, tok = r / p.group;
      denominators[threadIdx.x] =
          r < rows ? p.lse[((size_t)seq * p.tokens + tok) * p.heads + kv * p.group + r - tok * p.group] : INFINITY;
    }
    __syncthreads();
    if (row0 >= held) continue;
#pragma unroll 1
    for (uint32_t j = 0; j < tiles; ++j) {
      const uint32_t *f = frags + j * kFrag;
      float c[2][4] = {};
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        uint32_t b[2];
        *(uint2 *)b = *(const uint2 *)(f + (k * 32 + lane) * 2);
        mma_f16(c[0], a[0][k], b);
        mma_f16(c[1], a[1][k], b);
        if constexpr (kSplit) {
          *(uint2 *)b = *(const uint2 *)(f + ((kSteps + k) * 32 + lane) * 2);
          mma_f16(c[0], a[0][k], b);
          mma_f16(c[1], a[1][k], b);
        }
      }
#pragma unroll
      for (int z = 0; z < 2; ++z) {   // query rows 8j + 2t + z
        const uint32_t q = j * 8 + 2 * t + z;
        const float scale = factors[q], minus = denominators[q];
        const uint32_t seen = seens[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = exp2_fast(fmaf(c[i / 2][i % 2 * 2 + z], scale, -minus));
          sum[i] += row0 + 8 * i + g < seen ? e > 1.f ? 1.f : e : 0.f;   // a share; past 2^24, scores are off by more than 1
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    sum[i] += __shfl_xor_sync(~0u, sum[i], 1);
    sum[i] += __shfl_xor_sync(~0u, sum[i], 2);
    const uint32_t row = row0 + 8 * i + g;
    if (t == 0 && row < held) p.c.weights[(size_t)lane_row * p.c.capacity + row] = old[i] + sum[i];
  }
}

}  // namespace vg
