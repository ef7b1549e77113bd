// Attention of single tokens over a paged cache, over all of a sequence's pages or
// over a list of them, split over the length and joined.
//
// The mathematics. Up to 8 query heads of a KV head are the columns of m16n8k16
// MMAs: scores S^T = K Q^T and the output O^T = V^T P^T, cache rows as the A
// operand. q is held in as many terms of the cache's type as its bits need (fp32:
// two of fp16, three of bf16), P in two, three for fp32 output over a bf16 cache; so
// products are as exact as fp32's. Statistics and sums are fp32. The tensor cores
// add with rounding towards zero, so for fp32 queries O is summed afresh every 8
// steps and added with rounding to nearest.
//
// The bound is bytes: 4 D of them a row for 4 D multiply-adds a head. So one warp
// does nothing but keep copies in flight: it looks page numbers up 32 at a time and
// issues tensor copies of 16 rows (K and V; 8 KB at head_dim 128) into the rings of
// 8 consumer warps, 192 KB in all, through 128-byte swizzled boxes that ldmatrix
// reads without bank conflicts. A consumer takes every 8th block of 16 rows and
// keeps its own softmax state; the consumers meet when the piece ends.
//
// The split. A segment is a (query, KV head, 8 heads of it); it is cut into pieces
// of at most U blocks of 16 rows, U such that there is about one piece for each of
// the 148 CTAs (4, where segments are many). A segment of several pieces leaves a
// partial result for each, and the CTA that finishes last (a counter, left at zero)
// adds them in order: sums never depend on timing.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "kv4_rows_attention.cuh"
#include "paged.cuh"

namespace vg {

struct PagedAttnParams {
  PagedTable t;
  uint32_t kv_heads;
  const void *q;
  void *out;                 // [queries][heads][D]
  int64_t q_query, q_head;   // strides
  PagedQueries which;
  const int32_t *chosen;     // [queries][kv_heads][budget] pages of each (query, KV head), or null: all
  uint32_t budget;
  uint32_t queries, heads, group, head_tiles;   // head_tiles: of 8 heads, of a KV head
  float scale;               // of the scores, times log2(e)
  uint32_t *tickets;         // [segments], zero between calls
  float *parts;              // [pieces] partial results
};

constexpr uint32_t kPagedBlock = 16;     // cache rows of a block: never more than one page's
constexpr uint32_t kPagedWarps = 8;      // consumers
constexpr uint32_t kPagedThreads = (kPagedWarps + 1) * 32;
constexpr uint32_t kPagedCtas = 148;     // one per SM
constexpr uint32_t kPagedHeads = 8;      // columns of a tile
constexpr uint32_t kPagedLeast = 16;     // blocks of a piece: two rounds of the warps
constexpr uint32_t kPagedTickets = 1u << 14;   // segments that may be cut

template <int D>
struct PagedSmem {
  static constexpr uint32_t kHalf = 2 * kPagedBlock * 128;     // one copy: 64 channels of 16 K rows, then of 16 V rows
  static constexpr uint32_t kStage = kHalf * (D / 64);
  static constexpr uint32_t kStages = 24 / kPagedWarps * 128 / D;   // of a warp's ring
  static constexpr uint32_t kRing = kPagedWarps * kStages * kStage;
  static constexpr uint32_t kRow = 68;                         // floats of a row when results meet: 64 and 4 against bank conflicts
  static constexpr uint32_t kMerge = 20480;                    // results of 64 channels, or the weights of up to 640 pieces
  static constexpr uint32_t kBytes = kRing + kMerge + 1024;    // the ring starts on a multiple of 1024
  static_assert(kPagedWarps * kPagedHeads * kRow * 4 <= kMerge, "");
};

// Pieces that a call may be cut into: `segments` plus what the target allows.
__host__ __device__ __forceinline__ uint32_t paged_target(uint32_t segments) {
  return kPagedCtas * (segments * 4 <= kPagedCtas * 3 ? 1 : 4);
}
static_assert((kPagedCtas * 4 + 1) * kPagedHeads * 4 <= PagedSmem<128>::kMerge, "a segment's pieces have their weights there");
__host__ __device__ __forceinline__ uint64_t paged_pieces(uint64_t segments) {
  return segments > kPagedTickets ? 0 : segments + paged_target((uint32_t)segments);
}

// Blocks of 16 rows that a query's segments have: at least one, so that every output is written.
__device__ __forceinline__ uint32_t paged_blocks(const PagedAttnParams &p, uint32_t query) {
  if (query >= p.queries) return 0;
  if (p.chosen) return p.budget << (p.t.shift - 4);
  return max(1u, (paged_seen(p.t, p.which, query).seen + kPagedBlock - 1) / kPagedBlock);
}
// How segments are cut, as for the 4-bit cache: pieces of `size` blocks, `pieces` of them. A warp's work.
struct PagedPlan {
  uint32_t lanes, size, pieces;   // lanes: segments of a query
};
__device__ __forceinline__ uint32_t paged_pieces_of(uint32_t blocks, uint32_t size) { return (blocks + size - 1) / size; }
__device__ __forceinline__ PagedPlan paged_plan(const PagedAttnParams &p) {
  const uint32_t lane = threadIdx.x % 32, lanes = p.kv_heads * p.head_tiles, segments = p.queries * lanes;
  PagedPlan x{lanes, 1u << 30, segments};   // one piece a segment
  if (segments > kPagedTickets) return x;
  uint32_t total = 0;
#pragma unroll 1
  for (uint32_t s = lane; s < p.queries; s += 32) total += paged_blocks(p, s);
  total = __reduce_add_sync(~0u, total) * lanes;   // the host keeps it below 2^31
  const uint32_t target = paged_target(segments);
  x.size = max(kPagedLeast, (total + target - 1) / target);
#pragma unroll 1
  for (int i = 0;; ++i) {
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t s = lane; s < p.queries; s += 32) n += paged_pieces_of(paged_blocks(p, s), x.size);
    x.pieces = __reduce_add_sync(~0u, n) * lanes;
    if (x.pieces <= target || i == 3) return x;
    x.size = max(x.size + 1, (uint32_t)((uint64_t)x.size * x.pieces / target));
  }
}

struct PagedPiece {
  uint32_t query, lane;         // lane: (KV head, 8 heads of it)
  uint32_t part, parts;         // of the segment
  uint32_t first, blocks;       // of the piece, in the segment
};
__device__ __forceinline__ PagedPiece paged_piece(const PagedAttnParams &p, const PagedPlan &x, uint32_t index) {
  const uint32_t lane = threadIdx.x % 32;
  uint32_t before = 0;
#pragma unroll 1
  for (uint32_t base = 0; base < p.queries; base += 32) {
    const uint32_t blocks = paged_blocks(p, base + lane), n = paged_pieces_of(blocks, x.size);
    uint32_t sum = n * x.lanes;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > index);
    if (past) {
      const int at = __ffs(past) - 1;
      const uint32_t parts = __shfl_sync(~0u, n, at), all = __shfl_sync(~0u, blocks, at);
      const uint32_t into = index - before - (__shfl_sync(~0u, sum, at) - parts * x.lanes);
      PagedPiece y;
      y.query = base + at;
      y.lane = into / parts;
      y.part = into - y.lane * parts;
      y.parts = parts;
      y.first = y.part * x.size;
      y.blocks = min(x.size, all - y.first);
      return y;
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return PagedPiece{0, 0, 0, 1, 0, 0};   // past the last piece
}

// ---- MMA operands of either type ----
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __half) { mma_f16(c, a, b); }
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Two values rounded to a pair of type C, and what is left of them.
__device__ __forceinline__ uint32_t take_pair(float &x, float &y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x -= f.x, y -= f.y;
  return half2_bits(h);
}
__device__ __forceinline__ uint32_t take_pair(float &x, float &y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  x -= f.x, y -= f.y;
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
// One box of the pool: 64 channels from x on, 16 rows from `row` on, of K and V, of (page, KV head) `place`.
__device__ __forceinline__ void tensor_g2s(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t row, int32_t place, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(row), "r"(0), "r"(place), "r"(smem_u32(bar))
      : "memory");
}

// T: type of q and out; C: the cache's.
template <typename T, typename C>
constexpr int kQTerms = std::is_same<C, __half>::value ? (sizeof(T) == 4 ? 2 : 1)
                        : sizeof(T) == 4 ? 3 : std::is_same<T, __half>::value ? 2 : 1;
// P rounded once to fp16 adds to a bf16 output an eighth of its own rounding; once to bf16, as much as that.
template <typename T, typename C>
constexpr int kPTerms = std::is_same<C, __half>::value ? (std::is_same<T, __nv_bfloat16>::value ? 1 : 2) : sizeof(T) == 4 ? 3 : 2;
// P is held times 2^6 in fp16, for the range below a weight of 1 (kv4_rows_attention.cuh); bf16 has range enough.
template <typename C>
constexpr float kPagedPScale = std::is_same<C, __half>::value ? kPScale : 0.f;

template <int D, typename T, typename C>
__global__ void __launch_bounds__(kPagedThreads, 1)
    paged_attention_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ CUtensorMap map) {
  using S = PagedSmem<D>;
  constexpr int kSteps = D / 16;                // k-steps of a score, and m-tiles of the output
  constexpr int kQ = kQTerms<T, C>, kP = kPTerms<T, C>;
  constexpr bool kFresh = sizeof(T) == 4;       // O summed afresh
  constexpr uint32_t kFreshSteps = 8;
  extern __shared__ uint8_t paged_smem[];
  __shared__ uint64_t full[kPagedWarps][S::kStages], empty[kPagedWarps][S::kStages];
  __shared__ uint32_t valid_rows[kPagedWarps][S::kStages];
  __shared__ __align__(8) float w_max[kPagedWarps][kPagedHeads], w_sum[kPagedWarps][kPagedHeads];
  __shared__ float f_max[kPagedHeads], f_sum[kPagedHeads];
  __shared__ uint32_t last, gave_up;
  __shared__ __align__(8) uint32_t q_frag[kQ][kSteps][32][2];   // B fragments
  __shared__ __align__(8) float factors[kPagedHeads];
  __shared__ PagedPlan shared_plan;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const uint32_t base = smem_u32(paged_smem), ring = (base + 1023) & ~1023u;
  float *merge = (float *)(paged_smem + (ring - base) + S::kRing);
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map));
    gave_up = 0;
  }
  if (warp < kPagedWarps && lane < S::kStages) mbar_init(&full[warp][lane], 1), mbar_init(&empty[warp][lane], 1);
  fence_mbar_init();
  pdl_launch_dependents();
  pdl_wait();
  if (warp == kPagedWarps) {
    const PagedPlan x = paged_plan(p);
    if (lane == 0) shared_plan = x;
  }
  __syncthreads();
  const PagedPlan plan = shared_plan;

  if (warp == kPagedWarps) {
    // ================= the copying warp =================
    uint32_t round = 0;        // rounds of 8 blocks, over all pieces
    bool stopped = false;
#pragma unroll 1
    for (uint32_t index = blockIdx.x; index < plan.pieces && !stopped; index += gridDim.x) {
      const PagedPiece x = paged_piece(p, plan, index);
      const PagedSeen who = paged_seen(p.t, p.which, x.query);
      const uint32_t kv = x.lane / p.head_tiles, page_rows = p.t.page_rows();
      const int32_t *table = p.t.table + (size_t)who.seq * p.t.seq_pages;
      const int32_t *list = p.chosen ? p.chosen + ((size_t)x.query * p.kv_heads + kv) * p.budget : nullptr;
      // page and rows (1 to 16, 5 bits) of the piece's block i; 0: nothing to read
      const auto find = [&](uint32_t i) -> uint32_t {
        if (i >= x.blocks) return 0;
        const uint32_t row = (x.first + i) * kPagedBlock, entry = row >> p.t.shift, in = row & (page_rows - 1);
        const uint32_t at = list ? (uint32_t)list[entry] : entry;
        if (at >= p.t.seq_pages) return 0;
        const uint32_t first = (at << p.t.shift) + in;
        if (first >= who.seen) return 0;
        const uint32_t page = (uint32_t)table[at];
        return page < p.t.pages ? page << 5 | min(kPagedBlock, who.seen - first) : 0;
      };
      uint32_t next = find(lane);
#pragma unroll 1
      for (uint32_t i = 0; i < x.blocks && !stopped; i += 32) {
        const uint32_t now = next;
        next = find(i + 32 + lane);
#pragma unroll 1
        for (uint32_t j = 0; j < 4 && i + 8 * j < x.blocks; ++j, ++round) {
          const uint32_t block = __shfl_sync(~0u, now, 8 * j + lane % 8);
          bool in = true;
          if (lane < kPagedWarps) {
            const uint32_t stage = round % S::kStages, turn = round / S::kStages;
            if (turn) in = mbar_wait_bounded(&empty[lane][stage], (turn - 1) & 1);
            if (in) {
              valid_rows[lane][stage] = block & 31;
              uint64_t *bar = &full[lane][stage];
              if (block & 31) {
                mbar_arrive_expect_tx(bar, S::kStage);
                const int32_t place = (int32_t)((block >> 5) * p.kv_heads + kv);
                const int32_t row = (int32_t)(((x.first + i + 8 * j + lane) * kPagedBlock) & (page_rows - 1));
                const uint32_t dst = ring + (lane * S::kStages + stage) * S::kStage;
#pragma unroll
                for (int h = 0; h < D / 64; ++h) tensor_g2s(dst + h * S::kHalf, &map, h * 64, row, place, bar);
              } else {
                mbar_arrive(bar);
              }
            }
          }
          if (!__all_sync(~0u, in)) {
            if (lane == 0) *(volatile uint32_t *)&gave_up = 1;
            stopped = true;
            break;
          }
        }
      }
    }
    if (stopped && lane == 0) atomicOr(&p.t.pool[1], kPagedTimeout);
    return;
  }

  // ================= the consumers =================
  uint32_t round = 0;
  bool stopped = false;      // a wait ran out: nothing is waited for any more
  const uint32_t my_ring = ring + warp * S::kStages * S::kStage;
  // this lane's row of an ldmatrix, and which of the two 16-byte chunks it reads
  const uint32_t k_row = lane % 8 + (lane / 8 % 2) * 8, k_chunk = lane / 16;
  const uint32_t v_row = lane % 8 + (lane / 16) * 8, v_chunk = lane / 8 % 2;
#pragma unroll 1
  for (uint32_t index = blockIdx.x; index < plan.pieces; index += gridDim.x) {
    const PagedPiece seg = paged_piece(p, plan, index);
    const bool whole = seg.parts == 1;
    const uint32_t kv = seg.lane / p.head_tiles, head0 = (seg.lane - kv * p.head_tiles) * kPagedHeads;
    const uint32_t tile_heads = min(kPagedHeads, p.group - head0);
    // ---- the queries as B fragments, a warp a head: column `warp` of the MMA ----
    {
      constexpr uint32_t N = D / 32;
      float x[N];
      const T *q = (const T *)p.q + (int64_t)seg.query * p.q_query + (int64_t)(kv * p.group + head0 + warp) * p.q_head + lane * N;
      uint32_t top = 0;
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        x[i] = warp < tile_heads ? (float)q[i] : 0.f;
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
      }
      // fp16's range is met by a power of two a head; bf16 has fp32's
      float inverse = 1.f, power = 1.f;
      if constexpr (std::is_same<C, __half>::value) power = row_power(__uint_as_float(__reduce_max_sync(~0u, top)), inverse);
#pragma unroll
      for (uint32_t i = 0; i < N; i += 2) {   // channels c, c + 1: step c / 16, lane 4 warp + c % 8 / 2, register c % 16 / 8
        const uint32_t c = lane * N + i;
        float a = x[i] * power, b = x[i + 1] * power;
#pragma unroll
        for (int k = 0; k < kQ; ++k) q_frag[k][c / 16][warp * 4 + c % 8 / 2][c % 16 / 8] = take_pair(a, b, C{});
      }
      if (lane == 0) factors[warp] = fmaxf(p.scale * inverse, 0x1p-126f);
    }
    named_bar(1, kPagedWarps * 32);
    stopped |= __any_sync(~0u, *(volatile uint32_t *)&gave_up);
    uint32_t qf[kQ][kSteps][2];
#pragma unroll
    for (int k = 0; k < kQ; ++k)
#pragma unroll
      for (int i = 0; i < kSteps; ++i) *(uint2 *)qf[k][i] = *(const uint2 *)q_frag[k][i][lane];
    const float f0 = factors[2 * t], f1 = factors[2 * t + 1];   // scores of heads 2t and 2t + 1 are this lane's

    float o[kSteps][4], all_o[kFresh ? kSteps : 1][4], m0 = kNoScore, m1 = kNoScore, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    if constexpr (kFresh) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) all_o[j][0] = all_o[j][1] = all_o[j][2] = all_o[j][3] = 0.f;
    }
    uint32_t steps = 0;    // steps that this warp took
    const uint32_t rounds = (seg.blocks + kPagedWarps - 1) / kPagedWarps;
#pragma unroll 1
    for (uint32_t r = 0; r < rounds; ++r, ++round) {
      const uint32_t stage = round % S::kStages;
      if (!stopped && !__all_sync(~0u, mbar_wait_bounded(&full[warp][stage], round / S::kStages & 1))) {
        stopped = true;
        if (lane == 0) *(volatile uint32_t *)&gave_up = 1;
      }
      const uint32_t valid = stopped ? 0 : valid_rows[warp][stage];
      if (valid) {
        ++steps;
        const uint32_t st = my_ring + stage * S::kStage;
        // ---- scores ----
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t a[4];
          const uint32_t chunk = (k % 4) * 2 + k_chunk;
          ldmatrix4(a, st + k / 4 * S::kHalf + k_row * 128 + ((chunk ^ (k_row & 7)) << 4));
#pragma unroll
          for (int i = 0; i < kQ; ++i) mma_16(c, a, qf[i][k], C{});
        }
        // ---- softmax: c[2y + z] is cache row 8y + g, head 2t + z ----
        const bool tail = valid < kPagedBlock;
        if (tail) {   // rows past the last that is seen hold anything
          if (g >= valid) c[0] = c[1] = -INFINITY;
          if (g + 8 >= valid) c[2] = c[3] = -INFINITY;
        }
        float top0 = fmaxf(c[0], c[2]), top1 = fmaxf(c[1], c[3]);
        if (__any_sync(~0u, (top0 - m0) * f0 > kLead || (top1 - m1) * f1 > kLead)) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) {
            top0 = fmaxf(top0, __shfl_xor_sync(~0u, top0, x));
            top1 = fmaxf(top1, __shfl_xor_sync(~0u, top1, x));
          }
          top0 = fmaxf(top0, m0), top1 = fmaxf(top1, m1);
          const float r0 = exp2_fast((m0 - top0) * f0), r1 = exp2_fast((m1 - top1) * f1);
          m0 = top0, m1 = top1;
          l0 *= r0, l1 *= r1;
#pragma unroll
          for (int j = 0; j < kSteps; ++j) o[j][0] *= r0, o[j][1] *= r1, o[j][2] *= r0, o[j][3] *= r1;
          if constexpr (kFresh) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) all_o[j][0] *= r0, all_o[j][1] *= r1, all_o[j][2] *= r0, all_o[j][3] *= r1;
          }
        }
        uint32_t pf[kP][2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float x0 = exp2_fast(fmaf(c[2 * y] - m0, f0, kPagedPScale<C>)), x1 = exp2_fast(fmaf(c[2 * y + 1] - m1, f1, kPagedPScale<C>));
          l0 += x0, l1 += x1;
#pragma unroll
          for (int k = 0; k < kP; ++k) pf[k][y] = transpose8(take_pair(x0, x1, C{}));
        }
        // ---- values: m-tile j is channels 16 j + g and 16 j + 8 + g ----
        uint32_t keep[2] = {~0u, ~0u};   // of rows 2t, 2t + 1 and 2t + 8, 2t + 9
        if (tail) {
#pragma unroll
          for (uint32_t y = 0; y < 2; ++y)
            keep[y] = (8 * y + 2 * t < valid ? 0xFFFFu : 0u) | (8 * y + 2 * t + 1 < valid ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          uint32_t a[4];
          const uint32_t chunk = (j % 4) * 2 + v_chunk;
          ldmatrix4_trans(a, st + j / 4 * S::kHalf + kPagedBlock * 128 + v_row * 128 + ((chunk ^ (v_row & 7)) << 4));
          if (tail) a[0] &= keep[0], a[1] &= keep[0], a[2] &= keep[1], a[3] &= keep[1];
#pragma unroll
          for (int k = 0; k < kP; ++k) mma_16(o[j], a, pf[k], C{});
        }
        if constexpr (kFresh) {
          if (steps % kFreshSteps == 0) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
#pragma unroll
              for (int y = 0; y < 4; ++y) all_o[j][y] += o[j][y], o[j][y] = 0.f;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[warp][stage]);
    }
    if constexpr (kFresh) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[j][y] += all_o[j][y];
    }

    // ---- the warps' results meet ----
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(~0u, l0, x);
      l1 += __shfl_xor_sync(~0u, l1, x);
    }
    m0 = l0 == 0.f ? kNoScore : m0 * f0, m1 = l1 == 0.f ? kNoScore : m1 * f1;   // scaled from here on
    // a denominator of 0 where rows were seen (every score -infinity) is marked by a -1
    if (steps && l0 == 0.f) l0 = -1.f;
    if (steps && l1 == 0.f) l1 = -1.f;
    if (g == 0) {
      *(float2 *)&w_max[warp][2 * t] = make_float2(m0, m1);
      *(float2 *)&w_sum[warp][2 * t] = make_float2(l0, l1);
    }
    named_bar(1, kPagedWarps * 32);
    float top0 = kNoScore, top1 = kNoScore;
#pragma unroll
    for (uint32_t w = 0; w < kPagedWarps; ++w) {
      const float2 x = *(const float2 *)&w_max[w][2 * t];
      top0 = fmaxf(top0, x.x), top1 = fmaxf(top1, x.y);
    }
    const float e0 = exp2_fast(m0 - top0), e1 = exp2_fast(m1 - top1);
    if (warp == 0 && g < 2) {   // lanes of g = 0 and 1: the denominators of heads 2t and 2t + 1
      const float top = g ? top1 : top0;
      float all = 0.f;
      bool seen = false;
#pragma unroll
      for (uint32_t w = 0; w < kPagedWarps; ++w) {
        const float x = w_sum[w][2 * t + g];
        seen |= x < 0.f;
        all += (x < 0.f ? 0.f : x) * exp2_fast(w_max[w][2 * t + g] - top);
      }
      f_max[2 * t + g] = top;
      f_sum[2 * t + g] = all == 0.f && seen ? -1.f : all;
    }
    float *part = p.parts + (size_t)index * kPart<D>;
    T *out = (T *)p.out + ((size_t)seg.query * p.heads + kv * p.group + head0) * D;
    const auto inverse_of = [](float sum) {   // zeros where no row was seen, NaN where every score was -infinity
      return sum == 0.f ? 0.f : sum < 0.f ? NAN : 1.f / sum;
    };
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {   // 64 channels at a time
      if (h) named_bar(1, kPagedWarps * 32);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * h + i;
        float *dst = merge + (warp * kPagedHeads + 2 * t) * S::kRow + 16 * i + g;
        dst[0] = e0 * o[j][0], dst[8] = e0 * o[j][2];
        dst[S::kRow] = e1 * o[j][1], dst[S::kRow + 8] = e1 * o[j][3];
      }
      named_bar(1, kPagedWarps * 32);
      if (warp < tile_heads) {   // a warp a head, two channels a lane
        float2 x = make_float2(0.f, 0.f);
#pragma unroll
        for (uint32_t w = 0; w < kPagedWarps; ++w) {
          const float2 y = *(const float2 *)(merge + (w * kPagedHeads + warp) * S::kRow + 2 * lane);
          x.x += y.x, x.y += y.y;
        }
        const uint32_t ch = 64 * h + 2 * lane;
        if (whole) {
          const float inv = inverse_of(f_sum[warp]);
          T *dst = out + warp * D + ch;
          dst[0] = from_float<T>(x.x * inv), dst[1] = from_float<T>(x.y * inv);
        } else {
          *(float2 *)(part + warp * D + ch) = x;
        }
      }
    }
    if (!whole) {
      if (threadIdx.x < tile_heads) {
        part[kPagedHeads * D + threadIdx.x] = f_max[threadIdx.x];
        part[kPagedHeads * (D + 1) + threadIdx.x] = f_sum[threadIdx.x];
      }
      named_bar(1, kPagedWarps * 32);
      const uint32_t pieces = seg.parts;
      const float *others = p.parts + (size_t)(index - seg.part) * kPart<D>;
      uint32_t *ticket = p.tickets + seg.query * plan.lanes + seg.lane;
      if (threadIdx.x == 0) last = atomic_add_acq_rel(ticket, 1u) == pieces - 1;
      named_bar(1, kPagedWarps * 32);
      if (last) {
        if (threadIdx.x == 0) *ticket = 0;
        float *weight = merge;   // [pieces][kPagedHeads]
        const auto piece = [&](uint32_t i) { return others + (size_t)i * kPart<D>; };
        if (warp < tile_heads) {   // a warp a head, its lanes the pieces
          float top = kNoScore, all = 0.f;
          bool seen = false;
#pragma unroll 1
          for (uint32_t i = lane; i < pieces; i += 32) {
            const float m = __ldcg(piece(i) + kPagedHeads * D + warp);
            weight[i * kPagedHeads + warp] = m;
            top = fmaxf(top, m);
          }
#pragma unroll
          for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
#pragma unroll 1
          for (uint32_t i = lane; i < pieces; i += 32) {
            const float sum = __ldcg(piece(i) + kPagedHeads * (D + 1) + warp);
            const float w = exp2_fast(weight[i * kPagedHeads + warp] - top);
            seen |= sum < 0.f;
            all += w * (sum < 0.f ? 0.f : sum);
            weight[i * kPagedHeads + warp] = w;
          }
#pragma unroll
          for (int x = 16; x; x >>= 1) all += __shfl_xor_sync(~0u, all, x);
          seen = __any_sync(~0u, seen);
          const float inv = inverse_of(all == 0.f && seen ? -1.f : all);
          __syncwarp();
          constexpr uint32_t N = D / 32;   // channels of a lane
          float x[N];
#pragma unroll
          for (uint32_t k = 0; k < N; ++k) x[k] = 0.f;
#pragma unroll 16
          for (uint32_t i = 0; i < pieces; ++i) {
            const float w = weight[i * kPagedHeads + warp];
            const float *src = piece(i) + warp * D + lane * N;
            if constexpr (N == 4) {
              const float4 y = __ldcg((const float4 *)src);
              x[0] = fmaf(w, y.x, x[0]), x[1] = fmaf(w, y.y, x[1]), x[2] = fmaf(w, y.z, x[2]), x[3] = fmaf(w, y.w, x[3]);
            } else {
              const float2 y = __ldcg((const float2 *)src);
              x[0] = fmaf(w, y.x, x[0]), x[1] = fmaf(w, y.y, x[1]);
            }
          }
#pragma unroll
          for (uint32_t k = 0; k < N; ++k) out[warp * D + lane * N + k] = from_float<T>(x[k] * inv);
        }
      }
    }
    named_bar(1, kPagedWarps * 32);   // shared results are free for the next piece
  }
  if (stopped) {   // copies in flight land before the block ends
    for (uint32_t i = round - min(round, S::kStages); i < round; ++i)
      mbar_wait_bounded(&full[warp][i % S::kStages], i / S::kStages & 1);
    if (lane == 0) atomicOr(&p.t.pool[1], kPagedTimeout);
  }
}

}  // namespace vg
