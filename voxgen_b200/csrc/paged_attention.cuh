// Attention of single tokens over a paged cache, over all of a sequence's pages or
// over a list of them, split over the length and joined.
//
// The mathematics. Up to 8 query heads of a KV head are the columns of m16n8k16
// MMAs: scores S^T = K Q^T and the output O^T = V^T P^T, cache rows as the A
// operand. q is held in as many terms of the cache's type as its bits need (fp32:
// two of fp16, three of bf16), and P in two of fp16 or three of bf16; so products are
// as exact as fp32's. Statistics and sums are fp32. The tensor cores add with rounding
// towards zero, so O is summed afresh every 8 steps (fp32 queries) or 32 (others, where
// a warp's steps may be many) and added with rounding to nearest.
//
// The bound is bytes: 4 D of them a row for 4 D multiply-adds a head. So one warp
// does nothing but keep copies in flight: it looks page numbers up 24 at a time and
// issues tensor copies of 16 rows (K and V; 8 KB at head_dim 128) into a ring of 192
// KB, through 128-byte swizzled boxes that ldmatrix reads without bank conflicts.
//
// A tile is (query, 8 heads of a KV head), a warp's work. Up to 4 tiles that read the
// same rows make a segment: the tiles of more than 8 heads to a KV head, or consecutive
// queries of one sequence (a draft's tokens). A block of 16 rows is then read once for
// the T tiles, and the 12 consumer warps are 12 / T teams that take blocks in turn.
// Tiles never mix queries, so a row that one query sees and another does not is masked
// warp by warp, whatever it holds. A warp's step of 16 rows is one chain of dependent
// instructions (copies awaited, products, maximum, exponentials, transposes, products),
// so as many warps run as registers allow: 12 at 128 each (at head_dim 128 most kernels
// spill 8 to 44 bytes, fp32 queries over bf16 96), with q's terms read from shared memory.
//
// The split. Segments are cut into pieces of at most U blocks, U such that there is
// about one piece for each CTA (up to 4, where segments are many). The warps of a piece
// meet in shared memory. A segment of several pieces leaves a partial result for each, and
// the CTA that finishes last (a counter, left at zero) adds them in order: sums never
// depend on timing.
//
// Measured: 16 contexts of 24001 to 32768 rows, bf16, 465 MB: 77 us, 6.0 TB/s (93% of
// the measured copy rate). 16 ragged streams of 64 to 4096 rows, 34 MB: 13.7 us, of
// which 4 stream: the rest is code that runs once, at about 7 cycles an instruction, and
// so kept short (loops, not unrolled ones). 5 drafted tokens of those streams: 30 us.
#pragma once
#include <cuda.h>

#include <type_traits>

#include "kv4_rows_attention.cuh"
#include "paged.cuh"
#include "paged_mma.cuh"

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
  uint32_t queries, heads, group;
  uint32_t share;            // consecutive queries of a sequence share what they read
  uint32_t tiles;            // most tiles of a segment (a power of two); of each segment, where queries do not share
  uint32_t lanes;            // segments of a query
  float scale;               // of the scores, times log2(e)
  uint32_t *tickets;         // [queries * lanes], zero between calls
  float *parts;              // [pieces of cut segments][tiles] partial results
};

constexpr uint32_t kPagedBlock = 16;     // cache rows of a block: never more than one page's
// Consumer warps of a CTA: 12 in one CTA an SM, or 4 in each of two, where segments are many: while the warps of one CTA
// meet or load the next queries, those of the other go on.
constexpr uint32_t kPagedWarps = 12, kPagedFew = 4;
// Segments from which on a CTA has 4 warps. Sequences of 200 to 500 rows, 2 KV heads: 200 of them take 27 us with 12 warps and
// 28 with 4, 256 take 34 and 30, 1024 take 120 and 94.
constexpr uint32_t kPagedMany = 444;
constexpr uint32_t paged_ctas(uint32_t warps) { return 148 * (warps == kPagedWarps ? 1 : 2); }   // resident at once
constexpr uint32_t kPagedHeads = 8;      // columns of a tile
constexpr uint32_t kPagedTiles = 4;      // most tiles of a segment
constexpr uint32_t kPagedWhole = 48;     // blocks of a segment that is not cut: joining takes as long as five rounds
constexpr uint32_t kPagedTickets = 1u << 14;   // segments that may be cut
constexpr uint32_t paged_planned(uint32_t warps) { return warps == kPagedWarps ? 256 : 1024; }   // queries whose place in the plan is kept
constexpr uint32_t kPagedMost = 1u << 26;      // blocks of a segment
constexpr uint32_t kPagedUncut = ~0u;          // the size of pieces that are whole segments

template <int D, int W, int Q>   // W: consumer warps, Q: terms of a query
struct PagedSmem {
  static constexpr uint32_t kHalf = 2 * kPagedBlock * 128;     // one copy: 64 channels of 16 K rows, then of 16 V rows
  static constexpr uint32_t kStage = kHalf * (D / 64);
  static constexpr uint32_t kStages = 2 * W * 128 / D;
  // A warp that waits for a stage's next turn has to have waited for the one before (a wait for the turn after one in
  // flight returns at once): so within a piece a stage is always the same team's, and pieces take whole rounds of stages.
  static_assert(kStages % W == 0, "");
  static constexpr uint32_t kRing = kStages * kStage;
  static constexpr uint32_t kRow = 68;                         // floats of a row when results meet: 64 and 4 against bank conflicts
  static constexpr uint32_t kMerge = W * kPagedHeads * kRow * 4;
  static constexpr uint32_t kTileQ = D / 16 * 32 * 8;          // a tile's queries as B fragments, one term
  static constexpr uint32_t kShared = kMerge > Q * kPagedTiles * kTileQ ? kMerge : Q * kPagedTiles * kTileQ;   // first queries, then results
  static constexpr uint32_t kBytes = kRing + kShared + 1024;   // the ring starts on a multiple of 1024
};

// Pieces that a call is cut into, about: one for each CTA, or up to 4, so that there are a third more than segments. And the
// partial results that it may leave: a segment that is cut at all has fewer than twice its share of the target in pieces.
__host__ __device__ __forceinline__ uint32_t paged_target(uint32_t segments, uint32_t ctas) {
  const uint32_t rounds = (segments * 4 + ctas * 3 - 1) / (ctas * 3);   // segments: no more than kPagedTickets
  return ctas * (rounds < 1 ? 1 : rounds > 4 ? 4 : rounds);
}
__host__ __device__ __forceinline__ uint32_t paged_slots(uint64_t segments, uint32_t ctas) {
  return segments > kPagedTickets ? 0 : 2 * paged_target((uint32_t)segments, ctas);
}

// What the plan needs to know of a query. entry: blocks and tiles of the segments that it leads, blocks << 2 |
// log2(tiles), at least one block, so that every output is written; 0 where another query leads. Queries share within
// aligned eights, in runs of 1, 2 or 4. seen: rows that it sees, most: that any query of its segments sees.
struct PagedLead {
  uint32_t entry, seq, seen, most;
};
__device__ __forceinline__ PagedLead paged_lead(const PagedAttnParams &p, uint32_t i) {
  const auto entry = [&](uint32_t rows, uint32_t tiles) {
    return max(1u, (rows + kPagedBlock - 1) / kPagedBlock) << 2 | (31 - __clz(tiles));
  };
  if (!p.share) {
    const PagedSeen who = paged_seen(p.t, p.which, i);
    const uint32_t e = p.chosen ? entry(p.budget << p.t.shift, p.tiles) : entry(who.seen, p.tiles);
    return {e, who.seq, who.seen, who.seen};
  }
  const uint32_t from = i & ~7u;
  int32_t seqs[8], last[8];
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) {
    const uint32_t k = min(from + j, p.queries - 1);
    seqs[j] = p.which.sequences[k];
    last[j] = p.which.positions ? p.which.positions[k] : 0x7FFFFFFE;
  }
  const uint32_t at = i - from;
  int32_t mine = 0, here = 0;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (j == at) mine = seqs[j], here = last[j];
  uint32_t same = 0;   // of the eight
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (from + j < p.queries && seqs[j] == mine) same |= 1u << j;
  const uint32_t start = 32 - __clz(~same & ((1u << at) - 1)), end = __ffs(~same >> at) - 1 + at;   // of the run around i
  uint32_t first = start, size = 4;                  // of the part of the run that i is in
  while (at >= first + size || first + size > end) {
    if (first + size <= end) first += size;
    else size /= 2;
  }
  int32_t top = here;
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (j >= first && j < first + size) top = max(top, last[j]);
  const PagedSeen all = (uint32_t)mine < p.t.seqs ? PagedSeen{(uint32_t)mine, paged_held(p.t, mine)} : PagedSeen{0, 0};
  const auto seen = [&](int32_t x) { return min(all.seen, (uint32_t)max(x, -1) + 1u); };
  return {at == first ? entry(seen(top), size) : 0, all.seq, seen(here), seen(top)};
}
// A little more than a / b.
__device__ __forceinline__ uint32_t paged_over(uint32_t a, uint32_t b) {
  return (uint32_t)((float)a * __fdividef(1.f + 0x1p-20f, (float)b)) + 1;
}
// What a segment's block costs, in quarters: one tile is bound by the block's bytes, four by their arithmetic.
__device__ __forceinline__ uint32_t paged_weight(uint32_t entry) { return (entry & 3) == 0 ? 4 : (entry & 3) == 1 ? 6 : 10; }
__device__ __forceinline__ uint32_t paged_size(uint32_t entry, uint32_t size) {   // blocks of a piece that costs `size`
  if (size == kPagedUncut) return kPagedMost;
  return (entry & 3) == 0 ? min(size, kPagedMost) : (entry & 3) == 1 ? (2 * size + 2) / 3 : (2 * size + 4) / 5;
}
__device__ __forceinline__ uint32_t paged_parts(uint32_t entry, uint32_t size) {   // pieces of a segment
  const uint32_t b = entry >> 2, each = paged_size(entry, size);
  if (b * paged_weight(entry) <= kPagedWhole * 4) return entry != 0;
  uint32_t n = (uint32_t)((float)b * __fdividef(1.f - 0x1p-20f, (float)each));   // a little low
  n += n * each < b;
  while (n * each < b) ++n;   // millions of blocks
  return n;
}

// How segments are cut: pieces that cost at most `size`, `pieces` of them.
struct PagedPlan {
  uint32_t size, pieces;
};
struct PagedTally {   // in shared memory, zero before
  uint32_t total, leads, pieces[8];
};
// All threads: leads[] of the first queries, and the plan.
template <uint32_t N>
__device__ __forceinline__ PagedPlan paged_plan(const PagedAttnParams &p, PagedLead (&leads)[N], PagedTally &tally) {
  const uint32_t lane = threadIdx.x % 32;
  uint32_t total = 0, count = 0;
#pragma unroll 1
  for (uint32_t i = threadIdx.x; i < p.queries; i += blockDim.x) {
    const PagedLead x = paged_lead(p, i);
    if (i < N) leads[i] = x;
    total += ((x.entry >> 2) * paged_weight(x.entry) + 3) / 4;
    count += x.entry != 0;
  }
  total = __reduce_add_sync(~0u, total), count = __reduce_add_sync(~0u, count);
  if (lane == 0 && total) atomicAdd(&tally.total, total), atomicAdd(&tally.leads, count);
  __syncthreads();
  total = tally.total * p.lanes;   // the host keeps it below 2^31
  const uint32_t segments = tally.leads * p.lanes;
  if (p.queries * p.lanes > kPagedTickets) return PagedPlan{kPagedUncut, segments};   // one piece a segment
  const uint32_t target = paged_target(segments, gridDim.x);
  // total / target would do if nothing were rounded up; total / (target - segments) makes no more than target pieces. Of eight
  // sizes from the one to the other the least with no more pieces than the target is taken. Where there are more segments
  // than that, it is the first.
  const uint32_t least = max(blockDim.x / 32 - 1, paged_over(total, target));   // a round of the warps
  const uint32_t more = target > segments ? max(least, paged_over(total, target - segments)) - least : 0;
  const uint32_t k = lane / 4, size = least + (k == 7 ? more : more * k * k / 49);
  uint32_t n = 0;
#pragma unroll 1
  for (uint32_t i = threadIdx.x / 32 * 4 + lane % 4; i < p.queries; i += blockDim.x / 8)
    n += paged_parts(i < N ? leads[i].entry : paged_lead(p, i).entry, size);
  if (n) atomicAdd(&tally.pieces[k], n);
  __syncthreads();
  n = tally.pieces[k] * p.lanes;
  const int found = __ffs(__ballot_sync(~0u, n <= target) | 1u << 31) - 1;
  return PagedPlan{__shfl_sync(~0u, size, found), __shfl_sync(~0u, n, found)};
}

struct PagedPiece {
  uint32_t query, lane;         // lane: (KV head, 4 of its tiles)
  uint32_t part, parts;         // of the segment
  uint32_t slot;                // of the segment's first partial result
  uint32_t first, blocks;       // of the piece, in the segment
  uint32_t tiles;               // 1, 2 or 4
  uint32_t seq, seen;           // of the segment
};
// Where the search for a CTA's next piece goes on: 32 queries, and the pieces (all, and those of cut segments) before them.
struct PagedCursor {
  uint32_t base, before, cut;
};
template <typename E>
__device__ __forceinline__ PagedPiece paged_piece(const PagedAttnParams &p, const PagedPlan &x, uint32_t index, const E &lead,
                                                  PagedCursor &at32) {
  const uint32_t lane = threadIdx.x % 32;
#pragma unroll 1
  for (; at32.base < p.queries; at32.base += 32) {
    const uint32_t base = at32.base, before = at32.before, cut_before = at32.cut;
    const PagedLead who = base + lane < p.queries ? lead(base + lane) : PagedLead{0, 0, 0, 0};
    const uint32_t e = who.entry, n = paged_parts(e, x.size);
    uint32_t sum = n * p.lanes, cut = n > 1 ? sum : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o), more = __shfl_up_sync(~0u, cut, o);
      if (lane >= (uint32_t)o) sum += up, cut += more;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > index);
    if (past) {
      const int at = __ffs(past) - 1;
      const uint32_t parts = __shfl_sync(~0u, n, at), all = __shfl_sync(~0u, e, at);
      const uint32_t into = index - before - (__shfl_sync(~0u, sum, at) - parts * p.lanes);
      const uint32_t size = paged_size(all, x.size);
      PagedPiece y;
      y.query = base + at;
      y.lane = (uint32_t)__fdividef((float)into + 0.5f, (float)parts);   // exact: below 2^22
      y.part = into - y.lane * parts;
      y.parts = parts;
      y.slot = cut_before + __shfl_sync(~0u, cut, at) - parts * p.lanes + y.lane * parts;
      y.first = y.part * size;
      y.blocks = parts == 1 ? all >> 2 : min(size, (all >> 2) - y.first);
      y.tiles = 1u << (all & 3);
      y.seq = __shfl_sync(~0u, who.seq, at);
      y.seen = __shfl_sync(~0u, who.most, at);
      return y;
    }
    at32.before += __shfl_sync(~0u, sum, 31);
    at32.cut += __shfl_sync(~0u, cut, 31);
  }
  return PagedPiece{0, 0, 0, 1, 0, 0, 0, 1, 0, 0};   // past the last piece
}

// Stages that a piece takes.
template <uint32_t W>
__device__ __forceinline__ uint32_t paged_rounds(uint32_t blocks) { return (blocks + W - 1) / W * W; }

// Volatile keeps these behind the wait for their stage and before its release; products may move among them.
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address));
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
// P is held to 32 bits' precision whatever the output's type: rounded to nearest, two terms of fp16 leave 2^-24 of it, three of
// bf16 2^-26 (two would leave 2^-17, which shows where values cancel). Measured: no time, on 16 contexts of 24001 to 32768 rows in
// bf16 (77.3 us, 77.4 with two) or 4096 chosen rows of each (20.8 us with either).
template <typename C>
constexpr int kPTerms = std::is_same<C, __half>::value ? 2 : 3;
// Products that a warp adds to O for 16-bit queries before it has to be summed afresh: each is cut by 2^-24 of the sum on
// average, 2^-15 for all of them, where an fp16 output is rounded by up to 2^-12. (One warp that added 131072 rows left 2^-13 of
// sum(p |v|).) Kernels that sum afresh take as long for long contexts (16 of 32768 rows 76.9 us, 77.2 without), but for drafts
// of 5 tokens 31.4 us, 30.1 without, and for 64 tokens of 16 streams 396, 374 without: so where no context is that long they
// are not taken.
constexpr uint32_t kPagedProducts = 512;

// P is held times 2^6 in fp16, for the range below a weight of 1 (kv4_rows_attention.cuh), and times 2^-20 in bf16: there V goes
// up to fp32's largest number (an infinity is held as that), and sums of P V over a million rows must not pass it. At the other
// end outputs below 2^-104 lose bits, as products become subnormal (2^-32 would cost those below 2^-92).
template <typename C>
constexpr float kPagedPScale = std::is_same<C, __half>::value ? kPScale : -20.f;
// A power of two for a head's query whose largest magnitude is `top`. fp16's range is met by one that brings it to [2^14, 2^15).
// bf16 has fp32's range, and so do K's infinities, held as the largest number: no more than 2^-8, and no sum of 128
// products passes that number.
__device__ __forceinline__ float query_power(float top, float &inverse, __half) { return row_power(top, inverse); }
__device__ __forceinline__ float query_power(float top, float &inverse, __nv_bfloat16) {
  const int e = (int)(__float_as_uint(top) >> 23 & 255) - 127, k = min(max(-9 - e, -114), 0);
  inverse = __uint_as_float((uint32_t)(127 - k) << 23);
  return __uint_as_float((uint32_t)(127 + k) << 23);
}

template <int D, typename T, typename C, int W, bool kFresh>   // kFresh: O is summed afresh
__global__ void __launch_bounds__((W + 1) * 32, W == kPagedWarps ? 1 : 2)
    paged_attention_kernel(const __grid_constant__ PagedAttnParams p, const __grid_constant__ CUtensorMap map) {
  constexpr int kSteps = D / 16;                // k-steps of a score, and m-tiles of the output
  constexpr int kQ = kQTerms<T, C>, kP = kPTerms<C>;
  using S = PagedSmem<D, W, kQ>;
  constexpr uint32_t kLook = 32 / W * W;        // blocks whose pages are looked up at once
  constexpr uint32_t kFreshSteps = sizeof(T) == 4 ? 8 : 32;
  extern __shared__ __align__(128) uint8_t paged_smem[];
  __shared__ uint64_t full[S::kStages], empty[S::kStages];
  __shared__ uint32_t first_row[S::kStages];    // of a stage's block in its sequence; past every row: nothing was read
  __shared__ PagedLead leads[paged_planned(W)];
  __shared__ PagedTally tally;
  __shared__ __align__(8) float w_max[(uint32_t)W][kPagedHeads], w_sum[(uint32_t)W][kPagedHeads];
  __shared__ float f_max[kPagedTiles][kPagedHeads], f_sum[kPagedTiles][kPagedHeads];   // [tile][head]
  __shared__ __align__(8) float factors[kPagedTiles][kPagedHeads];                    // [tile][head]
  __shared__ uint32_t last, gave_up;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const uint32_t base = smem_u32(paged_smem), ring = (base + 1023) & ~1023u;
  float *merge = (float *)(paged_smem + (ring - base) + S::kRing);   // [warp][head][kRow]
  uint32_t *q_frag = (uint32_t *)merge;
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map));
    gave_up = 0;
  }
  if (threadIdx.x < S::kStages) mbar_init(&full[threadIdx.x], 1), mbar_init(&empty[threadIdx.x], (uint32_t)W);
  if (threadIdx.x < sizeof(PagedTally) / 4) ((uint32_t *)&tally)[threadIdx.x] = 0;
  fence_mbar_init();
  __syncthreads();
  pdl_wait();   // and no early start for what comes next: a selection would hold SMs that this call still needs (69 us for
                // both among 8192 pages of 16 sequences, 77 with it; one short call after another takes 8.2 us, 7.8 with it)
  const PagedPlan plan = paged_plan(p, leads, tally);
  const auto lead = [&](uint32_t i) { return i < paged_planned(W) ? leads[i] : paged_lead(p, i); };
  if (blockIdx.x >= plan.pieces) return;
  PagedCursor cursor{};
  PagedPiece piece = paged_piece(p, plan, blockIdx.x, lead, cursor);   // most CTAs have one: what runs once is short

  if (warp == (uint32_t)W) {
    // ================= the copying warp =================
    uint32_t n0 = 0;           // blocks of the pieces before
    uint32_t issued = lane;    // the number after the last that this lane issued: it issues lane, lane + W, ...
    bool stopped = false;
#pragma unroll 1
    for (uint32_t index = blockIdx.x; !stopped;) {
      const PagedPiece x = piece;
      const uint32_t kv = p.share ? x.lane : x.lane / (p.lanes / p.kv_heads), page_rows = p.t.page_rows();
      const int32_t *table = p.t.table + (size_t)x.seq * p.t.seq_pages;
      const int32_t *list = p.chosen ? p.chosen + ((size_t)x.query * p.kv_heads + kv) * p.budget : nullptr;
      // page and first row of the piece's block i
      struct Found {
        uint32_t page, row;
      };
      const auto find = [&](uint32_t i) -> Found {
        const Found none{~0u, ~0u};
        if (i >= x.blocks) return none;
        const uint32_t row = (x.first + i) * kPagedBlock, e = row >> p.t.shift, in = row & (page_rows - 1);
        const uint32_t at = list ? (uint32_t)list[e] : e;
        if (at >= p.t.seq_pages) return none;
        const uint32_t first = (at << p.t.shift) + in;
        if (first >= x.seen) return none;
        const uint32_t page = (uint32_t)table[at];
        return page < p.t.pages ? Found{page, first} : none;
      };
      Found next = find(lane);
#pragma unroll 1
      for (uint32_t i = 0; i < x.blocks && !stopped; i += kLook) {
        const Found now = next;
        next = find(i + kLook + lane);
#pragma unroll 1
        for (uint32_t j = 0; j < kLook && i + j < x.blocks; j += W) {   // whole rounds: stages past the last block hold nothing
          const uint32_t from = j + lane % W;
          const uint32_t page = __shfl_sync(~0u, now.page, from), row = __shfl_sync(~0u, now.row, from);
          bool in = true;
          if (lane < (uint32_t)W) {
            const uint32_t n = n0 + i + j + lane, stage = n % S::kStages, turn = n / S::kStages;
            if (turn) in = mbar_wait_bounded(&empty[stage], (turn - 1) & 1);
            if (in) {
              issued = n + W;
              first_row[stage] = row;
              uint64_t *bar = &full[stage];
              if (row != ~0u) {
                mbar_arrive_expect_tx(bar, S::kStage);
                const int32_t place = (int32_t)(page * p.kv_heads + kv);
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
                  tensor_g2s(ring + stage * S::kStage + h * S::kHalf, &map, h * 64, (int32_t)(row & (page_rows - 1)), place, bar);
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
      n0 += paged_rounds<W>(x.blocks);
      if ((index += gridDim.x) >= plan.pieces) break;
      piece = paged_piece(p, plan, index, lead, cursor);
    }
    // The block does not end before its copies have landed. A stage is issued again only after all W arrivals of those who saw its
    // turn land, so at most the last turn of each of this lane's stages is in flight, whatever consumers do.
    bool landed = true;
    if (lane < (uint32_t)W) {
#pragma unroll 1
      for (uint32_t k = 1; k <= S::kStages / W && landed && issued >= k * W; ++k) {
        const uint32_t n = issued - k * W;
        landed = mbar_wait_bounded(&full[n % S::kStages], n / S::kStages & 1);
      }
    }
    if (!__all_sync(~0u, landed && !stopped) && lane == 0) atomicOr(&p.t.pool[1], kPagedTimeout);
    return;
  }

  // ================= the consumers =================
  uint32_t n0 = 0;
  bool stopped = false;      // a wait ran out: nothing is waited for or released any more, and the copying warp's next wait runs out
  // this lane's row of an ldmatrix, and which of the two 16-byte chunks it reads
  // (swizzled: chunk c of row r lies at c ^ r % 8; chunks 2i and 2i + 1 of step i are those of step 0, ^ 2i)
  const uint32_t k_row = lane % 8 + (lane / 8 % 2) * 8, k_at = k_row * 128 + ((lane / 16 ^ k_row % 8) << 4);
  const uint32_t v_row = lane % 8 + (lane / 16) * 8, v_at = kPagedBlock * 128 + v_row * 128 + ((lane / 8 % 2 ^ v_row % 8) << 4);
#pragma unroll 1
  for (uint32_t index = blockIdx.x;;) {
    const PagedPiece seg = piece;
    const bool whole = seg.parts == 1;
    const uint32_t chunks = p.lanes / p.kv_heads;   // segments of a KV head, where it has more than 4 tiles
    const uint32_t kv = p.share ? seg.lane : seg.lane / chunks;
    const uint32_t tile0 = p.share ? 0 : (seg.lane - kv * chunks) * kPagedTiles;
    const uint32_t teams = (uint32_t)W / seg.tiles, team = warp / seg.tiles, tile = warp & (seg.tiles - 1);
    // query and first head (of the KV head's) of a tile of the segment
    const auto query_of = [&](uint32_t k) { return p.share ? seg.query + k : seg.query; };
    const auto head_of = [&](uint32_t k) { return p.share ? 0 : (tile0 + k) * kPagedHeads; };
    const uint32_t head0 = head_of(tile);
    const uint32_t seen = p.share ? lead(query_of(tile)).seen : seg.seen;
    // ---- the queries as B fragments, a head a warp at a time: column `col` of a tile's MMA ----
#pragma unroll 1
    for (uint32_t r = warp; r < seg.tiles * kPagedHeads; r += (uint32_t)W) {
      constexpr uint32_t N = D / 32;
      const uint32_t k = r / kPagedHeads, col = r % kPagedHeads, head = head_of(k) + col;
      const T *q = (const T *)p.q + (int64_t)query_of(k) * p.q_query + (int64_t)(kv * p.group + head) * p.q_head + lane * N;
      float x[N];
      uint32_t top = 0;
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        x[i] = head < p.group ? (float)q[i] : 0.f;
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
      }
      float inverse;
      const float power = query_power(__uint_as_float(__reduce_max_sync(~0u, top)), inverse, C{});
#pragma unroll
      for (uint32_t i = 0; i < N; i += 2) {   // channels c, c + 1: step c / 16, lane 4 col + c % 8 / 2, register c % 16 / 8
        const uint32_t c = lane * N + i;
        float a = x[i] * power, b = x[i + 1] * power;
#pragma unroll
        for (int j = 0; j < kQ; ++j)   // [tile][term][pair of steps][lane][step of the pair][register]
          q_frag[(((k * kQ + j) * (kSteps / 2) + c / 32) * 32 + col * 4 + c % 8 / 2) * 4 + c % 32 / 8] = take_pair(a, b, C{});
      }
      if (lane == 0) factors[k][col] = fmaxf(p.scale * inverse, 0x1p-126f);
    }
    named_bar(1, (uint32_t)W * 32);
    const uint32_t *my_q = q_frag + (tile * kQ * (kSteps / 2) * 32 + lane) * 4;
    const float f0 = factors[tile][2 * t], f1 = factors[tile][2 * t + 1];   // scores of heads 2t and 2t + 1 are this lane's
    stopped |= __any_sync(~0u, *(volatile uint32_t *)&gave_up);

    float o[kSteps][4], all_o[kFresh ? kSteps : 1][4], m0 = kNoScore, m1 = kNoScore, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    if constexpr (kFresh) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j) all_o[j][0] = all_o[j][1] = all_o[j][2] = all_o[j][3] = 0.f;
    }
    uint32_t steps = 0;    // steps that this warp took
    uint32_t stage = (n0 + team) % S::kStages, parity = (n0 + team) / S::kStages & 1;
#pragma unroll 1
    for (uint32_t b = team; b < paged_rounds<W>(seg.blocks); b += teams) {
      if (!stopped && !__all_sync(~0u, mbar_wait_bounded(&full[stage], parity))) {
        stopped = true;
        if (lane == 0) *(volatile uint32_t *)&gave_up = 1;
      }
      const uint32_t first = first_row[stage];
      if (!stopped && first < seen && head0 < p.group) {
        const uint32_t valid = seen - first;   // rows of the block that are seen, when below 16
        ++steps;
        const uint32_t st = ring + stage * S::kStage;
        // ---- scores ----
        // even and odd steps (and q's lower terms) in sums of their own: half the chain of dependent products
        float sums[kQ > 1 ? 3 : 2][4] = {};
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {   // 64 channels: four loads, then their products
          uint32_t a[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) ldmatrix4(a[k], (st + k_at + h * S::kHalf) ^ k << 5);
#pragma unroll
          for (int i = 0; i < kQ; ++i) {
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              const uint4 b = *(const uint4 *)(my_q + (i * (kSteps / 2) + 2 * h + k / 2) * 32 * 4);
              const uint32_t even[2] = {b.x, b.y}, odd[2] = {b.z, b.w};
              mma_16(sums[i ? 2 : 0], a[k], even, C{});
              mma_16(sums[i ? 2 : 1], a[k + 1], odd, C{});
            }
          }
        }
        float c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[i] = sums[0][i] + sums[1][i];
          if constexpr (kQ > 1) c[i] += sums[2][i];
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
        for (int h = 0; h < D / 64; ++h) {
          uint32_t a[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) ldmatrix4_trans(a[j], (st + v_at + h * S::kHalf) ^ j << 5);
          if (tail) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j][0] &= keep[0], a[j][1] &= keep[0], a[j][2] &= keep[1], a[j][3] &= keep[1];
          }
#pragma unroll
          for (int k = 0; k < kP; ++k) {
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_16(o[4 * h + j], a[j], pf[k], C{});
          }
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
      if (lane == 0 && !stopped) mbar_arrive_count(&empty[stage], teams);   // the team's T warps make up W arrivals
      stage += teams;
      if (stage >= S::kStages) stage -= S::kStages, parity ^= 1;
    }
    n0 += paged_rounds<W>(seg.blocks);
    if constexpr (kFresh) {
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[j][y] += all_o[j][y];
    }

    // ---- the teams' results meet, tile by tile ----
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(~0u, l0, x);
      l1 += __shfl_xor_sync(~0u, l1, x);
    }
    // maxima meet unscaled, as within a warp: a scaled one may pass fp32's range, and rounds by more than differences are
    if (l0 == 0.f) m0 = kNoScore;
    if (l1 == 0.f) m1 = kNoScore;
    // a denominator of 0 where rows were seen (every score -infinity) is marked by a -1
    if (steps && l0 == 0.f) l0 = -1.f;
    if (steps && l1 == 0.f) l1 = -1.f;
    if (g == 0) {
      *(float2 *)&w_max[warp][2 * t] = make_float2(m0, m1);
      *(float2 *)&w_sum[warp][2 * t] = make_float2(l0, l1);
    }
    named_bar(1, (uint32_t)W * 32);
    // lane (head, s) looks at every fourth warp from s on, of which those of this tile count
    float e0, e1;
    {
      const uint32_t h = lane / 4, s = lane % 4;
      const float f = factors[tile][h];
      float m[W / 4], l[W / 4], top = kNoScore, all = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < W / 4; ++i) {
        const uint32_t w = s + 4 * i;
        const bool mine = (w & (seg.tiles - 1)) == tile;
        m[i] = mine ? w_max[w][h] : kNoScore, l[i] = mine ? w_sum[w][h] : 0.f;
        top = fmaxf(top, m[i]);
      }
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      bool some = false;
#pragma unroll
      for (uint32_t i = 0; i < W / 4; ++i) {
        some |= l[i] < 0.f;
        all += (l[i] < 0.f ? 0.f : l[i]) * exp2_fast((m[i] - top) * f);
      }
      all += __shfl_xor_sync(~0u, all, 1);
      all += __shfl_xor_sync(~0u, all, 2);
      some = __ballot_sync(~0u, some) >> (lane & ~3u) & 15;
      if (team == 0 && s == 0) {
        f_max[tile][h] = top;
        f_sum[tile][h] = all == 0.f && some ? -1.f : all;
      }
      e0 = exp2_fast((m0 - __shfl_sync(~0u, top, 8 * t)) * f0), e1 = exp2_fast((m1 - __shfl_sync(~0u, top, 8 * t + 4)) * f1);
    }
    float *part = p.parts + (size_t)(seg.slot + seg.part) * p.tiles * kPart<D>;
    const auto out_of = [&](uint32_t k, uint32_t head) {   // of a tile's head
      return (T *)p.out + ((size_t)query_of(k) * p.heads + kv * p.group + head_of(k) + head) * D;
    };
    const auto inverse_of = [](float sum) {   // zeros where no row was seen, NaN where every score was -infinity
      return sum == 0.f ? 0.f : sum < 0.f ? NAN : 1.f / sum;
    };
#pragma unroll 1
    for (int h = 0; h < D / 64; ++h) {   // 64 channels at a time
      if (h) named_bar(1, (uint32_t)W * 32);
      const auto store = [&](const float(&x)[4], int i) {
        float *dst = merge + (warp * kPagedHeads + 2 * t) * S::kRow + 16 * i + g;
        dst[0] = e0 * x[0], dst[8] = e0 * x[2];
        dst[S::kRow] = e1 * x[1], dst[S::kRow + 8] = e1 * x[3];
      };
      if (D == 64 || h == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) store(o[i], i);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) store(o[kSteps - 4 + i], i);
      }
      named_bar(1, (uint32_t)W * 32);
#pragma unroll 1
      for (uint32_t r = warp; r < seg.tiles * kPagedHeads; r += (uint32_t)W) {   // a head a warp at a time, two channels a lane
        const uint32_t k = r / kPagedHeads, head = r % kPagedHeads;
        if (head_of(k) + head >= p.group) continue;
        float2 x = make_float2(0.f, 0.f);
        const float *src = merge + (k * kPagedHeads + head) * S::kRow + 2 * lane;
#pragma unroll 3
        for (uint32_t w = k; w < (uint32_t)W; w += seg.tiles, src += seg.tiles * kPagedHeads * S::kRow) {
          const float2 y = *(const float2 *)src;
          x.x += y.x, x.y += y.y;
        }
        const uint32_t ch = 64 * h + 2 * lane;
        if (whole) {
          const float inv = inverse_of(f_sum[k][head]);
          T *dst = out_of(k, head) + ch;
          dst[0] = from_float<T>(x.x * inv), dst[1] = from_float<T>(x.y * inv);
        } else {
          *(float2 *)(part + k * kPart<D> + head * D + ch) = x;
        }
      }
    }
    if (!whole) {
      if (threadIdx.x < seg.tiles * kPagedHeads) {
        float *dst = part + threadIdx.x / kPagedHeads * kPart<D> + kPagedHeads * D + threadIdx.x % kPagedHeads;
        dst[0] = f_max[0][threadIdx.x];
        dst[kPagedHeads] = f_sum[0][threadIdx.x];
      }
      named_bar(1, (uint32_t)W * 32);
      const uint32_t pieces = seg.parts;
      uint32_t *ticket = p.tickets + seg.query * p.lanes + seg.lane;
      if (threadIdx.x == 0) last = atomic_add_acq_rel(ticket, 1u) == pieces - 1;
      named_bar(1, (uint32_t)W * 32);
      if (last) {
        if (threadIdx.x == 0) *ticket = 0;
#pragma unroll 1
        for (uint32_t r = warp; r < seg.tiles * kPagedHeads; r += (uint32_t)W) {   // a head a warp at a time
          const uint32_t k = r / kPagedHeads, head = r % kPagedHeads;
          if (head_of(k) + head >= p.group) continue;
          constexpr uint32_t N = D / 32;   // channels of a lane
          constexpr uint32_t kAhead = 8;   // pieces whose values are loaded before their weights are known
          const float *from = p.parts + ((size_t)seg.slot * p.tiles + k) * kPart<D>;
          struct __align__(D / 8) Values {   // a lane's channels
            float x[N];
          };
          const size_t stride = (size_t)p.tiles * kPart<D>;
          const auto values = [&](uint32_t i) {
            const float *src = from + i * stride + head * D + lane * N;
            Values v;
            if constexpr (N == 4) *(float4 *)v.x = __ldcg((const float4 *)src);
            else *(float2 *)v.x = __ldcg((const float2 *)src);
            return v;
          };
          // lanes are pieces, 32 at a time
          const float f = factors[k][head];
          const float *stats = from + kPagedHeads * D + head;
          float m = lane < pieces ? __ldcg(stats + lane * stride) : kNoScore;
          float sum = lane < pieces ? __ldcg(stats + lane * stride + kPagedHeads) : 0.f;
          Values early[kAhead];
#pragma unroll
          for (uint32_t i = 0; i < kAhead; ++i) early[i] = values(min(i, pieces - 1));
          float top = m;
#pragma unroll 1
          for (uint32_t i = lane + 32; i < pieces; i += 32) top = fmaxf(top, __ldcg(stats + i * stride));
#pragma unroll
          for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
          float all = 0.f;
          bool some = false;
          Values x{};
#pragma unroll 1
          for (uint32_t at = 0; at < pieces; at += 32) {
            if (at) {
              const uint32_t i = at + lane;
              m = i < pieces ? __ldcg(stats + i * stride) : kNoScore;
              sum = i < pieces ? __ldcg(stats + i * stride + kPagedHeads) : 0.f;
            }
            const float w = exp2_fast((m - top) * f);
            some |= sum < 0.f;
            all += w * (sum < 0.f ? 0.f : sum);
            uint32_t i = 0;
            if (at == 0) {
#pragma unroll
              for (; i < kAhead; ++i) {
                const float wi = i < pieces ? __shfl_sync(~0u, w, i) : 0.f;
#pragma unroll
                for (uint32_t n = 0; n < N; ++n)
                  if (i < pieces) x.x[n] = fmaf(wi, early[i].x[n], x.x[n]);
              }
            }
            const uint32_t end = min(32u, pieces - at);
            constexpr uint32_t kTogether = 8;   // loads in flight; 16 take registers from the steps
#pragma unroll 1
            for (; i < end; i += kTogether) {
              Values v[kTogether];
#pragma unroll
              for (uint32_t u = 0; u < kTogether; ++u) v[u] = values(at + min(i + u, end - 1));
#pragma unroll
              for (uint32_t u = 0; u < kTogether; ++u) {
                const float wi = __shfl_sync(~0u, w, (i + u) & 31);
#pragma unroll
                for (uint32_t n = 0; n < N; ++n)
                  if (i + u < end) x.x[n] = fmaf(wi, v[u].x[n], x.x[n]);
              }
            }
          }
#pragma unroll
          for (int y = 16; y; y >>= 1) all += __shfl_xor_sync(~0u, all, y);
          const float inv = inverse_of(all == 0.f && __any_sync(~0u, some) ? -1.f : all);
          T *dst = out_of(k, head) + lane * N;
#pragma unroll
          for (uint32_t n = 0; n < N; ++n) dst[n] = from_float<T>(x.x[n] * inv);
        }
      }
    }
    if ((index += gridDim.x) >= plan.pieces) break;
    piece = paged_piece(p, plan, index, lead, cursor);
    named_bar(1, (uint32_t)W * 32);   // shared results are free for the next piece
  }
  if (stopped && lane == 0) atomicOr(&p.t.pool[1], kPagedTimeout);
}

}  // namespace vg
