// Attention of few query rows over a 4-bit cache: single tokens and short drafts.
//
// The mathematics. The query rows of a (sequence, KV head) are packed: row
// r = token * group + head of the group. A tile is 8 of them, the columns of an
// m16n8k16 MMA: scores are S^T = K Q^T and the output O^T = V^T P^T, with the
// cache as the A operand. Both K and V come out of the codes with one shift, one
// lop3 and one fused multiply-add a pair (kv4.cuh), exactly. fp32 queries are
// fp16 hi + lo, accumulated by a second MMA; 16-bit queries keep their bits in fp16
// (times a power of two a row; a bf16 value below 2^-28 of its row's largest is held
// to 2^-39 of that). P is hi + lo too, but for bf16, whose output keeps 8
// bits: rounded to fp16's 11 it would add as much error to an fp16 output as the
// output's own rounding. Softmax statistics and sums are fp32.
//
// The contraction over channels may run in any order as long as both operands
// agree, so lane (g, t) takes channels [t*D/4, (t+1)*D/4) of its K rows: one wide
// load, and at head_dim 128 one scale. An 8x8 transpose (movmatrix) turns the
// scores' C fragment into the B fragment of P^T. V needs pairs along rows: two
// byte permutes put the nibbles of two rows side by side. Row order within a
// tile is free too; kPerm's keeps K's 16-byte loads and V's 8-byte loads to the
// fewest bank conflicts (none, and 2-way).
//
// The split. A segment is a (sequence, KV head, row tile); its cache rows are cut
// into units of 32. Segments are cut into pieces of at most U units, with U such
// that there is about one piece for each of the 148 CTAs (4, where segments are
// many), so ragged lengths share the SMs evenly and a CTA seldom changes
// segments, which costs about as much as 16 units (q, the merge). A warp takes
// every 16th unit of the piece through a private ring of bulk copies (no CTA
// barrier while it streams) and keeps its own softmax state; the warps meet when
// the piece ends. A segment of several pieces leaves a partial result for each,
// and the CTA that finishes last (a counter, left at zero) adds them in order:
// sums never depend on timing.
//
// Measured: 16 contexts of 24001 to 32768 rows, bf16, 131 MB: 44 us, 3.0 TB/s (45% of
// the measured copy rate; 4.0 TB/s while it streams). A warp's 350 instructions for 16
// rows are one chain (scores, maximum, exponentials, transposes, values): with 16 warps
// an SM issues 2.2 a cycle, and no pipe is full. 16 ragged streams of 64 to 4096 rows:
// 11.7 us, one token over 513 rows: 8.5 us, both bound by what runs once.
//
// What one call pays once is mostly instruction fetch: code that runs once costs
// about 5 cycles an instruction here. So the loop body covers 16 cache rows and
// not 32, q becomes fragments once per CTA and not per warp, and divisions are
// 32-bit.
#pragma once
#include "kv4_rows.cuh"
#include "ptx.cuh"

#include <type_traits>

namespace vg {

struct Kv4AttnParams {
  Kv4View c;
  const void *q;
  void *out;                // [seqs][tokens][heads][D]
  float *lse;               // [seqs][tokens][heads]: log2 of the softmax's denominator, or null
  Strides qs;
  const int32_t *counts;    // new tokens of each sequence, may be null
  uint32_t tokens, heads, group;
  float scale;              // of the scores, times log2(e)
  uint32_t wide;            // 16-byte loads of q are aligned
  uint32_t row_tiles;       // tiles of a (sequence, KV head)'s query rows
  uint32_t *tickets;        // [segments], zero between calls
  float *parts;             // [pieces] partial results
};

__device__ __forceinline__ uint32_t kv4_held(const Kv4View &c, uint32_t seq) {
  return (uint32_t)min(max(c.state[seq].rows, 0), (int32_t)c.capacity);
}
__device__ __forceinline__ int32_t kv4_count(const Kv4AttnParams &p, uint32_t seq) {
  return p.counts ? min(max(p.counts[seq], 0), (int32_t)p.tokens) : (int32_t)p.tokens;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Transpose of an 8x8 matrix of halves held as one pair a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 2^x to within 2 units of the 22nd bit; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// hi and lo fp16 pairs of two fp32 values.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = half2_bits(h);
  lo = half2_bits(__floats2half2_rn(x - f.x, y - f.y));
}

// Power of two that brings a row's largest magnitude to [2^14, 2^15), and its inverse.
__device__ __forceinline__ float row_power(float top, float &inverse) {
  const int e = (int)(__float_as_uint(top) >> 23 & 255) - 127;  // of 0: -127, of inf and NaN: 128
  const int k = min(max(14 - e, -114), 114);
  inverse = __uint_as_float((uint32_t)(127 - k) << 23);
  return __uint_as_float((uint32_t)(127 + k) << 23);
}

// The places of a ring of bulk copies, as the thread that issues them counts. Waits are bounded; once one has run out
// (`stopped`) nothing is issued or waited for any more, places are passed over unread copies, and what was still in
// flight is waited for once more, again with a limit, before the block ends: a call is held up by a few limits, however
// many copies it has.
template <uint32_t kStages>
struct CopyRing {
  uint32_t issued = 0, passed = 0;
  uint32_t stopped = 0;   // a word: with a bool the few-row kernel took 44.5 us for 16 deep contexts and not 43.8

  // issue(stage)
  template <typename F>
  __host__ __device__ __forceinline__ void fetch(F &&issue) {
    if (stopped) return;
    issue(issued % kStages);
    ++issued;
  }
  // The next place is passed; wait(stage, parity) says whether its copy landed in time.
  template <typename F>
  __host__ __device__ __forceinline__ void take(F &&wait) {
    if (!stopped) stopped = !wait(passed % kStages, passed / kStages & 1);
    ++passed;
  }
  // The last copy of each stage: those before it landed before it was issued.
  template <typename F>
  __host__ __device__ __forceinline__ void drain(F &&wait) const {
    for (uint32_t i = issued - (issued < kStages ? issued : kStages); i < issued; ++i) wait(i % kStages, i / kStages & 1);
  }
};

constexpr uint32_t kUnit = 32;        // cache rows of a unit
constexpr uint32_t kRowsWarps = 16;
constexpr uint32_t kRowsStages = 2;
constexpr uint32_t kTileRows = 8;     // query rows of a tile
constexpr uint32_t kRowsThreads = kRowsWarps * 32;
constexpr uint32_t kRowsCtas = 148;   // one per SM
constexpr uint32_t kLeastUnits = 16;  // of a piece: one round of the warps
constexpr uint32_t kMostTickets = 1u << 14;   // segments that may be cut
// P is held times 2^6 relative to a maximum that is only raised once a score passes it by 2^8: raising costs as much as
// a quarter of a step and a new maximum, however small its lead, is common. P stays below 2^14, and fp16's smallest
// numbers lie 2^30 below a weight of 1.
constexpr float kPScale = 6.f, kLead = 8.f;
// The running maximum of a row that has met no score: finite, so that nothing has to be asked before a subtraction. A row
// that sees nothing keeps a denominator of 0.
//
// The maximum that a block runs is one of the products' sums, not yet scaled: the difference of two sums is scaled, and
// not two scaled numbers taken from one another, whose rounding passes P's range where scores pass 2^25 (the row of the
// largest score had a P of infinity or 0).
constexpr float kNoScore = -3e38f;

template <int D>
constexpr uint32_t kPart = kTileRows * (D + 2);   // floats of a partial result: values, maxima, denominators

template <int D>
struct RowsSmem {
  static constexpr uint32_t kCodes = kUnit * D / 2;    // of K or V
  static constexpr uint32_t kScales = kUnit * D / 16;
  static constexpr uint32_t kStage = 2 * (kCodes + kScales);
  static constexpr uint32_t kRing = kRowsWarps * kRowsStages * kStage;
  static constexpr uint32_t kMerge = kRowsWarps * kTileRows * D * 4;
  static constexpr uint32_t kBytes = kRing + kMerge;
};

// Pieces that a call may be cut into: `segments` plus what the target allows.
__host__ __device__ __forceinline__ uint32_t target_pieces(uint32_t segments) {
  return kRowsCtas * (segments * 4 <= kRowsCtas * 3 ? 1 : 4);
}
__host__ __device__ __forceinline__ uint64_t most_pieces(uint64_t segments) {
  return segments > kMostTickets ? 0 : segments + target_pieces((uint32_t)segments);
}

__device__ __forceinline__ uint32_t units_of(uint32_t rows) { return max(1u, (rows + kUnit - 1) / kUnit); }

// How segments are cut: `lanes` segments a sequence, pieces of `size` units, and
// how many pieces there are. A warp's work.
struct Plan {
  uint32_t lanes, size, pieces;
};
__device__ __forceinline__ uint32_t pieces_of(const Kv4View &c, uint32_t s, uint32_t size) {
  return s < c.seqs ? (units_of(kv4_held(c, s)) + size - 1) / size : 0u;
}
__device__ __forceinline__ Plan make_plan(const Kv4View &c, uint32_t lanes) {
  const uint32_t lane = threadIdx.x % 32, segments = c.seqs * lanes;
  Plan p{lanes, 1u << 30, segments};   // one piece a segment
  if (segments > kMostTickets) return p;
  uint32_t total = 0;
#pragma unroll 1
  for (uint32_t s = lane; s < c.seqs; s += 32) total += units_of(kv4_held(c, s));
  total = __reduce_add_sync(~0u, total) * lanes;   // the host keeps it below 2^31
  const uint32_t target = target_pieces(segments);
  p.size = max(kLeastUnits, (total + target - 1) / target);
#pragma unroll 1
  for (int i = 0;; ++i) {
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t s = lane; s < c.seqs; s += 32) n += pieces_of(c, s, p.size);
    p.pieces = __reduce_add_sync(~0u, n) * lanes;
    if (p.pieces <= target || i == 3) return p;
    p.size = max(p.size + 1, (uint32_t)((uint64_t)p.size * p.pieces / target));
  }
}

struct Piece {
  uint32_t seq, lane;          // lane: (KV head, row tile) of the sequence
  uint32_t part, parts;        // of the segment
  uint32_t first, units;       // of the piece, in the segment
};
__device__ __forceinline__ Piece find_piece(const Kv4View &c, const Plan &p, uint32_t index) {
  const uint32_t lane = threadIdx.x % 32;
  uint32_t before = 0;
#pragma unroll 1
  for (uint32_t base = 0; base < c.seqs; base += 32) {
    const uint32_t n = pieces_of(c, base + lane, p.size);
    uint32_t sum = n * p.lanes;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > index);
    if (past) {
      const int at = __ffs(past) - 1;
      const uint32_t parts = __shfl_sync(~0u, n, at);
      const uint32_t into = index - before - (__shfl_sync(~0u, sum, at) - parts * p.lanes);
      Piece x;
      x.seq = base + at;
      x.lane = into / parts;
      x.part = into - x.lane * parts;
      x.parts = parts;
      x.first = x.part * p.size;
      x.units = parts == 1 ? units_of(kv4_held(c, x.seq)) : min(p.size, units_of(kv4_held(c, x.seq)) - x.first);
      return x;
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return Piece{0, 0, 0, 1, 0, 0};   // past the last piece
}

// Cache row of a 16-row tile that MMA row i is (in both halves of the tile).
__device__ __forceinline__ uint32_t perm8(uint32_t i) { return i % 2 ? 4 + (i / 2 ^ 1) : i / 2; }

// A lane's channels of query row r of a (sequence, KV head), and how many cache
// rows it sees (0: none, or no such row).
template <int D, typename T>
__device__ __forceinline__ uint32_t load_query(const Kv4AttnParams &p, uint32_t seq, uint32_t kv, uint32_t r, uint32_t held,
                                               float (&x)[D / 32]) {
  constexpr uint32_t N = D / 32;
  const uint32_t lane = threadIdx.x % 32, tok = r / p.group;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) x[i] = 0.f;
  if (r >= p.tokens * p.group) return 0;
  const int32_t count = kv4_count(p, seq), n = (int32_t)held - count + (int32_t)tok + 1;
  const T *q = (const T *)p.q + (int64_t)seq * p.qs.seq + (int64_t)tok * p.qs.token +
               (int64_t)(kv * p.group + r - tok * p.group) * p.qs.head + lane * N;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) x[i] = (float)q[i];
  return (int32_t)tok < count && n > 0 ? (uint32_t)n : 0u;
}
// A warp puts a query row into column `col` of B fragments [hi, lo][step][lane][2]
// in shared memory; what its scores are to be multiplied by.
template <int D, typename T>
__device__ __forceinline__ float store_query(const Kv4AttnParams &p, const float (&x)[D / 32], uint32_t col, uint32_t *frag) {
  constexpr uint32_t N = D / 32, kLaneChannels = D / 4;   // channels of a lane here, and of a lane of the MMA
  const uint32_t lane = threadIdx.x % 32;
  uint32_t top = 0;
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  float inverse;
  const float power = row_power(__uint_as_float(__reduce_max_sync(~0u, top)), inverse);
  // channel c: lane t = c / (D/4) of its column, word (c % (D/4)) / 8, and within the word i = c % 8: pair i % 4 (half
  // i / 4), two pairs a step
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) {
    const uint32_t c = lane * N + i, in = c % kLaneChannels, y = c % 4;
    const uint32_t step = in / 8 * 2 + y / 2, half = c % 8 / 4;
    __half *dst = (__half *)(frag + (step * 32 + col * 4 + c / kLaneChannels) * 2 + y % 2) + half;
    const float v = x[i] * power;
    const __half hi = __float2half_rn(v);
    *dst = hi;
    if constexpr (sizeof(T) == 4) dst[D / 16 * 32 * 2 * 2] = __float2half_rn(v - __half2float(hi));
  }
  return fmaxf(p.scale * inverse, 0x1p-126f);
}

// T: type of q and out.
template <int D, typename T>
__global__ void __launch_bounds__(kRowsThreads, 1) kv4_rows_kernel(const Kv4AttnParams p) {
  using S = RowsSmem<D>;
  constexpr bool kSplit = sizeof(T) == 4, kSplitP = !std::is_same<T, __nv_bfloat16>::value;
  constexpr int kSteps = D / 16;                // k-steps of a score, and m-tiles of the output
  constexpr uint32_t kLaneChannels = D / 4;     // of K
  constexpr uint32_t kLaneValues = D / 8;       // channels of V
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRowsWarps][kRowsStages];
  __shared__ __align__(8) float w_max[kRowsWarps][kTileRows], w_sum[kRowsWarps][kTileRows];
  __shared__ float f_max[kTileRows], f_sum[kTileRows];
  __shared__ uint32_t last, gave_up;
  __shared__ __align__(8) uint32_t q_frag[kSplit ? 2 : 1][kSteps][32][2];   // B fragments: hi, lo
  __shared__ __align__(8) float factors[kTileRows];
  __shared__ __align__(8) uint32_t seens[kTileRows];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  if (p.lse) pdl_launch_dependents();   // the weights kernel may take the SMs that this one leaves
  __shared__ Plan shared_plan;
  __shared__ Piece shared_piece;
  if (warp == 0) {
    const Plan x = make_plan(p.c, p.c.kv_heads * p.row_tiles);
    if (lane == 0) shared_plan = x;
    if (blockIdx.x < x.pieces) {
      const Piece y = find_piece(p.c, x, blockIdx.x);
      if (lane == 0) shared_piece = y;
    }
  }
  const size_t run_bytes = (size_t)p.c.tiles * Kv4<D>::kTileBytes;
  uint8_t *ring = smem + warp * kRowsStages * S::kStage;
  float *merge = (float *)(smem + S::kRing);

  if (lane == 0)
    for (uint32_t i = 0; i < kRowsStages; ++i) mbar_init(&bars[warp][i], 1);
  if (threadIdx.x == 0) gave_up = 0;
  fence_mbar_init();
  __syncthreads();
  const Plan plan = shared_plan;
  if (blockIdx.x >= plan.pieces) return;

  CopyRing<kRowsStages> copies;
  // this lane's places in a stage
  const uint32_t k_codes = perm8(g) * (D / 2) + t * (D / 8);
  const uint32_t k_scale = 2 * S::kCodes + perm8(g) * (D / 16) + t * kLaneChannels / 32 * 2;
  const uint32_t v_row[2] = {perm8(2 * t), perm8(2 * t + 1)};
  const uint32_t v_codes = S::kCodes + g * (D / 16), v_scale = 2 * S::kCodes + S::kScales + g * kLaneValues / 32 * 2;

  // units of a piece from this warp's `unit` on, one each call, into the next stage of the ring
  auto fetch = [&](const Piece &x, uint32_t unit) {
    copies.fetch([&](uint32_t stage) {
      if (lane == 0) {
        uint8_t *dst = ring + stage * S::kStage;
        const uint32_t row = (x.first + unit) * kUnit;
        const uint8_t *run = p.c.data + ((size_t)x.seq * p.c.kv_heads + x.lane / p.row_tiles) * run_bytes;
        uint64_t *bar = &bars[warp][stage];
        mbar_arrive_expect_tx(bar, S::kStage);
        bulk_g2s(dst, run + Kv4<D>::codes(row, 0), S::kCodes, bar);
        bulk_g2s(dst + S::kCodes, run + Kv4<D>::codes(row, 1), S::kCodes, bar);
        bulk_g2s(dst + 2 * S::kCodes, run + Kv4<D>::scales(row, 0), S::kScales, bar);
        bulk_g2s(dst + 2 * S::kCodes + S::kScales, run + Kv4<D>::scales(row, 1), S::kScales, bar);
      }
    });
  };

  Piece seg = shared_piece;
  uint32_t ahead = warp;    // next unit of the piece to fetch
#pragma unroll 1
  for (uint32_t i = 0; i < kRowsStages && ahead < seg.units; ++i, ahead += kRowsWarps) fetch(seg, ahead);

#pragma unroll 1
  for (uint32_t index = blockIdx.x; index < plan.pieces; index += gridDim.x) {
    const Piece next = index + gridDim.x < plan.pieces ? find_piece(p.c, plan, index + gridDim.x) : Piece{0, 0, 0, 1, 0, 0};
    uint32_t next_ahead = warp;
    const bool whole = seg.parts == 1;
    const uint32_t kv = seg.lane / p.row_tiles, row0 = (seg.lane - kv * p.row_tiles) * kTileRows;
    const uint32_t rows = p.tokens * p.group, tile_rows = min(kTileRows, rows - row0);
    const uint32_t held = kv4_held(p.c, seg.seq);
    // ---- the queries as B fragments, a warp a row: column `warp` of the MMA is query row row0 + warp ----
    if (warp < kTileRows) {
      float x[D / 32];
      const uint32_t seen = load_query<D, T>(p, seg.seq, kv, row0 + warp, held, x);
      const float factor = store_query<D, T>(p, x, warp, &q_frag[0][0][0][0]);
      if (lane == 0) factors[warp] = factor, seens[warp] = seen;
    }
    __syncthreads();
    copies.stopped |= __any_sync(~0u, *(volatile uint32_t *)&gave_up);   // a wait of any warp in an earlier piece ran out
    uint32_t q_hi[kSteps][2], q_lo[kSplit ? kSteps : 1][2];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      *(uint2 *)q_hi[i] = *(const uint2 *)q_frag[0][i][lane];
      if constexpr (kSplit) *(uint2 *)q_lo[i] = *(const uint2 *)q_frag[1][i][lane];
    }
    // scores of query rows 2t and 2t + 1 are this lane's
    const float f0 = factors[2 * t], f1 = factors[2 * t + 1];
    const uint32_t seen0 = seens[2 * t], seen1 = seens[2 * t + 1];
    const uint32_t least = min(seens[0], seens[tile_rows - 1]);   // every row sees these

    float o[kSteps][4], m0 = kNoScore, m1 = kNoScore, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

#pragma unroll 1
    for (uint32_t unit = warp; unit < seg.units; unit += kRowsWarps) {
      const uint32_t stage = copies.passed % kRowsStages;
      copies.take([&](uint32_t at, uint32_t parity) {
        const bool in = __all_sync(~0u, mbar_wait_bounded(&bars[warp][at], parity));
        if (!in && lane == 0) *(volatile uint32_t *)&gave_up = 1;
        return in;
      });
      const uint32_t unit_row = (seg.first + unit) * kUnit;
#pragma unroll 1
      for (uint32_t half = 0; half < kUnit; half += 16) {
        const uint8_t *st = ring + stage * S::kStage + half * (D / 2);            // codes
        const uint8_t *sc = ring + stage * S::kStage + half * (D / 16);           // scales
        const uint32_t first = unit_row + half;   // the first of 16 cache rows
        const bool tail = first + 16 > least;
        // ---- scores ----
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        {
          uint32_t w[2][kSteps / 2];
          __half2 d[2], d72[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint8_t *b = st + k_codes + 8 * y * (D / 2);
            if constexpr (D == 128) {
              const uint4 v = *(const uint4 *)b;
              w[y][0] = v.x, w[y][1] = v.y, w[y][2] = v.z, w[y][3] = v.w;
            } else {
              const uint2 v = *(const uint2 *)b;
              w[y][0] = v.x, w[y][1] = v.y;
            }
            d[y] = __half2half2(*(const __half *)(sc + k_scale + 8 * y * (D / 16)));
            d72[y] = minus72(d[y]);
          }
#pragma unroll
          for (int k = 0; k < kSteps / 2; ++k) {
            __half2 a[4], b[4];
            unpack8(w[0][k], d[0], d72[0], a);
            unpack8(w[1][k], d[1], d72[1], b);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t x[4] = {half2_bits(a[2 * y]), half2_bits(b[2 * y]), half2_bits(a[2 * y + 1]), half2_bits(b[2 * y + 1])};
              mma_f16(c, x, q_hi[2 * k + y]);
              if constexpr (kSplit) mma_f16(c, x, q_lo[2 * k + y]);
            }
          }
        }
        // ---- softmax: c[2y + z] is cache row 8y + perm8(g), query row 2t + z ----
        if (tail) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t r = first + 8 * y + perm8(g);
            if (r >= seen0) c[2 * y] = -INFINITY;
            if (r >= seen1) c[2 * y + 1] = -INFINITY;
          }
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
        }
        uint32_t p_hi[2], p_lo[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float x0 = exp2_fast(fmaf(c[2 * y] - m0, f0, kPScale)), x1 = exp2_fast(fmaf(c[2 * y + 1] - m1, f1, kPScale));
          l0 += x0, l1 += x1;
          if constexpr (kSplitP) {
            split2(x0, x1, p_hi[y], p_lo[y]);
            p_lo[y] = transpose8(p_lo[y]);
          } else {
            p_hi[y] = half2_bits(__floats2half2_rn(x0, x1));
          }
          p_hi[y] = transpose8(p_hi[y]);
        }
        // ---- values: m-tile j is channels g*D/8 + 2j (row g) and the next (row g + 8) ----
        uint32_t w[4][D / 64];
        __half d[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t r = y / 2 * 8 + v_row[y % 2];
          const uint8_t *b = st + v_codes + r * (D / 2);
          if constexpr (D == 128) {
            const uint2 v = *(const uint2 *)b;
            w[y][0] = v.x, w[y][1] = v.y;
          } else {
            w[y][0] = *(const uint32_t *)b;
          }
          d[y] = *(const __half *)(sc + v_scale + r * (D / 16));
          if (tail && first + r >= held) d[y] = __half(0.f);   // bytes past the rows held may be anything
        }
        const __half2 da = __halves2half2(d[0], d[1]), db = __halves2half2(d[2], d[3]);
        const __half2 da72 = minus72(da), db72 = minus72(db);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {   // channels 0-3, 4-7 of the word
            const uint32_t sel = y ? 0x7632 : 0x5410;
            __half2 a[4], b[4];
            unpack8(__byte_perm(w[0][j], w[1][j], sel), da, da72, a);
            unpack8(__byte_perm(w[2][j], w[3][j], sel), db, db72, b);
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t x[4] = {half2_bits(a[2 * z]), half2_bits(a[2 * z + 1]), half2_bits(b[2 * z]), half2_bits(b[2 * z + 1])};
              mma_f16(o[j * 4 + y * 2 + z], x, p_hi);
              if constexpr (kSplitP) mma_f16(o[j * 4 + y * 2 + z], x, p_lo);
            }
          }
        }
      }
      __syncwarp();
      if (ahead < seg.units) fetch(seg, ahead), ahead += kRowsWarps;
      else if (next_ahead < next.units) fetch(next, next_ahead), next_ahead += kRowsWarps;
    }

    // ---- the warps' results meet ----
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
      l0 += __shfl_xor_sync(~0u, l0, x);
      l1 += __shfl_xor_sync(~0u, l1, x);
    }
    m0 = l0 == 0.f ? kNoScore : m0 * f0, m1 = l1 == 0.f ? kNoScore : m1 * f1;   // scaled from here on
    if (g == 0) {
      *(float2 *)&w_max[warp][2 * t] = make_float2(m0, m1);
      *(float2 *)&w_sum[warp][2 * t] = make_float2(l0, l1);
    }
    __syncthreads();
    float top0 = kNoScore, top1 = kNoScore;
#pragma unroll
    for (uint32_t w = 0; w < kRowsWarps; ++w) {
      const float2 x = *(const float2 *)&w_max[w][2 * t];
      top0 = fmaxf(top0, x.x), top1 = fmaxf(top1, x.y);
    }
    // [warp][query row][channel], 16-byte chunks of a lane's channels turned by its query rows: no bank conflicts
    constexpr uint32_t kChunks = kLaneValues / 4;
    {
      const float e0 = exp2_fast(m0 - top0), e1 = exp2_fast(m1 - top1);
      float4 *dst = (float4 *)(merge + (warp * kTileRows + 2 * t) * D + g * kLaneValues);
#pragma unroll
      for (uint32_t i = 0; i < kChunks; ++i) {
        dst[i ^ (t % kChunks)] = make_float4(e0 * o[2 * i][0], e0 * o[2 * i][2], e0 * o[2 * i + 1][0], e0 * o[2 * i + 1][2]);
        dst[D / 4 + (i ^ (t % kChunks))] =
            make_float4(e1 * o[2 * i][1], e1 * o[2 * i][3], e1 * o[2 * i + 1][1], e1 * o[2 * i + 1][3]);
      }
    }
    if (warp == 0 && g < 2) {   // lanes of g = 0 and 1: the denominators of rows 2t and 2t + 1
      const float top = g ? top1 : top0;
      float all = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < kRowsWarps; ++w) {
        all += w_sum[w][2 * t + g] * exp2_fast(w_max[w][2 * t + g] - top);
      }
      f_max[2 * t + g] = top;
      f_sum[2 * t + g] = all;
    }
    __syncthreads();
    auto place = [&](uint32_t r) {   // of a query row in out and lse
      const uint32_t tok = (row0 + r) / p.group, head = kv * p.group + (row0 + r) % p.group;
      return ((size_t)seg.seq * p.tokens + tok) * p.heads + head;
    };
    // a row whose softmax sums up to 0: zeros where it sees no cache row, NaN where every score was -infinity
    auto blank = [&](uint32_t r) { return seens[r] ? NAN : 0.f; };
    auto emit = [&](uint32_t r, uint32_t ch, float4 x, float sum) {   // finished output values
      const float inv = sum == 0.f ? blank(r) : 1.f / sum;
      T y[4] = {from_float<T>(x.x * inv), from_float<T>(x.y * inv), from_float<T>(x.z * inv), from_float<T>(x.w * inv)};
      T *dst = (T *)p.out + place(r) * D + ch;
      if constexpr (sizeof(T) == 4) *(float4 *)dst = *(const float4 *)y;
      else *(uint2 *)dst = *(const uint2 *)y;
    };
    auto emit_lse = [&](uint32_t r, float top, float sum) {
      p.lse[place(r)] = sum == 0.f ? INFINITY + blank(r) : top + log2f(sum) - kPScale;
    };
    float *part = p.parts + (size_t)index * kPart<D>;
    if (threadIdx.x < tile_rows * (D / 4)) {
      const uint32_t r = threadIdx.x / (D / 4), ch = threadIdx.x % (D / 4) * 4;
      const float *src = merge + r * D + ch / kLaneValues * kLaneValues + (ch / 4 % kChunks ^ (r / 2 % kChunks)) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (uint32_t w = 0; w < kRowsWarps; ++w) {
        const float4 y = *(const float4 *)(src + w * kTileRows * D);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
      }
      if (whole) emit(r, ch, x, f_sum[r]);
      else *(float4 *)(part + r * D + ch) = x;
    }
    if (threadIdx.x < tile_rows) {
      if (!whole) {
        part[kTileRows * D + threadIdx.x] = f_max[threadIdx.x];
        part[kTileRows * (D + 1) + threadIdx.x] = f_sum[threadIdx.x];
      } else if (p.lse) {
        emit_lse(threadIdx.x, f_max[threadIdx.x], f_sum[threadIdx.x]);
      }
    }
    __syncthreads();
    if (!whole) {
      const uint32_t pieces = seg.parts;
      const float *others = p.parts + (size_t)(index - seg.part) * kPart<D>;
      uint32_t *ticket = p.tickets + seg.seq * plan.lanes + seg.lane;
      if (threadIdx.x == 0) last = atomic_add_acq_rel(ticket, 1u) == pieces - 1;
      __syncthreads();
      if (last) {
        if (threadIdx.x == 0) *ticket = 0;
        float *weight = merge;   // [pieces][kTileRows]
        auto piece = [&](uint32_t i) { return others + (size_t)i * kPart<D>; };
        if (warp < tile_rows) {   // a warp a query row, its lanes the pieces
          float top = kNoScore, all = 0.f;
#pragma unroll 1
          for (uint32_t i = lane; i < pieces; i += 32) {
            const float m = __ldcg(piece(i) + kTileRows * D + warp);
            weight[i * kTileRows + warp] = m;
            top = fmaxf(top, m);
          }
#pragma unroll
          for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, x));
#pragma unroll 1
          for (uint32_t i = lane; i < pieces; i += 32) {
            const float m = weight[i * kTileRows + warp], sum = __ldcg(piece(i) + kTileRows * (D + 1) + warp);
            const float w = exp2_fast(m - top);
            all += w * sum;
            weight[i * kTileRows + warp] = w;
          }
#pragma unroll
          for (int x = 16; x; x >>= 1) all += __shfl_xor_sync(~0u, all, x);
          if (lane == 0) {
            f_sum[warp] = all;
            if (p.lse) emit_lse(warp, top, all);
          }
        }
        __syncthreads();
        // threads are [share of the pieces][query row][4 channels]
        constexpr uint32_t kItems = kTileRows * (D / 4), kShares = kRowsThreads / kItems;
        const uint32_t item = threadIdx.x % kItems, share = threadIdx.x / kItems;
        const uint32_t r = item / (D / 4), ch = item % (D / 4) * 4;
        float4 *shared = (float4 *)(merge + S::kMerge / 4 - kRowsThreads * 4);   // [kShares][kItems]
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < tile_rows) {
#pragma unroll 8
          for (uint32_t i = share; i < pieces; i += kShares) {
            const float w = weight[i * kTileRows + r];
            const float4 y = __ldcg((const float4 *)(piece(i) + r * D + ch));
            x.x = fmaf(w, y.x, x.x), x.y = fmaf(w, y.y, x.y), x.z = fmaf(w, y.z, x.z), x.w = fmaf(w, y.w, x.w);
          }
        }
        shared[share * kItems + item] = x;
        __syncthreads();
        if (share == 0 && r < tile_rows) {
#pragma unroll
          for (uint32_t i = 1; i < kShares; ++i) {
            const float4 y = shared[i * kItems + item];
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
          }
          emit(r, ch, x, f_sum[r]);
        }
        __syncthreads();
      }
    }
    // what of the next piece no unit of this one made room for
    if (index + gridDim.x < plan.pieces) {
      const uint32_t had = (seg.units + kRowsWarps - 1 - warp) / kRowsWarps;   // units that this warp took
#pragma unroll 1
      for (uint32_t i = had; i < kRowsStages; ++i)
        if (next_ahead < next.units) fetch(next, next_ahead), next_ahead += kRowsWarps;
    }
    seg = next;
    ahead = next_ahead;
  }
  if (copies.stopped && lane == 0) {
    copies.drain([&](uint32_t at, uint32_t parity) { mbar_wait_bounded(&bars[warp][at], parity); });
    atomicOr(&p.c.state[0].status, kKv4Timeout);
  }
}

}  // namespace vg
