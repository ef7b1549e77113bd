// Attention of few query rows over a 4-bit cache: single tokens and short drafts.
//
// The mathematics. The query rows of a (sequence, KV head) are packed: row
// r = token * group + head of the group. A tile is 16 rows of one m16n8k16 MMA
// A operand; fp32 queries are split into fp16 hi + lo, which takes two rows, so
// a tile is then 8 query rows and C row g + C row g + 8 is the score. Scores are
// Q K^T with the cache's K rows as the B operand, and the output P V with its V
// rows as B: both come out of the codes with one shift, one lop3 and one fused
// multiply-add a pair (kv4.cuh), exactly. P is kept as hi + lo for fp32 queries
// and rounded to fp16 (11 bits) for 16-bit ones, where the output's rounding is
// as large. Softmax statistics and sums are fp32.
//
// The contraction over channels may run in any order as long as both operands
// agree, so lane (g, t) takes channels [t*D/4, (t+1)*D/4) of K row g: one wide
// load, and at head_dim 128 one scale. The scores' C fragment (rows = heads,
// columns = cache rows) is the A fragment of P without a shuffle, when lane t's
// V rows are those of its score columns. V needs pairs along rows: two bytes
// permutes put the nibbles of two rows side by side.
//
// The split. All (sequence, KV head, row tile) segments are cut into units of
// 32 cache rows, and the units of all segments are dealt out evenly to one CTA
// per SM, in order: ragged lengths balance by themselves. A warp takes every
// kWarps-th unit of its CTA's range through a private ring of bulk copies (no
// CTA barrier while it streams), keeps its own softmax state, and the warps
// meet when a segment ends. A segment that spans CTAs leaves one partial result
// per CTA; the last CTA to arrive (a counter, left at zero) adds them in CTA
// order. Sums therefore never depend on timing.
#pragma once
#include "kv4_rows.cuh"
#include "ptx.cuh"

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
  uint32_t *tickets;        // [CTAs], zero between calls
  float *parts;             // [2 * CTAs][rows of a tile][D + 2]
};

__device__ __forceinline__ uint32_t kv4_held(const Kv4View &c, uint32_t seq) {
  return (uint32_t)min(max(c.state[seq].rows, 0), (int32_t)c.capacity);
}
__device__ __forceinline__ int32_t kv4_count(const Kv4AttnParams &p, uint32_t seq) {
  return p.counts ? min(max(p.counts[seq], 0), (int32_t)p.tokens) : (int32_t)p.tokens;
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

constexpr uint32_t kUnit = 32;      // cache rows of a unit
constexpr uint32_t kRowsWarps = 12;
constexpr uint32_t kRowsStages = 3;
constexpr uint32_t kRowsThreads = kRowsWarps * 32;
constexpr float kPScale = 14.f;     // P is held times 2^14: fp16's smallest numbers then lie 2^38 below the largest

template <int D>
struct RowsSmem {
  static constexpr uint32_t kCodes = kUnit * D / 2;    // of K or V
  static constexpr uint32_t kScales = kUnit * D / 16;
  static constexpr uint32_t kStage = 2 * (kCodes + kScales);
  static constexpr uint32_t kRing = kRowsWarps * kRowsStages * kStage;
  static constexpr uint32_t kMerge = kRowsWarps * 8 * D * 4;
  static constexpr uint32_t kBytes = kRing + kMerge;
};

// Position in the dealt-out order of units.
struct UnitCursor {
  uint32_t seq, lane, unit, units;  // lane: (KV head, row tile) of the sequence
};

__device__ __forceinline__ uint32_t units_of(uint32_t rows) { return max(1u, (rows + kUnit - 1) / kUnit); }

// Total units of all sequences times lanes, and where unit `x` lies. Every warp
// computes them for itself.
__device__ __forceinline__ uint64_t total_units(const Kv4View &c, uint32_t lanes) {
  uint64_t n = 0;
  for (uint32_t s = threadIdx.x % 32; s < c.seqs; s += 32) n += units_of(kv4_held(c, s));
#pragma unroll
  for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
  return n * lanes;
}
__device__ __forceinline__ UnitCursor find_unit(const Kv4View &c, uint32_t lanes, uint64_t x) {
  const uint32_t lane = threadIdx.x % 32;
  uint64_t before = 0;
  for (uint32_t base = 0; base < c.seqs; base += 32) {
    const uint32_t s = base + lane;
    const uint32_t u = s < c.seqs ? units_of(kv4_held(c, s)) : 0;
    uint64_t sum = (uint64_t)u * lanes;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > x);
    if (past) {
      const int at = __ffs(past) - 1;
      const uint32_t units = __shfl_sync(~0u, u, at);
      const uint64_t into = x - before - (__shfl_sync(~0u, sum, at) - (uint64_t)units * lanes);
      return UnitCursor{base + at, (uint32_t)(into / units), (uint32_t)(into % units), units};
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return UnitCursor{c.seqs, 0, 0, 1};
}

// T: type of q and out. fp32 queries take two MMA rows each.
template <int D, typename T>
__global__ void __launch_bounds__(kRowsThreads, 1) kv4_rows_kernel(const Kv4AttnParams p) {
  using S = RowsSmem<D>;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr uint32_t kRows = kSplit ? 8 : 16;   // query rows of a tile
  constexpr int kSteps = D / 16;                // MMAs of a score, and n-tiles of the output (D / 8) / 2
  constexpr uint32_t kLaneChannels = D / 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRowsWarps][kRowsStages];
  __shared__ float w_max[kRowsWarps][16], w_sum[kRowsWarps][16];
  __shared__ float f_max[16], f_sum[16];
  __shared__ uint32_t last;
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const uint32_t lanes = p.c.kv_heads * p.row_tiles, rows = p.tokens * p.group;
  const uint64_t total = total_units(p.c, lanes);
  const uint32_t ctas = (uint32_t)min((uint64_t)gridDim.x, total);   // every one of them has a unit
  if (blockIdx.x >= ctas) return;
  const uint64_t begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
  const size_t run_bytes = (size_t)p.c.tiles * Kv4<D>::kTileBytes;
  uint8_t *ring = smem + warp * kRowsStages * S::kStage;
  float *merge = (float *)(smem + S::kRing);

  if (lane == 0)
    for (uint32_t i = 0; i < kRowsStages; ++i) mbar_init(&bars[warp][i], 1);
  fence_mbar_init();
  __syncwarp();

  UnitCursor seg = find_unit(p.c, lanes, begin);   // segment being worked on (the same in every warp)
  UnitCursor ahead = seg;                          // next unit of this warp to fetch
  uint64_t fetch = begin + warp;
  uint32_t fetched = 0;
  auto advance = [&](UnitCursor &u, uint32_t by) {
    u.unit += by;
    while (u.unit >= u.units && u.seq < p.c.seqs) {
      u.unit -= u.units;
      if (++u.lane == lanes) {
        u.lane = 0;
        if (++u.seq < p.c.seqs) u.units = units_of(kv4_held(p.c, u.seq));
      }
    }
  };
  advance(ahead, warp);
  auto fetch_next = [&]() {  // one lane
    if (fetch >= end) return;
    const uint32_t stage = fetched % kRowsStages;
    uint8_t *dst = ring + stage * S::kStage;
    const uint32_t row = ahead.unit * kUnit;
    const uint8_t *run = p.c.data + ((size_t)ahead.seq * p.c.kv_heads + ahead.lane / p.row_tiles) * run_bytes;
    uint64_t *bar = &bars[warp][stage];
    mbar_arrive_expect_tx(bar, S::kStage);
    bulk_g2s(dst, run + Kv4<D>::codes(row, 0), S::kCodes, bar);
    bulk_g2s(dst + S::kCodes, run + Kv4<D>::codes(row, 1), S::kCodes, bar);
    bulk_g2s(dst + 2 * S::kCodes, run + Kv4<D>::scales(row, 0), S::kScales, bar);
    bulk_g2s(dst + 2 * S::kCodes + S::kScales, run + Kv4<D>::scales(row, 1), S::kScales, bar);
    ++fetched;
    fetch += kRowsWarps;
    advance(ahead, kRowsWarps);
  };
  if (lane == 0)
    for (uint32_t i = 0; i < kRowsStages; ++i) fetch_next();

  uint32_t used = 0;            // units taken by this warp
  uint64_t mine = begin + warp; // its next unit
  bool timed_out = false;
  for (uint64_t at = begin; at < end;) {
    const uint64_t seg_end = min(end, at + (seg.units - seg.unit));
    const bool whole = seg.unit == 0 && at + seg.units <= end;
    const uint32_t kv = seg.lane / p.row_tiles, row0 = seg.lane % p.row_tiles * kRows;
    const uint32_t held = kv4_held(p.c, seg.seq);
    const int32_t count = kv4_count(p, seg.seq);
    // cache rows that this lane's query rows (g, and g + 8) see, and the fewest of the tile
    uint32_t seen[2] = {0, 0};
    float factor[2] = {0.f, 0.f};
    uint32_t qa[kSteps][4];
#pragma unroll
    for (int h = 0; h < (kSplit ? 1 : 2); ++h) {
      const uint32_t r = row0 + g + 8 * h;
      float x[kLaneChannels], top = 0.f;
      if (r < rows) {
        const uint32_t tok = r / p.group, head = kv * p.group + r % p.group;
        const int32_t n = (int32_t)held - count + (int32_t)tok + 1;
        seen[h] = (int32_t)tok < count && n > 0 ? (uint32_t)n : 0u;
        const T *q = (const T *)p.q + (int64_t)seg.seq * p.qs.seq + (int64_t)tok * p.qs.token +
                     (int64_t)head * p.qs.head + t * kLaneChannels;
#pragma unroll
        for (uint32_t i = 0; i < kLaneChannels; i += 8) {
          if (p.wide) load8<T, true>(q + i, *(float(*)[8])(x + i));
          else load8<T, false>(q + i, *(float(*)[8])(x + i));
        }
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kLaneChannels; ++i) x[i] = 0.f;
      }
#pragma unroll
      for (uint32_t i = 0; i < kLaneChannels; ++i) top = fmaxf(top, fabsf(x[i]));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
      top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
      float inverse;
      const float power = row_power(top, inverse);
      factor[h] = p.scale * inverse;
      // step s = word s/2 of the lane's channels, pairs (i, i + 4) with i = 2 * (s % 2) and the next
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int c = s / 2 * 8 + s % 2 * 2;
        if constexpr (kSplit) {
          split2(x[c] * power, x[c + 4] * power, qa[s][0], qa[s][1]);
          split2(x[c + 1] * power, x[c + 5] * power, qa[s][2], qa[s][3]);
        } else {
          qa[s][h] = half2_bits(__floats2half2_rn(x[c] * power, x[c + 4] * power));
          qa[s][2 + h] = half2_bits(__floats2half2_rn(x[c + 1] * power, x[c + 5] * power));
        }
      }
    }
    uint32_t least = held;
    if (row0 + g < rows) least = min(least, seen[0]);
    if (!kSplit && row0 + g + 8 < rows) least = min(least, seen[1]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) least = min(least, __shfl_xor_sync(~0u, least, o));

    float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    for (; mine < seg_end; mine += kRowsWarps, ++used) {
      const uint32_t stage = used % kRowsStages;
      const uint8_t *st = ring + stage * S::kStage;
      const uint32_t first = (seg.unit + (uint32_t)(mine - at)) * kUnit;   // its first cache row
      if (!mbar_wait_bounded(&bars[warp][stage], used / kRowsStages & 1)) timed_out = true;
      const bool tail = first + kUnit > least;
      // ---- scores: columns of n-tile i are cache rows 8i + {t, 4 + (t^1)} ----
      float c[kUnit / 8][4];
      const uint32_t krow = g % 2 ? 4 + (g / 2 ^ 1) : g / 2;
#pragma unroll
      for (int i = 0; i < (int)kUnit / 8; ++i) {
        const uint32_t r = 8 * i + krow;
        uint32_t w[kSteps / 2];
        if constexpr (D == 128) {
          const uint4 v = *(const uint4 *)(st + r * (D / 2) + t * 16);
          w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
          const uint2 v = *(const uint2 *)(st + r * (D / 2) + t * 8);
          w[0] = v.x, w[1] = v.y;
        }
        const __half2 d = __half2half2(*(const __half *)(st + 2 * S::kCodes + r * (D / 16) + t * kLaneChannels / 32 * 2));
        const __half2 d72 = minus72(d);
        c[i][0] = c[i][1] = c[i][2] = c[i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < kSteps / 2; ++k) {
          __half2 h[4];
          unpack8(w[k], d, d72, h);
          mma_f16(c[i], qa[2 * k], half2_bits(h[0]), half2_bits(h[1]));
          mma_f16(c[i], qa[2 * k + 1], half2_bits(h[2]), half2_bits(h[3]));
        }
      }
      // ---- softmax ----
      float s[2][kUnit / 4], top[2] = {m[0], m[1]};
#pragma unroll
      for (int i = 0; i < (int)kUnit / 8; ++i) {
        if constexpr (kSplit) {
          s[0][2 * i] = (c[i][0] + c[i][2]) * factor[0];
          s[0][2 * i + 1] = (c[i][1] + c[i][3]) * factor[0];
        } else {
          s[0][2 * i] = c[i][0] * factor[0], s[0][2 * i + 1] = c[i][1] * factor[0];
          s[1][2 * i] = c[i][2] * factor[1], s[1][2 * i + 1] = c[i][3] * factor[1];
        }
      }
#pragma unroll
      for (int h = 0; h < (kSplit ? 1 : 2); ++h) {
        if (tail) {
#pragma unroll
          for (int i = 0; i < (int)kUnit / 4; ++i) {
            const uint32_t r = first + i / 2 * 8 + (i % 2 ? 4 + (t ^ 1) : t);
            if (r >= seen[h]) s[h][i] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < (int)kUnit / 4; ++i) top[h] = fmaxf(top[h], s[h][i]);
        top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(~0u, top[h], 2));
      }
      if (__any_sync(~0u, top[0] > m[0] || top[1] > m[1])) {
        const float f0 = m[0] == top[0] ? 1.f : exp2f(m[0] - top[0]), f1 = m[1] == top[1] ? 1.f : exp2f(m[1] - top[1]);
        l[0] *= f0, l[1] *= f1;
        m[0] = top[0], m[1] = top[1];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[j][0] *= f0, o[j][1] *= f0;
          o[j][2] *= kSplit ? f0 : f1, o[j][3] *= kSplit ? f0 : f1;
        }
      }
      uint32_t pa[kUnit / 16][4];
#pragma unroll
      for (int h = 0; h < (kSplit ? 1 : 2); ++h) {
        const float base = kPScale - (m[h] == -INFINITY ? 0.f : m[h]);
#pragma unroll
        for (int i = 0; i < (int)kUnit / 4; ++i) {
          s[h][i] = exp2f(s[h][i] + base);
          l[h] += s[h][i];
        }
#pragma unroll
        for (int i = 0; i < (int)kUnit / 8; ++i) {
          if constexpr (kSplit) split2(s[0][2 * i], s[0][2 * i + 1], pa[i / 2][i % 2 * 2], pa[i / 2][i % 2 * 2 + 1]);
          else pa[i / 2][i % 2 * 2 + h] = half2_bits(__floats2half2_rn(s[h][2 * i], s[h][2 * i + 1]));
        }
      }
      // ---- values: lane t's rows are its score columns; its channels [g*D/8, (g+1)*D/8), n-tile j the j-th ----
#pragma unroll
      for (int k = 0; k < (int)kUnit / 16; ++k) {
        uint32_t w[4][D / 64];
        __half d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t r = 16 * k + i / 2 * 8 + (i % 2 ? 4 + (t ^ 1) : t);
          const uint8_t *b = st + S::kCodes + r * (D / 2) + g * (D / 16);
          if constexpr (D == 128) {
            const uint2 v = *(const uint2 *)b;
            w[i][0] = v.x, w[i][1] = v.y;
          } else {
            w[i][0] = *(const uint32_t *)b;
          }
          d[i] = *(const __half *)(st + 2 * S::kCodes + S::kScales + r * (D / 16) + g * (D / 8) / 32 * 2);
          if (tail && first + r >= held) d[i] = __half(0.f);   // bytes past the rows held may be anything
        }
        const __half2 da = __halves2half2(d[0], d[1]), db = __halves2half2(d[2], d[3]);
        const __half2 da72 = minus72(da), db72 = minus72(db);
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {   // channels 0-3, 4-7 of the word
            const uint32_t sel = x ? 0x7632 : 0x5410;
            __half2 a[4], b[4];
            unpack8(__byte_perm(w[0][j], w[1][j], sel), da, da72, a);
            unpack8(__byte_perm(w[2][j], w[3][j], sel), db, db72, b);
#pragma unroll
            for (int y = 0; y < 4; ++y) mma_f16(o[j * 8 + x * 4 + y], pa[k], half2_bits(a[y]), half2_bits(b[y]));
          }
        }
      }
      __syncwarp();
      if (lane == 0) fetch_next();
    }

    // ---- the warps' results meet ----
#pragma unroll
    for (int h = 0; h < (kSplit ? 1 : 2); ++h) {
      l[h] += __shfl_xor_sync(~0u, l[h], 1);
      l[h] += __shfl_xor_sync(~0u, l[h], 2);
      if (t == 0) w_max[warp][g + 8 * h] = m[h], w_sum[warp][g + 8 * h] = l[h];
    }
    __syncthreads();
    const uint32_t tile_rows = min(kRows, rows - row0);
    if (threadIdx.x < kRows) {
      float top = -INFINITY, all = 0.f;
      for (uint32_t w = 0; w < kRowsWarps; ++w) top = fmaxf(top, w_max[w][threadIdx.x]);
      for (uint32_t w = 0; w < kRowsWarps; ++w) {
        const float wm = w_max[w][threadIdx.x];
        all += w_sum[w][threadIdx.x] * (wm == -INFINITY ? 0.f : exp2f(wm - top));
      }
      f_max[threadIdx.x] = top;
      f_sum[threadIdx.x] = all;
    }
    __syncthreads();
    // partial results: this CTA's piece of a segment begun before it is slot 0, else slot 1
    const uint32_t slot = blockIdx.x * 2 + (seg.unit == 0);
    float *part = p.parts + (size_t)slot * kRows * (D + 2);
    auto emit = [&](uint32_t r, uint32_t ch, float x, float sum) {   // a finished output value
      const uint32_t tok = (row0 + r) / p.group, head = kv * p.group + (row0 + r) % p.group;
      const size_t i = ((size_t)seg.seq * p.tokens + tok) * p.heads + head;
      ((T *)p.out)[i * D + ch] = from_float<T>(sum == 0.f ? 0.f : x / sum);
    };
    auto emit_lse = [&](uint32_t r, float top, float sum) {
      const uint32_t tok = (row0 + r) / p.group, head = kv * p.group + (row0 + r) % p.group;
      p.lse[((size_t)seg.seq * p.tokens + tok) * p.heads + head] = sum == 0.f ? INFINITY : top + log2f(sum) - kPScale;
    };
#pragma unroll
    for (uint32_t h = 0; h < (kSplit ? 1 : 2); ++h) {
      if (h * 8 >= tile_rows) break;
      const float top = f_max[g + 8 * h], f = m[h] == -INFINITY ? 0.f : exp2f(m[h] - top);
      float *dst = merge + warp * 8 * D + lane * kLaneChannels;   // row g, channels [t*D/4, (t+1)*D/4)
      // column 2t of n-tile j is channel 2t*D/8 + j, column 2t + 1 the one D/8 on
#pragma unroll
      for (int j = 0; j < D / 8; j += 4) {
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float4 v;
          float *e = (float *)&v;
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = f * (kSplit ? o[j + i][y] + o[j + i][y + 2] : o[j + i][y + 2 * h]);
          const uint32_t chunk = y * (D / 32) + j / 4;
          ((float4 *)dst)[chunk ^ (lane % (D / 16))] = v;
        }
      }
      __syncthreads();
      const uint32_t n = min(8u, tile_rows - 8 * h) * D;
      for (uint32_t e = threadIdx.x; e < n; e += kRowsThreads) {
        const uint32_t r = e / D, ch = e % D, ln = r * 4 + ch / kLaneChannels, in = ch % kLaneChannels;
        const uint32_t at4 = ln * kLaneChannels + (((in / 4) ^ (ln % (D / 16))) * 4 + in % 4);
        float x = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kRowsWarps; ++w) x += merge[w * 8 * D + at4];
        if (whole) emit(r + 8 * h, ch, x, f_sum[r + 8 * h]);
        else part[(r + 8 * h) * (D + 2) + ch] = x;
      }
      __syncthreads();
    }
    if (threadIdx.x < tile_rows) {
      if (whole) {
        if (p.lse) emit_lse(threadIdx.x, f_max[threadIdx.x], f_sum[threadIdx.x]);
      } else {
        part[threadIdx.x * (D + 2) + D] = f_max[threadIdx.x];
        part[threadIdx.x * (D + 2) + D + 1] = f_sum[threadIdx.x];
      }
    }
    if (!whole) {
      // CTAs that share the segment: those that hold its first and its last unit, and all between
      const uint64_t seg_first = at - seg.unit, seg_last = seg_first + seg.units - 1;
      const uint32_t c0 = (uint32_t)(((seg_first + 1) * ctas - 1) / total);
      const uint32_t c1 = (uint32_t)(((seg_last + 1) * ctas - 1) / total);
      const uint32_t pieces = c1 - c0 + 1;
      uint32_t *ticket = p.tickets + c0;   // a CTA begins at most one segment that others finish
      __syncthreads();
      if (threadIdx.x == 0) last = atomic_add_acq_rel(ticket, 1u) == pieces - 1;
      __syncthreads();
      if (last) {
        if (threadIdx.x == 0) *ticket = 0;
        float *weight = merge;   // [pieces][kRows]: at most 148 * 16 floats
        auto piece = [&](uint32_t i) { return p.parts + (size_t)((c0 + i) * 2 + (i == 0)) * kRows * (D + 2); };
        for (uint32_t i = threadIdx.x; i < pieces * tile_rows; i += kRowsThreads)
          weight[i] = __ldcg(piece(i / tile_rows) + i % tile_rows * (D + 2) + D);
        __syncthreads();
        if (threadIdx.x < tile_rows) {
          const uint32_t r = threadIdx.x;
          float top = -INFINITY, all = 0.f;
          for (uint32_t i = 0; i < pieces; ++i) top = fmaxf(top, weight[i * tile_rows + r]);
          for (uint32_t i = 0; i < pieces; ++i) {
            const float wm = weight[i * tile_rows + r], w = wm == -INFINITY ? 0.f : exp2f(wm - top);
            weight[i * tile_rows + r] = w;
            all += w * __ldcg(piece(i) + r * (D + 2) + D + 1);
          }
          f_sum[r] = all;
          if (p.lse) emit_lse(r, top, all);
        }
        __syncthreads();
        for (uint32_t e = threadIdx.x; e < tile_rows * D; e += kRowsThreads) {
          const uint32_t r = e / D, ch = e % D;
          float x = 0.f;
          for (uint32_t i = 0; i < pieces; ++i) x += weight[i * tile_rows + r] * __ldcg(piece(i) + r * (D + 2) + ch);
          emit(r, ch, x, f_sum[r]);
        }
        __syncthreads();
      }
    }
    advance(seg, (uint32_t)(seg_end - at));
    at = seg_end;
  }
  if (timed_out && lane == 0) atomicOr(&p.c.state[0].status, kKv4Timeout);
}

}  // namespace vg
