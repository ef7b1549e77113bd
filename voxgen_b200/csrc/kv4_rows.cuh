// Rows of the 4-bit cache: quantising store, read-back, and eviction.
#pragma once
#include "kv4.cuh"

namespace vg {

struct Kv4View {  // one cache, as the kernels see it
  uint8_t *data;
  Kv4Seq *state;
  float *weights;      // [seqs][kv_heads][capacity], may be null
  int32_t *positions;  // likewise
  uint32_t seqs, kv_heads, capacity, tiles;
};

struct Strides {  // in elements; channels are contiguous
  int64_t seq, token, head;
};

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendParams {
  Kv4View c;
  const void *k, *v;
  Strides ks, vs;
  const int32_t *at, *counts;  // per sequence, may be null
  uint32_t tokens, blocks;     // blocks per sequence
};

constexpr uint32_t kRowThreads = 256, kAppendBlocks = 4;   // kAppendBlocks: resident on an SM

// One lane quantises 16 channels of a K row and of the V row beside it; the two
// lanes of a block agree on its extremes by a shuffle. Bound by the input's bytes
// and, for 16-bit inputs, nearly as much by the instructions: 16 channels a lane
// and packed fp32 arithmetic bring them to about 8 a value. 28 x 4096 x 2 fp16 rows
// of 128, K and V (150 MB moved, 23 us at the measured 6.54 TB/s): 49 us with 8
// channels a lane and single operations, 37 us so, 32 us with the blocks of one
// wave (4 an SM, 64 registers; 3 take 35 us, 5 spill and take 34).
//
// The rows held are advanced by the last block of a sequence to finish: every
// block has read them by then, since what it did depended on them. One launch
// does the whole append.
template <int D, typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads, kAppendBlocks) kv4_append_kernel(const AppendParams p) {
  constexpr uint32_t L = D / 16;                 // lanes of a row
  constexpr uint32_t kRows = kRowThreads / L;    // (token, head) pairs per pass
  const uint32_t seq = blockIdx.x / p.blocks, block = blockIdx.x % p.blocks;
  Kv4Seq *st = p.c.state + seq;
  const int4 s = *(const int4 *)st;
  const int32_t at = p.at ? p.at[seq] : s.x;
  const int32_t count = p.counts ? p.counts[seq] : (int32_t)p.tokens;
  const bool bad = at < 0 || at > s.x || count < 0 || count > (int32_t)p.tokens;
  const bool full = !bad && (uint32_t)at + (uint32_t)count > p.c.capacity;
  const uint32_t items = bad || full ? 0 : (uint32_t)count * p.c.kv_heads;
  const uint32_t lane = threadIdx.x % L;
  const T *k = (const T *)p.k + (int64_t)seq * p.ks.seq + lane * 16;
  const T *v = (const T *)p.v + (int64_t)seq * p.vs.seq + lane * 16;
  bool odd = false;  // met a value that it holds as another: a NaN, an infinity or one past the largest
  for (uint32_t base = block * kRows; base < items; base += p.blocks * kRows) {
    const uint32_t item = base + threadIdx.x / L;
    const bool on = item < items;
    const uint32_t token = on ? item / p.c.kv_heads : 0, head = on ? item - token * p.c.kv_heads : 0;
    float x[2][16];
    const T *src[2] = {k + (int64_t)token * p.ks.token + (int64_t)head * p.ks.head,
                       v + (int64_t)token * p.vs.token + (int64_t)head * p.vs.head};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      load8<T, VEC>(src[i], *(float(*)[8])x[i]);
      load8<T, VEC>(src[i] + 8, *(float(*)[8])(x[i] + 8));
    }
    const uint32_t row = (uint32_t)at + token;
    const size_t lane_row = (size_t)seq * p.c.kv_heads + head;
    uint8_t *run = p.c.data + lane_row * p.c.tiles * Kv4<D>::kTileBytes;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float(&y)[16] = x[i];
      const float2 none = make_float2(0.f, 0.f);
      float high = y[0], low = y[0];
      float2 zero = none;   // NaN once a value is not finite
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        zero = fma2(make_float2(y[j], y[j + 1]), none, zero);
        high = max3(high, y[j], y[j + 1]);
        low = min3(low, y[j], y[j + 1]);
      }
      const bool wild = !(zero.x + zero.y == 0.f);
      if (wild || high > kKv4Largest || low < -kKv4Largest) {
        odd |= on;
        high = -kKv4Largest, low = kKv4Largest;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          y[j] = y[j] == y[j] ? fminf(fmaxf(y[j], -kKv4Largest), kKv4Largest) : 0.f;
          high = fmaxf(high, y[j]);
          low = fminf(low, y[j]);
        }
      }
      high = fmaxf(high, __shfl_xor_sync(~0u, high, 1));
      low = fminf(low, __shfl_xor_sync(~0u, low, 1));
      const float d = kv4_scale(high, low);
      const float inv = d == 0.f ? 0.f : __frcp_rn(d);
      // |x * inv| < 8.1, so only 8 has to be brought back to 7. Adding 1.5 * 2^23 rounds to a whole number, ties to
      // even, as rintf does, and leaves it in the low bits; the codes shift in from the last one on, and the magic
      // number's own bits leave by one subtraction.
      const float2 inv2 = make_float2(inv, inv), magic = make_float2(12582912.f, 12582912.f);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int j = 14; j >= 0; j -= 2) {
        float2 n = mul2(make_float2(y[j], y[j + 1]), inv2);
        n = add2(make_float2(fminf(n.x, 7.f), fminf(n.y, 7.f)), magic);
        uint32_t &c = w[j / 8];
        c = c * 16 + __float_as_uint(n.y);
        c = c * 16 + __float_as_uint(n.x);
      }
      constexpr uint32_t kMagic = (0x4B400000u - 8u) * 0x11111111u;
      if (on) {
        *(uint2 *)(run + Kv4<D>::codes(row, i) + lane * 8) = make_uint2(w[0] - kMagic, w[1] - kMagic);
        if (lane % 2 == 0) *(__half *)(run + Kv4<D>::scales(row, i) + lane) = __float2half_rn(d);
      }
    }
    if (on && lane == 0) {
      if (p.c.weights) p.c.weights[lane_row * p.c.capacity + row] = 0.f;
      if (p.c.positions) p.c.positions[lane_row * p.c.capacity + row] = s.y - s.x + at + (int32_t)token;
    }
  }
  if (__syncthreads_or(odd) && threadIdx.x == 0) atomicOr(&st->status, kKv4NonFinite);
  if (threadIdx.x == 0) {
    const uint32_t done = p.blocks > 1 ? atomicAdd((uint32_t *)&st->ticket, 1u) : 0;
    if (done == p.blocks - 1) {
      if (bad || full) {
        atomicOr(&st->status, bad ? kKv4BadRow : kKv4Full);
      } else {
        st->rows = at + count;
        st->next = s.y + at + count - s.x;
      }
      st->ticket = 0;
    }
  }
}

// ---------------------------------------------------------------------------
// read
// ---------------------------------------------------------------------------
struct ReadParams {
  Kv4View c;
  void *k, *v;            // [seqs][tokens][kv_heads][D]
  const int32_t *first;   // per sequence, may be null (row 0)
  uint32_t tokens, blocks;
};

// The values of rows [first, first + tokens) of every sequence; rows that a
// sequence does not hold read as 0. One lane unpacks 8 channels of K and of V,
// of two rows at a time. Bound by the bytes written: 28 x 4096 x 2 rows of 128 as
// fp16 in 29 us, 5.2 TB/s.
template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const ReadParams p) {
  constexpr uint32_t L = D / 8, kRows = kRowThreads / L;
  const uint32_t seq = blockIdx.x / p.blocks, block = blockIdx.x % p.blocks, lane = threadIdx.x % L;
  const uint32_t items = p.tokens * p.c.kv_heads;
  const int64_t first = p.first ? p.first[seq] : 0;
  const int64_t held = min(max(p.c.state[seq].rows, 0), (int32_t)p.c.capacity);
  const uint8_t *seq_run = p.c.data + (size_t)seq * p.c.kv_heads * p.c.tiles * Kv4<D>::kTileBytes;
  T *k = (T *)p.k + (size_t)seq * items * D + lane * 8, *v = (T *)p.v + (size_t)seq * items * D + lane * 8;
  for (uint32_t base = block * kRows * 2; base < items; base += p.blocks * kRows * 2) {
    uint32_t w[2][2] = {};
    __half d[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t item = base + u * kRows + threadIdx.x / L;
      const uint32_t token = item / p.c.kv_heads, head = item - token * p.c.kv_heads;
      const int64_t row = first + token;
      d[u][0] = d[u][1] = __half(0.f);
      if (item < items && row >= 0 && row < held) {
        const uint8_t *run = seq_run + (size_t)head * p.c.tiles * Kv4<D>::kTileBytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          w[u][i] = *((const uint32_t *)(run + Kv4<D>::codes((uint32_t)row, i)) + lane);
          d[u][i] = *(const __half *)(run + Kv4<D>::scales((uint32_t)row, i) + lane / 4 * 2);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t item = base + u * kRows + threadIdx.x / L;
      if (item >= items) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 d2 = __half2half2(d[u][i]);
        __half2 h[4];
        unpack8(w[u][i], d2, minus72(d2), h);
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __low2float(h[j]), x[j + 4] = __high2float(h[j]);
        store8((i ? v : k) + (size_t)item * D, x);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
struct EvictParams {
  Kv4View c;
  Kv4Seq *state_out;
  float *weights_out;
  int32_t *positions_out;
  uint32_t budget, recent, sinks, list;  // list: entries of each row list in shared memory
};

constexpr uint32_t kEvictThreads = 512, kEvictWarps = kEvictThreads / 32, kEvictBins = 2048;
constexpr uint32_t kEvictSmem = 200 * 1024;

// Rank of a row: larger is kept first. Protected rows come before all others; a
// NaN weight ranks last. -0 and +0 rank alike.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t pos, int32_t next, uint32_t recent, uint32_t sinks) {
  if ((int64_t)pos >= (int64_t)next - (int64_t)recent || (int64_t)pos < (int64_t)sinks) return 0xFFFFFFFFu;
  if (!(w == w)) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix over the warps of one count a warp, and the total. Two counts
// of up to 16 bits may share a word.
__device__ __forceinline__ uint32_t warps_before(uint32_t mine, uint32_t *counts, uint32_t &total) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  __syncthreads();
  if (lane == 0) counts[warp] = mine;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (uint32_t i = 0; i < kEvictWarps; ++i) {
    const uint32_t n = counts[i];
    before += i < warp ? n : 0;
    total += n;
  }
  return before;
}

// One block per (sequence, head). A radix selection over 11, 11 and 10 bits of
// the keys finds the key of the last row kept and how many rows of that key stay
// (the lowest ones). Attention does not depend on the order of rows, so nothing
// is compacted: kept rows past the budget move, in order, into the places of
// dropped rows before it, and every other row stays where it is. Sources lie
// past the budget and destinations before it, so the moves need no order.
//
// 448 heads of 4096 rows cut to 1024 take 60 us: 20 us of selection, then moves that
// read and write 147 MB (117 MB if no sector were read for 8 bytes of scales). One
// row of 2049 in 32 heads takes 9.4 us, dependent passes over shared memory.
//
// KEYS: the keys fit in shared memory, else they are computed again from the
// weights and positions for every pass. Each warp ranks a contiguous run of
// rows with ballots, so a pass over the rows has no block barrier.
template <int D, bool KEYS>
__global__ void __launch_bounds__(kEvictThreads, 4) kv4_evict_kernel(const EvictParams p) {
  extern __shared__ __align__(16) uint32_t evict_smem[];   // histogram (read 16 bytes at a time), keys, holes, movers
  __shared__ uint32_t counts[kEvictWarps], chosen[2];
  uint32_t *hist = evict_smem, *keys = hist + kEvictBins;
  uint16_t *holes = (uint16_t *)(keys + (KEYS ? p.c.capacity : 0)), *movers = holes + p.list;
  const uint32_t tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const uint32_t lane_row = blockIdx.x, seq = lane_row / p.c.kv_heads;
  Kv4Seq *st = p.c.state + seq;
  const int4 s = *(const int4 *)st;
  const uint32_t n = min((uint32_t)max(s.x, 0), p.c.capacity), budget = p.budget;
  const size_t at = (size_t)lane_row * p.c.capacity;
  const float *w = p.c.weights + at;
  const int32_t *pos = p.c.positions + at;
  float *w_out = p.weights_out + at;
  int32_t *pos_out = p.positions_out + at;
  const bool copy = p.weights_out != p.c.weights;
  if (n <= budget) {
    if (copy)
      for (uint32_t i = tid; i < n; i += kEvictThreads) w_out[i] = w[i], pos_out[i] = pos[i];
  } else {
    auto key_of = [&](uint32_t i) { return KEYS ? keys[i] : evict_key(w[i], pos[i], s.y, p.recent, p.sinks); };
    uint32_t prefix = 0, need = budget;  // rows still to take among those whose high bits are `prefix`
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, top = pass == 1 ? 21 : 10;
      const uint32_t mask = pass == 2 ? 1023u : 2047u;
      for (uint32_t i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (uint32_t i = tid; i < n; i += kEvictThreads) {
        uint32_t key;
        if (pass == 0) {
          key = evict_key(w[i], pos[i], s.y, p.recent, p.sinks);
          if constexpr (KEYS) keys[i] = key;
        } else {
          key = key_of(i);
        }
        if (pass == 0 || key >> top == prefix >> top) atomicAdd(&hist[key >> shift & mask], 1u);
      }
      __syncthreads();
      // thread t's bins, from the largest digit down: 2047 - 4t .. 2044 - 4t
      const uint4 b = ((const uint4 *)hist)[kEvictBins / 4 - 1 - tid];
      uint32_t sum = b.x + b.y + b.z + b.w, all = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, all, o);
        if (lane >= (uint32_t)o) all += up;
      }
      if (lane == 31) counts[warp] = all;
      __syncthreads();
#pragma unroll
      for (uint32_t i = 0; i < kEvictWarps; ++i) all += i < warp ? counts[i] : 0;
      if (all >= need && all - sum < need) {   // one thread
        uint32_t left = need - (all - sum), digit = kEvictBins - 1 - 4 * tid;
        const uint32_t bins[4] = {b.w, b.z, b.y, b.x};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          if (bins[i] >= left) break;
          left -= bins[i];
          --digit;
        }
        chosen[0] = digit;
        chosen[1] = left;
      }
      __syncthreads();
      prefix |= chosen[0] << shift;
      need = chosen[1];
    }
    // rows of this warp
    const uint32_t run_rows = (n + kEvictThreads - 1) / kEvictThreads * 32;
    const uint32_t begin = min(n, warp * run_rows), end = min(n, begin + run_rows);
    const uint32_t below = (1u << lane) - 1;
    uint32_t same = 0, total;
    for (uint32_t base = begin; base < end; base += 32) {
      const uint32_t i = base + lane;
      same += __popc(__ballot_sync(~0u, i < end && key_of(i) == prefix));
    }
    same = warps_before(same, counts, total);
    // f(row, kept, place among the holes, place among the movers) for every row of this warp
    auto walk = [&](uint32_t rank, uint32_t hole, uint32_t mover, auto &&f) {
      for (uint32_t base = begin; base < end; base += 32) {
        const uint32_t i = base + lane;
        const uint32_t key = i < end ? key_of(i) : 0;
        const uint32_t eq = __ballot_sync(~0u, i < end && key == prefix);
        const bool keep = i < end && (key > prefix || (key == prefix && rank + __popc(eq & below) < need));
        const uint32_t h = __ballot_sync(~0u, i < end && i < budget && !keep);
        const uint32_t m = __ballot_sync(~0u, i >= budget && keep);
        f(i, keep, h >> lane & 1 ? hole + __popc(h & below) : ~0u, m >> lane & 1 ? mover + __popc(m & below) : ~0u);
        rank += __popc(eq);
        hole += __popc(h);
        mover += __popc(m);
      }
      return hole | mover << 16;
    };
    // holes and movers number at most 32768 each (the list's size); a warp's count needs 16 bits
    uint32_t both = walk(same, 0, 0, [](uint32_t, bool, uint32_t, uint32_t) {});
    both = warps_before(both, counts, total);
    walk(same, both & 0xFFFF, both >> 16, [&](uint32_t i, bool keep, uint32_t hole, uint32_t mover) {
      if (hole < p.list) holes[hole] = (uint16_t)i;
      if (mover < p.list) movers[mover] = (uint16_t)i;
      if (copy && keep && i < budget) w_out[i] = w[i], pos_out[i] = pos[i];
    });
    __syncthreads();
    const uint32_t moves = min(min(total & 0xFFFF, total >> 16), p.list);
    for (uint32_t i = tid; i < moves; i += kEvictThreads) {
      w_out[holes[i]] = w[movers[i]];
      pos_out[holes[i]] = pos[movers[i]];
    }
    // a row is D/32 pieces of 16 code bytes and one of D/16 scale bytes, twice
    constexpr uint32_t kPieces = D / 32 + 1;
    uint8_t *run = p.c.data + (size_t)lane_row * p.c.tiles * Kv4<D>::kTileBytes;
#pragma unroll 4
    for (uint32_t i = tid; i < moves * 2 * kPieces; i += kEvictThreads) {
      const uint32_t m = i / (2 * kPieces), piece = i % kPieces;
      const int v = i / kPieces & 1;
      const uint32_t from = movers[m], to = holes[m];
      if (piece < D / 32) {
        *(uint4 *)(run + Kv4<D>::codes(to, v) + piece * 16) = *(const uint4 *)(run + Kv4<D>::codes(from, v) + piece * 16);
      } else {
        using S = typename std::conditional<D == 128, uint2, uint32_t>::type;
        *(S *)(run + Kv4<D>::scales(to, v)) = *(const S *)(run + Kv4<D>::scales(from, v));
      }
    }
  }
  // the last head of a sequence to finish sets its rows: every head has read them by then
  if (tid == 0 && atomicAdd((uint32_t *)&st->ticket, 1u) == p.c.kv_heads - 1) {
    *(int4 *)(p.state_out + seq) = make_int4((int)min(n, budget), s.y, s.z, 0);
    if (p.state_out != p.c.state) st->ticket = 0;
  }
}

}  // namespace vg
