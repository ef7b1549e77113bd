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

constexpr uint32_t kRowThreads = 256;

// One lane quantises 8 channels of a K row and of the V row beside it; the four
// lanes of a block agree on its extremes by shuffles. Bound by the input's
// bytes: each value is read once, and the stores are 0.56 bytes a value.
//
// The rows held are advanced by the last block of a sequence to finish (every
// block has read them by then), so one launch does the whole append.
template <int D, typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const AppendParams p) {
  constexpr uint32_t L = D / 8;                  // lanes of a row
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
  bool odd = false;  // met a NaN or an infinity
  for (uint32_t base = block * kRows; base < items; base += p.blocks * kRows) {
    const uint32_t item = base + threadIdx.x / L;
    const bool on = item < items;
    const uint32_t token = on ? item / p.c.kv_heads : 0, head = on ? item % p.c.kv_heads : 0;
    float x[2][8];
    load8<T, VEC>((const T *)p.k + (int64_t)seq * p.ks.seq + (int64_t)token * p.ks.token + (int64_t)head * p.ks.head + lane * 8, x[0]);
    load8<T, VEC>((const T *)p.v + (int64_t)seq * p.vs.seq + (int64_t)token * p.vs.token + (int64_t)head * p.vs.head + lane * 8, x[1]);
    const uint32_t row = (uint32_t)at + token;
    const size_t lane_row = (size_t)seq * p.c.kv_heads + head;
    uint8_t *run = p.c.data + lane_row * p.c.tiles * Kv4<D>::kTileBytes;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      float high = -kKv4Largest, low = kKv4Largest;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y = x[v][i];
        odd |= on && !(fabsf(y) < __int_as_float(0x7f800000));
        y = y == y ? fminf(fmaxf(y, -kKv4Largest), kKv4Largest) : 0.f;
        x[v][i] = y;
        high = fmaxf(high, y);
        low = fminf(low, y);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        high = fmaxf(high, __shfl_xor_sync(~0u, high, o));
        low = fminf(low, __shfl_xor_sync(~0u, low, o));
      }
      const float d = kv4_scale(high, low);
      const float inv = d == 0.f ? 0.f : __frcp_rn(d);
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float n = fminf(fmaxf(rintf(x[v][i] * inv), -8.f), 7.f);
        w |= (uint32_t)((int32_t)n + 8) << (4 * i);
      }
      if (on) {
        *(uint32_t *)(run + Kv4<D>::codes(row, v) + lane * 4) = w;
        if (lane % 4 == 0) *(__half *)(run + Kv4<D>::scales(row, v) + lane / 4 * 2) = __float2half_rn(d);
      }
    }
    if (on && lane == 0) {
      if (p.c.weights) p.c.weights[lane_row * p.c.capacity + row] = 0.f;
      if (p.c.positions) p.c.positions[lane_row * p.c.capacity + row] = s.y - s.x + at + (int32_t)token;
    }
  }
  if (__syncthreads_or(odd) && threadIdx.x == 0) atomicOr(&st->status, kKv4NonFinite);
  if (threadIdx.x == 0) {
    uint32_t done = 0;
    if (p.blocks > 1) {
      __threadfence();
      done = atomicAdd((uint32_t *)&st->ticket, 1u);
    }
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
  uint32_t tokens;
};

// The values of rows [first, first + tokens) of every sequence; rows that a
// sequence does not hold read as 0. One lane unpacks 8 channels of K and of V.
template <int D, typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const ReadParams p) {
  constexpr uint32_t L = D / 8;
  const uint64_t items = (uint64_t)p.c.seqs * p.tokens * p.c.kv_heads;
  const uint64_t item = (uint64_t)blockIdx.x * (kRowThreads / L) + threadIdx.x / L;
  if (item >= items) return;
  const uint32_t lane = threadIdx.x % L;
  const uint32_t head = (uint32_t)(item % p.c.kv_heads);
  const uint64_t r = item / p.c.kv_heads;
  const uint32_t token = (uint32_t)(r % p.tokens), seq = (uint32_t)(r / p.tokens);
  const int64_t row = (int64_t)(p.first ? p.first[seq] : 0) + token;
  const bool on = row >= 0 && row < p.c.state[seq].rows && row < (int64_t)p.c.capacity;
  const uint8_t *run = p.c.data + ((size_t)seq * p.c.kv_heads + head) * p.c.tiles * Kv4<D>::kTileBytes;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    float x[8] = {};
    if (on) {
      const uint32_t w = __ldg((const uint32_t *)(run + Kv4<D>::codes((uint32_t)row, v)) + lane);
      const __half2 d = __half2half2(*(const __half *)(run + Kv4<D>::scales((uint32_t)row, v) + lane / 4 * 2));
      __half2 h[4];
      unpack8(w, d, minus72(d), h);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __low2float(h[i]), x[i + 4] = __high2float(h[i]);
    }
    store8((T *)(v ? p.v : p.k) + item * D + lane * 8, x);
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

constexpr uint32_t kEvictThreads = 512;

// Rank of a row: larger is kept first. Protected rows come before all others; a
// NaN weight ranks last. -0 and +0 rank alike.
__device__ __forceinline__ uint32_t evict_key(float w, int32_t pos, int32_t next, uint32_t recent, uint32_t sinks) {
  if ((int64_t)pos >= (int64_t)next - (int64_t)recent || (int64_t)pos < (int64_t)sinks) return 0xFFFFFFFFu;
  if (!(w == w)) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix of a 0/1 flag over the block in thread order, plus its total.
__device__ __forceinline__ uint32_t block_rank(bool flag, uint32_t *warp_sums, uint32_t &total) {
  const uint32_t m = __ballot_sync(~0u, flag), lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  if (lane == 0) warp_sums[warp] = __popc(m);
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (uint32_t i = 0; i < kEvictThreads / 32; ++i) {
    const uint32_t n = warp_sums[i];
    before += i < warp ? n : 0;
    all += n;
  }
  __syncthreads();
  total = all;
  return before + __popc(m & ((1u << lane) - 1));
}

// One block per (sequence, head). A radix selection over 8 bits at a time finds
// the key of the last row kept and how many rows of that key stay (the lowest
// ones). Attention does not depend on the order of rows, so nothing is
// compacted: kept rows past the budget move, in order, into the places of
// dropped rows before it, and every other row stays where it is. Sources lie
// past the budget and destinations before it, so the moves need no order.
template <int D>
__global__ void __launch_bounds__(kEvictThreads) kv4_evict_kernel(const EvictParams p) {
  extern __shared__ uint16_t lists[];  // holes, then movers
  __shared__ uint32_t hist[256], sums[kEvictThreads / 32], chosen[2];
  uint16_t *holes = lists, *movers = lists + p.list;
  const uint32_t tid = threadIdx.x, lane_row = blockIdx.x, seq = lane_row / p.c.kv_heads;
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
    uint32_t prefix = 0, need = budget;  // rows still to take among those whose high bits are `prefix`
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (uint32_t i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (uint32_t i = tid; i < n; i += kEvictThreads) {
        const uint32_t key = evict_key(w[i], pos[i], s.y, p.recent, p.sinks);
        if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[key >> shift & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t left = need;
        int b = 255;
        for (; b > 0 && hist[b] < left; --b) left -= hist[b];
        chosen[0] = (uint32_t)b;
        chosen[1] = left;
      }
      __syncthreads();
      prefix |= chosen[0] << shift;
      need = chosen[1];
    }
    uint32_t equal = 0, n_holes = 0, n_movers = 0;
    for (uint32_t base = 0; base < n; base += kEvictThreads) {
      const uint32_t i = base + tid;
      const uint32_t key = i < n ? evict_key(w[i], pos[i], s.y, p.recent, p.sinks) : 0;
      uint32_t total;
      const bool same = i < n && key == prefix;
      const uint32_t rank = equal + block_rank(same, sums, total);
      equal += total;
      const bool keep = i < n && (key > prefix || (same && rank < need));
      const bool hole = i < budget && !keep, mover = i >= budget && keep;
      uint32_t k = n_holes + block_rank(hole, sums, total);
      if (hole && k < p.list) holes[k] = (uint16_t)i;
      n_holes += total;
      k = n_movers + block_rank(mover, sums, total);
      if (mover && k < p.list) movers[k] = (uint16_t)i;
      n_movers += total;
      if (copy && keep && i < budget) w_out[i] = w[i], pos_out[i] = pos[i];
    }
    __syncthreads();
    const uint32_t moves = min(min(n_holes, n_movers), p.list);
    for (uint32_t i = tid; i < moves; i += kEvictThreads) {
      w_out[holes[i]] = w[movers[i]];
      pos_out[holes[i]] = pos[movers[i]];
    }
    // a row is D/32 pieces of 16 code bytes and one of D/16 scale bytes, twice
    constexpr uint32_t kPieces = D / 32 + 1;
    uint8_t *run = p.c.data + (size_t)lane_row * p.c.tiles * Kv4<D>::kTileBytes;
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
  // the last head of a sequence to finish sets its rows
  if (tid == 0) {
    __threadfence();
    if (atomicAdd((uint32_t *)&st->ticket, 1u) == p.c.kv_heads - 1) {
      *(int4 *)(p.state_out + seq) = make_int4((int)min(n, budget), s.y, st->status, 0);
      if (p.state_out != p.c.state) st->ticket = 0;
    }
  }
}

}  // namespace vg
