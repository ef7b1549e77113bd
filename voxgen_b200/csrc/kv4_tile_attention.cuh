// Attention of many query rows over a 4-bit cache: drafts and prompts, on tcgen05.
//
// The mathematics. The query rows of a (sequence, KV head) are packed: row
// r = token * group + head of the group, so a token's whole group shares the
// cache's rows. A tile is 128 query rows (M) against 128 cache rows (N):
//   S = Q K^T     128 x 128 x D, both operands in shared memory
//   P = exp2(S * f - m)          a thread a row, S and P in tensor memory
//   O += P V      128 x D x 128, P from tensor memory, V in shared memory
// K and V are unpacked from their codes to fp16 exactly (kv4.cuh), so a 32-bit
// call needs hi + lo only of its own operands: Q hi and lo against the same K,
// P hi and lo against the same V, 4 products instead of 2. 16-bit queries are
// exact in fp16 (times a power of two), and P is rounded to 11 bits, like the
// output. Statistics and sums are fp32. The running maximum is raised, and O
// rescaled, only when a score passes it by 2^8.
//
// The layout. K and V tiles are stored the same way: 128 cache rows of 64
// channels (128 bytes) a panel, 16-byte chunks turned by the row (the 128-byte
// swizzle). For S that is a K-major operand; for O the same bytes are an
// MN-major one, so V needs no transpose. A chunk is one word of codes, unpacked
// in the order 0 4 1 5 2 6 3 7: Q's channels are stored in that order, and O's
// columns come out in it.
//
// The roles. Two softmax warpgroups, each with its own S and O in tensor memory
// (4 x 128 columns), one warp that issues the products, three that unpack. With
// more than 128 rows of 16-bit queries the groups hold two query tiles, and an
// unpacked tile serves 256 rows; otherwise they take every other cache tile of
// one query tile and their results are added at the end. The products of one
// group run while the other does its softmax. Bound: at head_dim 128 a tile's two
// products take as long as its 16,384 exponentials; unpacking hides behind both.
//
// The split. Units of 128 cache rows, of all (sequence, query rows, KV head)
// segments in order, are dealt out evenly to one CTA per SM. A segment that spans
// CTAs leaves a partial result per CTA; the CTA that finishes last (a counter,
// left at zero) adds them in order.
#pragma once
#include "kv4_rows_attention.cuh"

namespace vg {

constexpr uint32_t kTileM = 128, kTileN = 128;
constexpr uint32_t kTileThreads = 384;          // 8 softmax warps, 1 of products, 3 that unpack
constexpr uint32_t kUnpackThreads = 96;
constexpr uint32_t kTileCtas = 148;
constexpr uint32_t kRawStages = 3;
constexpr float kTilePScale = 6.f;              // as kPScale: P below 2^14 with a lead of 2^8

template <int D>
struct TileSmem {
  static constexpr uint32_t kOperand = kTileN * D * 2;          // a K, V or Q tile
  static constexpr uint32_t kQ = 0;                             // 2: two tiles, or hi and lo
  static constexpr uint32_t kK = 2 * kOperand, kV = 4 * kOperand;   // 2 stages each
  static constexpr uint32_t kRaw = 6 * kOperand;
  static constexpr uint32_t kRawStage = Kv4<D>::kTileBytes;
  static constexpr uint32_t kBytes = kRaw + kRawStages * kRawStage + 1024;   // + alignment
};

template <int D>
constexpr uint32_t kTilePart = 2 * kTileM * (D + 2);   // floats of a partial result

// ---- tcgen05 ----
__device__ __forceinline__ void tmem_alloc512(uint32_t *where) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(where)) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free512(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(addr));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(add)
      : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float *x) {
  uint32_t *r = (uint32_t *)x;
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Registers that a tensor-memory load has filled, tied to the point after the wait.
template <int N>
__device__ __forceinline__ void loaded(float (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(x[i]));
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand descriptor: 128-byte swizzle; lbo: bytes between panels
// (MN-major only), 8-row groups are 1024 bytes apart.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lbo) {
  return (uint64_t)(addr >> 4 & 0x3FFF) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// fp16 operands, fp32 accumulator, M = 128; b_mn: B is MN-major.
constexpr uint32_t tile_idesc(uint32_t n, bool b_mn) {
  return 1u << 4 | (b_mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (kTileM >> 4) << 24;
}

// ---- the work of a CTA ----
// A block is the query rows of a sequence that a CTA takes at a time (kRows of
// them); each block has a segment per KV head.
struct TileWork {
  uint32_t seq, block, kv;
  uint32_t first, units, seg_units;   // cache tiles of this piece, and of its segment
};
template <uint32_t kRows>
__device__ __forceinline__ uint32_t tile_units(const Kv4AttnParams &p, uint32_t seq, uint32_t block) {
  // the last of the block's tokens that the sequence has sees the most rows
  const uint32_t held = kv4_held(p.c, seq), rows = p.tokens * p.group;
  const int32_t count = kv4_count(p, seq);
  const int32_t tok = min((int32_t)((min(rows, (block + 1) * kRows) - 1) / p.group), count - 1);
  const int32_t seen = (int32_t)held - count + tok + 1;
  return (uint32_t)(max(seen, 1) + (int32_t)kTileN - 1) / kTileN;
}
// Total units, and (found) the piece that starts at unit x.
template <uint32_t kRows>
__device__ __forceinline__ uint32_t tile_total(const Kv4AttnParams &p) {
  uint32_t n = 0;
#pragma unroll 1
  for (uint32_t i = threadIdx.x % 32; i < p.c.seqs * p.row_tiles; i += 32)
    n += tile_units<kRows>(p, i / p.row_tiles, i % p.row_tiles);
  return __reduce_add_sync(~0u, n) * p.c.kv_heads;
}
template <uint32_t kRows>
__device__ __forceinline__ TileWork tile_find(const Kv4AttnParams &p, uint32_t x) {
  const uint32_t lane = threadIdx.x % 32, blocks = p.c.seqs * p.row_tiles;
  uint32_t before = 0;
#pragma unroll 1
  for (uint32_t base = 0; base < blocks; base += 32) {
    const uint32_t i = base + lane;
    const uint32_t u = i < blocks ? tile_units<kRows>(p, i / p.row_tiles, i % p.row_tiles) : 0;
    uint32_t sum = u * p.c.kv_heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(~0u, sum, o);
      if (lane >= (uint32_t)o) sum += up;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > x);
    if (past) {
      const int at = __ffs(past) - 1;
      const uint32_t units = __shfl_sync(~0u, u, at);
      const uint32_t into = x - before - (__shfl_sync(~0u, sum, at) - units * p.c.kv_heads);
      TileWork w;
      w.seq = (base + at) / p.row_tiles;
      w.block = (base + at) % p.row_tiles;
      w.kv = into / units;
      w.first = into - w.kv * units;
      w.units = w.seg_units = units;
      return w;
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return TileWork{0, 0, 0, 0, 1, 1};
}

struct TileBars {
  uint64_t q_full, s_full[2], p_full[2], o_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], raw_full[kRawStages], drained;
};

// What the softmax groups do when a piece ends: join the groups' results where
// they shared a query tile, then finish the rows, or leave a partial result and,
// last of the segment's CTAs, add them all. 256 threads.
template <int D, typename T>
__device__ __forceinline__ void tile_results(const Kv4AttnParams &p, const TileWork &w, uint32_t at, bool pair, uint32_t x,
                                             uint32_t row, uint32_t row0, float m, float l, bool mine, uint32_t o_addr,
                                             float *shared_o, float *other_max, float *other_sum, uint32_t *last,
                                             uint32_t c0, uint32_t c1) {
  constexpr uint32_t kChunks = D / 4;   // 16-byte chunks of a row
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, rows = p.tokens * p.group;
  const uint32_t block_rows = min(pair ? 2 * kTileM : kTileM, rows - row0);
  const bool whole = w.units == w.seg_units;
  float w0 = 1.f, w1 = 0.f;
  if (!pair) {
    if (x == 1) {
      other_max[row] = mine ? m : -INFINITY;
      other_sum[row] = mine ? l : 0.f;
      if (mine) {
#pragma unroll 1
        for (uint32_t c = 0; c < D; c += 32) {
          float o[32];
          tmem_load32(o_addr + c, o);
          tmem_wait_load();
          loaded(o);
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i)
            ((float4 *)shared_o)[row * kChunks + ((c / 4 + i) ^ (row % kChunks))] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
    }
    named_bar(2, 256);
    if (x == 0) {
      const float om = other_max[row], top = fmaxf(m, om);
      w0 = m == -INFINITY ? 0.f : exp2_fast(m - top);
      w1 = om == -INFINITY ? 0.f : exp2_fast(om - top);
      l = l * w0 + other_sum[row] * w1;
      m = top;
    }
  }
  const uint32_t r = pair ? x * kTileM + row : row;   // row of the block
  const bool writer = (pair || x == 0) && r < block_rows;
  auto place = [&](uint32_t i) {
    const uint32_t tok = (row0 + i) / p.group, head = w.kv * p.group + (row0 + i) % p.group;
    return ((size_t)w.seq * p.tokens + tok) * p.heads + head;
  };
  auto lse = [&](float top, float sum) { return sum == 0.f ? INFINITY : top + log2f(sum) - kTilePScale; };
  auto slot = [&](uint32_t i) { return p.parts + (size_t)i * kTilePart<D>; };
  float *part = slot(blockIdx.x * 2 + (w.first == 0));
  const bool joined = !pair && w.units > 1;           // group 1 had a tile
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (pair || x == 0) {   // whole warps: the loads are collective
#pragma unroll 1
    for (uint32_t c = 0; c < D; c += 32) {
      float o[32];
      tmem_load32(o_addr + c, o);
      tmem_wait_load();
      loaded(o);
      if (writer && joined) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          const float4 y = ((const float4 *)shared_o)[row * kChunks + ((c / 4 + i) ^ (row % kChunks))];
          o[4 * i] = o[4 * i] * w0 + y.x * w1, o[4 * i + 1] = o[4 * i + 1] * w0 + y.y * w1;
          o[4 * i + 2] = o[4 * i + 2] * w0 + y.z * w1, o[4 * i + 3] = o[4 * i + 3] * w0 + y.w * w1;
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < 32; i += 8) {   // columns hold channels 0 4 1 5 2 6 3 7
        const float z[8] = {o[i], o[i + 2], o[i + 4], o[i + 6], o[i + 1], o[i + 3], o[i + 5], o[i + 7]};
        if (writer && whole) {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = z[k] * inv;
          store8((T *)p.out + place(r) * D + c + i, y);
        } else if (writer) {
          store8(part + r * D + c + i, z);
        }
      }
      __syncwarp();
    }
    if (writer) {
      if (!whole) {
        part[2 * kTileM * D + r] = m;
        part[2 * kTileM * (D + 1) + r] = l;
      } else if (p.lse) {
        p.lse[place(r)] = lse(m, l);
      }
    }
  }
  if (!whole) {
    const uint32_t pieces = c1 - c0 + 1;
    named_bar(2, 256);
    if (threadIdx.x == 0) {
      *last = atomic_add_acq_rel(p.tickets + c0, 1u) == pieces - 1;   // a CTA begins at most one segment that others finish
      if (*last) p.tickets[c0] = 0;
    }
    named_bar(2, 256);
    if (*last) {
      constexpr uint32_t N = D / 32;
      auto piece = [&](uint32_t i) { return (const float *)slot((c0 + i) * 2 + (i == 0)); };
#pragma unroll 1
      for (uint32_t i = warp; i < block_rows; i += 8) {
        float top = -INFINITY, sum = 0.f, y[N] = {};
#pragma unroll 4
        for (uint32_t k = 0; k < pieces; ++k) top = fmaxf(top, __ldcg(piece(k) + 2 * kTileM * D + i));
#pragma unroll 4
        for (uint32_t k = 0; k < pieces; ++k) {
          const float pm = __ldcg(piece(k) + 2 * kTileM * D + i), pw = pm == -INFINITY ? 0.f : exp2_fast(pm - top);
          sum += pw * __ldcg(piece(k) + 2 * kTileM * (D + 1) + i);
#pragma unroll
          for (uint32_t j = 0; j < N; ++j) y[j] += pw * __ldcg(piece(k) + i * D + j * 32 + lane);
        }
        const float f = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) ((T *)p.out)[place(i) * D + j * 32 + lane] = from_float<T>(y[j] * f);
        if (p.lse && lane == 0) p.lse[place(i)] = lse(top, sum);
      }
    }
  }
  named_bar(2, 256);   // Q's place and the shared words may change
}

template <int D, typename T>
__global__ void __launch_bounds__(kTileThreads, 1) kv4_tile_kernel(const Kv4AttnParams p) {
  using S = TileSmem<D>;
  constexpr bool kSplit = sizeof(T) == 4;
  constexpr uint32_t kRows = kSplit ? kTileM : 2 * kTileM;    // query rows of a block
  constexpr uint32_t kPanel = kTileN * 128;                   // bytes of 64 channels of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ TileBars bars;
  __shared__ uint32_t tmem_base, aborted, last;
  __shared__ float factors[2 * kTileM], other_max[kTileM], other_sum[kTileM];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rows = p.tokens * p.group;

  const uint32_t total = tile_total<kRows>(p);
  const uint32_t ctas = min(gridDim.x, total);
  if (blockIdx.x >= ctas) return;
  const uint32_t each = total / ctas, more = total - each * ctas;   // the first `more` CTAs have one unit more
  const uint32_t begin = each * blockIdx.x + min(blockIdx.x, more), end = begin + each + (blockIdx.x < more);
  auto owner = [&](uint32_t x) { return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each; };

  if (threadIdx.x == 0) {
    mbar_init(&bars.q_full, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], kTileM);
      mbar_init(&bars.o_full[i], 1);
      mbar_init(&bars.k_full[i], kUnpackThreads);
      mbar_init(&bars.k_empty[i], 1);
      mbar_init(&bars.v_full[i], kUnpackThreads);
      mbar_init(&bars.v_empty[i], 1);
    }
    for (uint32_t i = 0; i < kRawStages; ++i) mbar_init(&bars.raw_full[i], 1);
    mbar_init(&bars.drained, 1);
    fence_mbar_init();
    aborted = 0;
  }
  if (warp == 8) tmem_alloc512(&tmem_base);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t *)&tmem_base;
  // a wait that runs out makes every later one return at once: the roles then run to their ends on whatever is there
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity) || *(volatile uint32_t *)&aborted) return;
    if (!mbar_wait_bounded(bar, parity)) *(volatile uint32_t *)&aborted = 1;
  };
  // two query tiles, or one whose cache tiles the softmax groups share
  auto paired = [&](const TileWork &w) { return !kSplit && rows - w.block * kRows > kTileM; };
  // f(work, its place in the CTA's units) for every piece of this CTA
  const TileWork first_work = tile_find<kRows>(p, begin);   // the whole warp takes part
  auto each_work = [&](auto &&f) {
    TileWork w = first_work;
#pragma unroll 1
    for (uint32_t at = begin; at < end;) {
      w.units = min(end - at, w.seg_units - w.first);
      f(w, at);
      at += w.units;
      w.first = 0;
      if (at < end && ++w.kv == p.c.kv_heads) {
        w.kv = 0;
        if (++w.block == p.row_tiles) w.block = 0, ++w.seq;
        w.seg_units = tile_units<kRows>(p, w.seq, w.block);
      }
    }
  };

  if (warp == 8) {
    // ---------------- products ----------------
    if (lane == 0) {
      const uint32_t q = smem_u32(smem + S::kQ), k = smem_u32(smem + S::kK), v = smem_u32(smem + S::kV);
      constexpr uint32_t kScoreDesc = tile_idesc(kTileN, false), kValueDesc = tile_idesc(D, true);
      uint32_t works = 0, tiles = 0, jobs[2] = {0, 0};   // jobs: of each group
      each_work([&](const TileWork &w, uint32_t) {
        const bool pair = paired(w);
        const uint32_t n = pair ? 2 * w.units : w.units;
        wait(&bars.q_full, works++ & 1);
        tc_fence_after();
#pragma unroll 1
        for (uint32_t j = 0; j <= n; ++j) {
          if (j < n) {   // scores of job j
            const uint32_t x = j & 1, tile = tiles + (pair ? j >> 1 : j), st = tile & 1;
            if (!pair || x == 0) {
              wait(&bars.k_full[st], tile >> 1 & 1);
              tc_fence_after();
            }
            const uint32_t d = tmem + x * 128, qa = q + (pair ? x * S::kOperand : 0), ka = k + st * S::kOperand;
#pragma unroll
            for (uint32_t c = 0; c < D / 16; ++c) {
              const uint32_t off = c / 4 * kPanel + c % 4 * 32;
              mma_ss(d, operand(qa + off, 0), operand(ka + off, 0), kScoreDesc, c > 0);
              if constexpr (kSplit) mma_ss(d, operand(qa + S::kOperand + off, 0), operand(ka + off, 0), kScoreDesc, 1);
            }
            tc_commit(&bars.s_full[x]);
            if (!pair || x == 1) tc_commit(&bars.k_empty[st]);
          }
          if (j > 0) {   // values of job j - 1
            const uint32_t i = j - 1, x = i & 1, tile = tiles + (pair ? i >> 1 : i), st = tile & 1;
            wait(&bars.p_full[x], jobs[x] & 1);
            if (!pair || x == 0) wait(&bars.v_full[st], tile >> 1 & 1);
            tc_fence_after();
            const uint32_t d = tmem + 256 + x * 128, pa = tmem + x * 128, va = v + st * S::kOperand;
#pragma unroll
            for (uint32_t c = 0; c < kTileN / 16; ++c) {
              const uint64_t b = operand(va + c * 2048, kPanel);
              mma_ts(d, pa + c * 8, b, kValueDesc, i > 1 || c > 0);
              if constexpr (kSplit) mma_ts(d, pa + 64 + c * 8, b, kValueDesc, 1);
            }
            if (!pair || x == 1) tc_commit(&bars.v_empty[st]);
            if (i + 2 >= n) tc_commit(&bars.o_full[x]);
            ++jobs[x];
          }
        }
        tiles += w.units;
      });
      tc_commit(&bars.drained);   // tensor memory is freed after the last product, even when waits ran out
      mbar_wait_bounded(&bars.drained, 0);
    }
    __syncwarp();
  } else if (warp > 8) {
    // ---------------- unpacking ----------------
    const uint32_t tid = threadIdx.x - 288;
    const size_t run_bytes = (size_t)p.c.tiles * Kv4<D>::kTileBytes;
    // one thread streams the cache's 64-row tiles; a stage is refilled once all have unpacked it
    TileWork ahead = first_work;
    uint32_t ahead_raw = 0, ahead_at = begin, fetched = 0;   // raw: 64-row tile of the piece
    ahead.units = min(end - ahead_at, ahead.seg_units - ahead.first);
    auto fetch = [&]() {
      if (ahead_at >= end || *(volatile uint32_t *)&aborted) return;
      const uint32_t raw = ahead.first * 2 + ahead_raw;
      if (raw < p.c.tiles) {
        const uint32_t st = fetched % kRawStages;
        mbar_arrive_expect_tx(&bars.raw_full[st], S::kRawStage);
        bulk_g2s(smem + S::kRaw + st * S::kRawStage,
                 p.c.data + ((size_t)ahead.seq * p.c.kv_heads + ahead.kv) * run_bytes + (size_t)raw * S::kRawStage, S::kRawStage,
                 &bars.raw_full[st]);
        ++fetched;
      }
      if (++ahead_raw == 2 * ahead.units) {
        ahead_raw = 0;
        ahead_at += ahead.units;
        ahead.first = 0;
        if (ahead_at < end) {
          if (++ahead.kv == p.c.kv_heads) {
            ahead.kv = 0;
            if (++ahead.block == p.row_tiles) ahead.block = 0, ++ahead.seq;
            ahead.seg_units = tile_units<kRows>(p, ahead.seq, ahead.block);
          }
          ahead.units = min(end - ahead_at, ahead.seg_units);
        }
      }
    };
    if (tid == 0) {
      fetch();
      fetch();
      fetch();
    }
    __syncwarp();
    constexpr uint32_t kQuads = D / 32;                 // threads of a row, 32 channels each
    uint32_t tiles = 0, used = 0;
    each_work([&](const TileWork &w, uint32_t) {
      const uint32_t held = kv4_held(p.c, w.seq);
#pragma unroll 1
      for (uint32_t u = 0; u < w.units; ++u, ++tiles) {
        const uint32_t st = tiles & 1, raw0 = (w.first + u) * 2;
        const uint32_t have = raw0 + 1 < p.c.tiles ? 2 : 1;    // a run's last tile may have no second half
        for (uint32_t h = 0; h < have; ++h) wait(&bars.raw_full[(used + h) % kRawStages], (used + h) / kRawStages & 1);
#pragma unroll 1
        for (int v = 0; v < 2; ++v) {
          if (tiles >= 2) wait(v ? &bars.v_empty[st] : &bars.k_empty[st], (tiles >> 1) - 1 & 1);
          uint8_t *dst = smem + (v ? S::kV : S::kK) + st * S::kOperand;
#pragma unroll 1
          for (uint32_t i = tid; i < kTileN * kQuads; i += kUnpackThreads) {
            const uint32_t row = i / kQuads, quad = i % kQuads, h = row / kKv4Tile, r = row % kKv4Tile;
            const uint8_t *src = smem + S::kRaw + (used + (h < have ? h : 0)) % kRawStages * S::kRawStage;
            const uint4 x = *(const uint4 *)(src + Kv4<D>::codes(r, v) + quad * 16);
            __half2 d = __half2half2(*(const __half *)(src + Kv4<D>::scales(r, v) + quad * 2));
            if (raw0 * kKv4Tile + row >= held) d = __half2half2(__half(0.f));   // bytes past the rows held may be anything
            const __half2 d72 = minus72(d);
            // threads of the second panel write their chunks two on, which keeps a row pair's 8 threads off each other
            const bool turn = quad & 2;
            const uint32_t word[4] = {turn ? x.z : x.x, turn ? x.w : x.y, turn ? x.x : x.z, turn ? x.y : x.w};
            uint8_t *out = dst + quad / 2 * kPanel + row * 128;
            const uint32_t chunk = quad % 2 * 4 + (turn ? 2 : 0);
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
              __align__(16) __half2 y[4];
              unpack8(word[k], d, d72, y);
              *(uint4 *)(out + (((chunk & 4) | ((chunk + k) & 3)) ^ (row & 7)) * 16) = *(const uint4 *)y;
            }
          }
          fence_async_smem();
          mbar_arrive(v ? &bars.v_full[st] : &bars.k_full[st]);
        }
        used += have;
        __syncwarp();
        named_bar(1, kUnpackThreads);   // all have read the raw stages
        if (tid == 0)
          for (uint32_t h = 0; h < 2; ++h) fetch();
        __syncwarp();
      }
    });
    // nothing is left in flight but after a wait that ran out
    if (tid == 0)
      for (; used < fetched; ++used) mbar_wait_bounded(&bars.raw_full[used % kRawStages], used / kRawStages & 1);
  } else {
    // ---------------- softmax ----------------
    const uint32_t x = warp / 4, row = threadIdx.x % kTileM;       // group, and its row of the tile
    const uint32_t lanes = (warp % 4) << 21;                       // this warp's lanes of tensor memory
    const uint32_t s_addr = tmem + x * 128 + lanes, o_addr = tmem + 256 + x * 128 + lanes;
    uint32_t done = 0, works = 0;   // tiles of this group, pieces in which it had some
    each_work([&](const TileWork &w, uint32_t at) {
      const bool pair = paired(w);
      const uint32_t row0 = w.block * kRows, held = kv4_held(p.c, w.seq);
      const int32_t count = kv4_count(p, w.seq);
      // ---- Q to shared memory, a warp a row: two tiles, or one (as hi and lo) that both groups load half of ----
      const uint32_t q_rows = pair ? 2 * kTileM : kTileM;
#pragma unroll 1
      for (uint32_t r = warp; r < q_rows; r += 8) {
        constexpr uint32_t N = D / 32;
        float y[N];
        uint32_t top = 0;
        const bool on = row0 + r < rows;
        const uint32_t tok = (row0 + r) / p.group, head = w.kv * p.group + (row0 + r) % p.group;
        const T *src = (const T *)p.q + (int64_t)w.seq * p.qs.seq + (int64_t)tok * p.qs.token + (int64_t)head * p.qs.head + lane * N;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
          y[i] = on ? (float)src[i] : 0.f;
          top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
        }
        float inverse;
        const float power = row_power(__uint_as_float(__reduce_max_sync(~0u, top)), inverse);
        if (lane == 0) factors[r] = fmaxf(p.scale * inverse, 0x1p-126f);
        uint8_t *dst = smem + S::kQ + r / kTileM * S::kOperand;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) {
          const uint32_t c = lane * N + i, place = c % 4 * 2 + c % 8 / 4;   // 0 4 1 5 2 6 3 7
          const uint32_t off = c / 64 * kPanel + r % kTileM * 128 + ((c % 64 / 8) ^ (r & 7)) * 16 + place * 2;
          const float z = y[i] * power;
          const __half hi = __float2half_rn(z);
          *(__half *)(dst + off) = hi;
          if constexpr (kSplit) *(__half *)(dst + S::kOperand + off) = __float2half_rn(z - __half2float(hi));
        }
      }
      fence_async_smem();
      mbar_arrive(&bars.q_full);
      named_bar(2, 256);   // factors
      const uint32_t qr = pair ? x * kTileM + row : row;           // this thread's row of the block
      const float f = factors[qr];
      const uint32_t tok = (row0 + qr) / p.group;
      const int32_t sees = (int32_t)held - count + (int32_t)tok + 1;
      const uint32_t seen = row0 + qr < rows && (int32_t)tok < count && sees > 0 ? (uint32_t)sees : 0u;
      const bool used_row = row0 + qr < rows;
      uint32_t least = used_row ? seen : 0xFFFFFFFFu;              // fewest of the warp's rows
      least = __reduce_min_sync(~0u, least);
      float m = -INFINITY, l = 0.f;
      const uint32_t step = pair ? 1 : 2;
#pragma unroll 1
      for (uint32_t u = pair ? 0 : x; u < w.units; u += step, ++done) {
        wait(&bars.s_full[x], done & 1);
        __syncwarp();
        tc_fence_after();
        float s[kTileN];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_load32(s_addr + c * 32, s + c * 32);
        tmem_wait_load();
        loaded(s);
        const uint32_t first = (w.first + u) * kTileN;
        if (first + kTileN > least) {
#pragma unroll
          for (uint32_t c = 0; c < kTileN; ++c)
            if (first + c >= seen) s[c] = -INFINITY;
        }
        float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int c = 4; c < (int)kTileN; c += 4)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], s[c + i]);
        const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * f;
        if (__any_sync(~0u, best > m + kLead)) {
          const float up = fmaxf(m, best), r = up == m ? 1.f : exp2_fast(m - up);
          m = up;
          l *= r;
          if (u >= step) {   // O has something: the products before these scores are done
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              asm volatile(
                  "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                  : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3]), "=r"(o[4]), "=r"(o[5]), "=r"(o[6]), "=r"(o[7]),
                    "=r"(o[8]), "=r"(o[9]), "=r"(o[10]), "=r"(o[11]), "=r"(o[12]), "=r"(o[13]), "=r"(o[14]), "=r"(o[15])
                  : "r"(o_addr + c));
              tmem_wait_load();
#pragma unroll
              for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(o[i]));
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * r);
              tmem_store16(o_addr + c, o);
            }
          }
        }
        const float base = kTilePScale - (m == -INFINITY ? 0.f : m);
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < (int)kTileN; c += 32) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float a = exp2_fast(fmaf(s[c + 2 * i], f, base)), b = exp2_fast(fmaf(s[c + 2 * i + 1], f, base));
            sum[0] += a, sum[1] += b;
            if constexpr (kSplit) split2(a, b, hi[i], lo[i]);
            else hi[i] = half2_bits(__floats2half2_rn(a, b));
          }
          tmem_store16(s_addr + c / 2, hi);
          if constexpr (kSplit) tmem_store16(s_addr + 64 + c / 2, lo);
        }
        l += sum[0] + sum[1];
        tmem_wait_store();
        tc_fence_before();
        mbar_arrive(&bars.p_full[x]);
      }
      // ---- results ----
      const bool mine = pair || w.units > x;    // this group had a tile
      if (mine) wait(&bars.o_full[x], works++ & 1);
      __syncwarp();
      tc_fence_after();
      const uint32_t seg = at - w.first;
      tile_results<D, T>(p, w, at, pair, x, row, row0, m, l, mine, o_addr, (float *)(smem + S::kQ), other_max, other_sum, &last,
                         owner(seg), owner(seg + w.seg_units - 1));
      tc_fence_before();
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 8) tmem_free512(tmem);
  if (threadIdx.x == 0 && aborted) atomicOr(&p.c.state[0].status, kKv4Timeout);
}

}  // namespace vg
