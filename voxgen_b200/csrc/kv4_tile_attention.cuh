// Attention of many query rows over a 4-bit cache: drafts and prompts, on tcgen05.
//
// The mathematics. The query rows of a (sequence, KV head) are packed: row
// r = token * group + head of the group, so a token's whole group shares the
// cache's rows. A tile is 128 query rows (M) against 128 cache rows (N):
//   S = Q K^T     128 x 128 x D, both operands in shared memory
//   P = exp2((S - m) * f)        a thread a row, S and P in tensor memory
//   O += P V      128 x D x 128, P from tensor memory, V in shared memory
// K and V are unpacked from their codes to fp16 exactly (kv4.cuh), so a 32-bit
// call needs hi + lo only of its own operands: Q hi and lo against the same K,
// P hi and lo against the same V, 4 products instead of 2. 16-bit queries keep
// their bits in fp16 (times a power of two a row; a bf16 value below 2^-28 of its
// row's largest is held to 2^-39 of that). Their P is rounded to 11 bits: hi and lo
// would take fp16 outputs from 2.9e-4 off (a prompt) and 2.5e-4 (a draft) to 2.2e-4
// and 2.1e-4, the output's own rounding, in 1195 us and not 969, 33.6 us and not
// 31.4. Statistics and sums are fp32. The running maximum m is raised, and O
// rescaled, only when a score passes it by 2^8. It is taken off before the scaling
// (kNoScore says why), which costs 1% against one multiply-add with S * f - m.
//
// The layout. K and V tiles are stored the same way: 128 cache rows of 64
// channels (128 bytes) a panel, 16-byte chunks turned by the row (the 128-byte
// swizzle). For S that is a K-major operand; for O the same bytes are an
// MN-major one, so V needs no transpose. A chunk is one word of codes, unpacked
// in the order 0 4 1 5 2 6 3 7: Q's channels are stored in that order, and O's
// columns come out in it.
//
// The roles. Two softmax warpgroups, each with its own S and O in tensor memory
// (4 x 128 columns), a warpgroup that unpacks, and one warp that issues the
// products. With more than 128 rows of 16-bit queries the groups hold two query
// tiles, and an unpacked tile serves 256 rows; otherwise they take every other
// cache tile of one query tile and their results are added at the end. The
// products of one group run while the other does its softmax.
//
// Measured: the last 4096 tokens of a prompt over 32768 rows, fp16, 1.03 TFLOP: 970 us,
// 1.06 PFLOP/s (64% of the measured burst rate). A unit of 256 query rows takes about
// 4000 cycles, of which the products need 2048 and the softmax's 32768 exponentials as
// many; the two wait for each other through S, whose place P takes.
//
// The split. A segment is a block of query rows of a (sequence, KV head) with the
// cache rows it sees, in units of 128. Few segments are cut into pieces of equal
// size, about one for each CTA, since changing segments costs several units; many
// are dealt out evenly to one CTA per SM, in order, unit by unit. A segment that
// is cut leaves partial results; the CTA that finishes it last (a counter, left
// at zero) adds them in order.
#pragma once
#include "kv4_rows_attention.cuh"

namespace vg {

constexpr uint32_t kTileM = 128, kTileN = 128;
constexpr uint32_t kTileThreads = 512;          // 8 softmax warps, 4 that unpack, 1 of products, 3 idle
constexpr uint32_t kUnpackThreads = 128;
// registers of a thread: 512 x 128 at launch, then 2 x 168 + 2 x 88 for the four warpgroups
constexpr uint32_t kSoftmaxRegs = 168, kOtherRegs = 88;
// The products' accumulation rounds towards zero, about 2^-22 of O for a tile of hi and lo. For fp32 queries O therefore
// starts afresh every kFreshTiles tiles of a group, and what it was is added, with rounding to nearest, to a sum in global
// memory (it stays in L2): a prompt of 512 tokens over 32768 rows was off by 1.5e-5 of its result, and is by 1.4e-6 (the
// plain fp32 form by 3e-6; with 4 tiles 2e-6, and 7% less time). 16-bit results keep 11 bits or fewer and need none of this.
constexpr uint32_t kFreshTiles = 2;
constexpr uint32_t kSwitchUnits = 8;            // what changing segments costs, in units
constexpr uint32_t kTileCtas = 148;
constexpr uint32_t kTileSlots = 2 * kTileCtas;  // partial results
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
  // Two query tiles' results: each softmax group stages kStep channels of its O at a time where its own Q tile was.
  static constexpr uint32_t kStep = D / 2;
  static constexpr uint32_t kStaged = kTileM * kStep * 4;
  static_assert(kStaged <= kOperand, "past a group's Q tile lies the other's, or K of the next piece");
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
// One lane of a converged warp. Unlike a test of the lane number it tells the
// compiler that what follows runs in one thread, so that descriptors are computed
// in uniform registers, where the products want them.
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
  return x != 0;
}
// add: whether the product is added to what is there (a constant, or a predicate of the loop).
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
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
template <uint32_t N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <uint32_t N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand descriptor: 128-byte swizzle; panel: bytes between panels
// (MN-major only), 8-row groups are 1024 bytes apart. The low word holds the
// address, so a step along the operand is one 32-bit addition to it.
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand_low(uint32_t addr, uint32_t panel) { return addr >> 4 | (panel >> 4) << 16; }
__device__ __forceinline__ uint64_t operand(uint32_t low, uint32_t bytes_on) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low + (bytes_on >> 4)), "n"(kOperandHigh));
  return d;
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
  uint32_t at;                        // place of its first unit, or its number among the pieces
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
struct TileDeal {
  uint32_t blocks, ctas;
  uint32_t each, more, begin, end;   // dealt out: units of a CTA, the first `more` with one more; this CTA's
  uint32_t size, pieces;             // cut: units of a piece (0: dealt out), pieces
};
// One warp plans for the CTA, all lanes together; the others take the result.
template <uint32_t kRows>
struct TilePlan : TileDeal {
  const Kv4AttnParams &p;

  __device__ uint32_t pieces_of(uint32_t i, uint32_t of) const {
    return i < blocks ? (tile_units<kRows>(p, i / p.row_tiles, i % p.row_tiles) + of - 1) / of : 0u;
  }
  __device__ uint32_t sum_of(uint32_t of) const {
    uint32_t n = 0;
#pragma unroll 1
    for (uint32_t i = threadIdx.x % 32; i < blocks; i += 32) n += pieces_of(i, of);
    return __reduce_add_sync(~0u, n) * p.c.kv_heads;
  }
  __device__ TilePlan(const Kv4AttnParams &p, const TileDeal &d) : TileDeal(d), p(p) {}
  __device__ explicit TilePlan(const Kv4AttnParams &p) : p(p) {
    blocks = p.c.seqs * p.row_tiles;
    size = pieces = 0;
    const uint32_t total = sum_of(1), fair = (total + kTileCtas - 1) / kTileCtas;
    // cut where one or two pieces a CTA share the work about as well as dealing it out does
    const uint32_t segments = blocks * p.c.kv_heads, rounds = segments * 4 <= kTileCtas * 3 ? 1 : 2;
    if (segments * 4 <= kTileCtas * 6) {
      const uint32_t target = kTileCtas * rounds;
      uint32_t of = max(1u, (total + target - 1) / target);
#pragma unroll 1
      for (int i = 0;; ++i) {
        pieces = sum_of(of);
        if (pieces <= target || i == 3) break;
        of = max(of + 1, (uint32_t)((uint64_t)of * pieces / target));
      }
      if (of * rounds <= fair + kSwitchUnits && pieces <= kTileSlots) size = of;
    }
    ctas = min(gridDim.x, size ? pieces : total);
    each = total / ctas;
    more = total - each * ctas;
    begin = each * blockIdx.x + min(blockIdx.x, more);
    end = begin + each + (blockIdx.x < more);
  }
  __device__ uint32_t owner(uint32_t x) const {
    return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each;
  }
  // The segment, and what of it, in which number x of the units (of = 1) or of the pieces lies.
  __device__ TileWork find(uint32_t x, uint32_t of) const {
    const uint32_t lane = threadIdx.x % 32;
    uint32_t before = 0;
#pragma unroll 1
    for (uint32_t base = 0; base < blocks; base += 32) {
      const uint32_t n = pieces_of(base + lane, of);
      uint32_t sum = n * p.c.kv_heads;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(~0u, sum, o);
        if (lane >= (uint32_t)o) sum += up;
      }
      const uint32_t past = __ballot_sync(~0u, before + sum > x);
      if (past) {
        const int at = __ffs(past) - 1;
        const uint32_t parts = __shfl_sync(~0u, n, at);
        const uint32_t into = x - before - (__shfl_sync(~0u, sum, at) - parts * p.c.kv_heads);
        TileWork w;
        w.seq = (base + at) / p.row_tiles;
        w.block = (base + at) % p.row_tiles;
        w.kv = into / parts;
        w.first = (into - w.kv * parts) * of;
        w.seg_units = tile_units<kRows>(p, w.seq, w.block);
        w.units = min(of, w.seg_units - w.first);
        w.at = x;
        return w;
      }
      before += __shfl_sync(~0u, sum, 31);
    }
    return TileWork{0, 0, 0, 0, 0, 1, x};
  }
  __device__ TileWork start() const {
    if (size) return find(blockIdx.x, size);
    TileWork w = find(begin, 1);
    w.units = min(end - begin, w.seg_units - w.first);
    return w;
  }
  // The CTA's next piece; false after the last.
  __device__ bool advance(TileWork &w) const {
    if (size) {
      if (w.at + ctas >= pieces) return false;
      w = find(w.at + ctas, size);
      return true;
    }
    w.at += w.units;
    if (w.at >= end) return false;
    w.first = 0;
    if (++w.kv == p.c.kv_heads) {
      w.kv = 0;
      if (++w.block == p.row_tiles) w.block = 0, ++w.seq;
      w.seg_units = tile_units<kRows>(p, w.seq, w.block);
    }
    w.units = min(end - w.at, w.seg_units);
    return true;
  }
  // Partial results of the segment: where this piece's goes, and those of its parts.
  struct Parts {
    uint32_t own, first, second, step, count, ticket;
    __device__ uint32_t slot(uint32_t i) const { return i == 0 ? first : second + (i - 1) * step; }
  };
  __device__ Parts parts(const TileWork &w) const {
    Parts x;
    if (size) {
      const uint32_t part = w.first / size;
      x.own = w.at;
      x.first = w.at - part;
      x.second = x.first + 1;
      x.step = 1;
      x.count = (w.seg_units + size - 1) / size;
      x.ticket = (w.seq * p.row_tiles + w.block) * p.c.kv_heads + w.kv;
    } else {   // a CTA has at most two: of a segment begun before it, and of one that goes on after it
      const uint32_t c0 = owner(w.at - w.first);
      x.own = blockIdx.x * 2 + (w.first == 0);
      x.first = c0 * 2 + 1;
      x.second = (c0 + 1) * 2;
      x.step = 2;
      x.count = owner(w.at - w.first + w.seg_units - 1) - c0 + 1;
      x.ticket = c0;
    }
    return x;
  }
};

struct TileBars {
  uint64_t q_full, s_full[2], p_half[2], p_full[2], o_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], raw_full[kRawStages], drained;
};

// A row of shared memory in 16-byte chunks, turned by the row: a warp that writes
// one chunk of each of 32 rows, and one that reads a whole row, meet no conflicts.
template <uint32_t kChunks>
__device__ __forceinline__ float4 *row_chunk(float *base, uint32_t row, uint32_t chunk) {
  return (float4 *)base + row * kChunks + (chunk ^ (row % kChunks));
}
// Eight columns of O, which hold channels 0 4 1 5 2 6 3 7.
__device__ __forceinline__ void in_order(const float *o, float4 &low, float4 &high) {
  low = make_float4(o[0], o[2], o[4], o[6]);
  high = make_float4(o[1], o[3], o[5], o[7]);
}

// What the softmax groups do when a piece ends: join the groups' results where
// they shared a query tile, then finish the rows, or leave a partial result and,
// last of the segment's CTAs, add them all. O goes through Q's place in shared
// memory, so that rows leave in whole lines. 256 threads.
template <int D, typename T, typename Plan>
__device__ __forceinline__ void tile_results(const Kv4AttnParams &p, const Plan &plan, const TileWork &w, bool pair, uint32_t x,
                                             uint32_t row, uint32_t row0, float m, float l, bool mine, uint32_t o_addr,
                                             const float *kept, float kept_scale,
                                             float *shared_o, float (*group_max)[kTileM], float (*group_sum)[kTileM], float *factors, uint32_t *last) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, rows = p.tokens * p.group;
  const uint32_t block_rows = min(pair ? 2 * kTileM : kTileM, rows - row0);
  const bool whole = w.units == w.seg_units;
  const typename Plan::Parts parts = plan.parts(w);
  auto place = [&](uint32_t i) {
    const uint32_t tok = (row0 + i) / p.group, head = w.kv * p.group + (row0 + i) - tok * p.group;
    return ((size_t)w.seq * p.tokens + tok) * p.heads + head;
  };
  // a row whose softmax sums up to 0: zeros where it sees no cache row, NaN where every score was -infinity
  auto blank = [&](uint32_t i) {
    const int32_t tok = (int32_t)((row0 + i) / p.group), count = kv4_count(p, w.seq);
    return i < block_rows && tok < count && (int32_t)kv4_held(p.c, w.seq) - count + tok + 1 > 0 ? NAN : 0.f;
  };
  auto lse = [&](uint32_t i, float top, float sum) { return sum == 0.f ? INFINITY + blank(i) : top + log2f(sum) - kTilePScale; };
  auto slot = [&](uint32_t i) { return p.parts + (size_t)i * kTilePart<D>; };
  float *part = slot(parts.own);
  // 4 channels of row r, final or partial
  auto leave = [&](uint32_t r, uint32_t ch, float4 v) {
    if (whole) {
      T y[4] = {from_float<T>(v.x), from_float<T>(v.y), from_float<T>(v.z), from_float<T>(v.w)};
      T *dst = (T *)p.out + place(r) * D + ch;
      if constexpr (sizeof(T) == 4) *(float4 *)dst = *(const float4 *)y;
      else *(uint2 *)dst = *(const uint2 *)y;
    } else {
      *(float4 *)(part + r * D + ch) = v;
    }
  };
  auto leave_sums = [&](uint32_t r) {
    if (!whole) {
      part[2 * kTileM * D + r] = m;
      part[2 * kTileM * (D + 1) + r] = l;
    } else if (p.lse) {
      p.lse[place(r)] = lse(r, m, l);
    }
  };
  if (!pair) {
    constexpr uint32_t kChunks = D / 4;
    group_max[x][row] = mine ? m : kNoScore;
    group_sum[x][row] = mine ? l : 0.f;
    named_bar(2, 256);
    const float m0 = group_max[0][row], m1 = group_max[1][row], top = fmaxf(m0, m1);
    const float w0 = exp2_fast(m0 - top), w1 = exp2_fast(m1 - top);
    l = group_sum[0][row] * w0 + group_sum[1][row] * w1;
    m = top;
    const float f = (x ? w1 : w0) * (!whole ? 1.f : l == 0.f ? blank(row) : 1.f / l);
    // each group hands over its share of the other's half of the channels, then adds what it was handed to its own half
#pragma unroll 1
    for (uint32_t pass = 0; pass < 2; ++pass) {
      const uint32_t from = (x ^ pass ^ 1) * (D / 2);
      const bool add = pass && (x == 1 || w.units > 1);   // the other group had a tile
#pragma unroll 1
      for (uint32_t c = from; c < from + D / 2; c += 32) {
        float o[32];
        tmem_load32(o_addr + c, o);
        tmem_wait_load();
        loaded(o);
        if (sizeof(T) == 4 && kept) {
#pragma unroll
          for (uint32_t i = 0; i < 32; ++i) o[i] = fmaf(kept[(c + i) * kTileM + row], kept_scale, o[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < 32; i += 8) {
          float4 v[2];
          in_order(o + i, v[0], v[1]);
#pragma unroll
          for (uint32_t k = 0; k < 2; ++k) {
            float4 *at = row_chunk<kChunks>(shared_o, row, (c + i) / 4 + k);
            float4 y = add ? *at : make_float4(0.f, 0.f, 0.f, 0.f);
            if (mine) y.x = fmaf(v[k].x, f, y.x), y.y = fmaf(v[k].y, f, y.y), y.z = fmaf(v[k].z, f, y.z), y.w = fmaf(v[k].w, f, y.w);
            *at = y;
          }
        }
      }
      __syncwarp();
      named_bar(2, 256);
    }
    constexpr uint32_t kPer = 32 / kChunks;   // rows of a warp's pass
#pragma unroll 4
    for (uint32_t r = warp * kPer + lane / kChunks; r < block_rows; r += 8 * kPer)
      leave(r, lane % kChunks * 4, *row_chunk<kChunks>(shared_o, r, lane % kChunks));
    if (x == 0 && row < block_rows) leave_sums(row);
  } else {
    // each group where its own Q tile was, half of the channels at a time
    constexpr uint32_t kStep = TileSmem<D>::kStep, kChunks = kStep / 4;
    constexpr uint32_t kPer = 32 / kChunks;   // rows of a warp's pass
    float *own = shared_o + x * (TileSmem<D>::kOperand / 4);
    const float inv = !whole ? 1.f : l == 0.f ? blank(x * kTileM + row) : 1.f / l;
    const uint32_t n = x * kTileM < block_rows ? min(kTileM, block_rows - x * kTileM) : 0;   // rows of this group
#pragma unroll 1
    for (uint32_t c0 = 0; c0 < D; c0 += kStep) {
#pragma unroll 1
      for (uint32_t c = 0; c < kStep; c += 32) {
        float o[32];
        tmem_load32(o_addr + c0 + c, o);
        tmem_wait_load();
        loaded(o);
#pragma unroll
        for (uint32_t i = 0; i < 32; i += 8) {
          float4 v[2];
          in_order(o + i, v[0], v[1]);
#pragma unroll
          for (uint32_t k = 0; k < 2; ++k)
            *row_chunk<kChunks>(own, row, (c + i) / 4 + k) = make_float4(v[k].x * inv, v[k].y * inv, v[k].z * inv, v[k].w * inv);
        }
      }
      named_bar(3 + x, kTileM);
#pragma unroll 4
      for (uint32_t r = warp % 4 * kPer + lane / kChunks; r < n; r += 4 * kPer)
        leave(x * kTileM + r, c0 + lane % kChunks * 4, *row_chunk<kChunks>(own, r, lane % kChunks));
      named_bar(3 + x, kTileM);
    }
    if (row < n) leave_sums(x * kTileM + row);
  }
  if (!whole) {
    const uint32_t pieces = parts.count;
    __syncwarp();
    named_bar(2, 256);
    if (threadIdx.x == 0) {
      *last = atomic_add_acq_rel(p.tickets + parts.ticket, 1u) == pieces - 1;
      if (*last) p.tickets[parts.ticket] = 0;
    }
    __syncwarp();
    named_bar(2, 256);
    if (*last) {
      constexpr uint32_t N = D / 32;   // channels of a lane
      using V = typename std::conditional<N == 4, float4, float2>::type;
      auto piece = [&](uint32_t i) { return (const float *)slot(parts.slot(i)); };
      // a thread a row: the weight of each piece, in Q's place, as many rows at a time as it holds
      const uint32_t some = min(block_rows, 2 * kTileM * D / 2 / pieces);
#pragma unroll 1
      for (uint32_t r0 = 0; r0 < block_rows; r0 += some) {
        const uint32_t n = min(some, block_rows - r0);
        if (threadIdx.x < n) {
          const uint32_t i = r0 + threadIdx.x;
          float top = kNoScore, sum = 0.f;
#pragma unroll 8
          for (uint32_t k = 0; k < pieces; ++k) {
            const float pm = __ldcg(piece(k) + 2 * kTileM * D + i);
            shared_o[k * n + threadIdx.x] = pm;
            top = fmaxf(top, pm);
          }
#pragma unroll 8
          for (uint32_t k = 0; k < pieces; ++k) {
            const float ps = __ldcg(piece(k) + 2 * kTileM * (D + 1) + i);
            const float pw = exp2_fast(shared_o[k * n + threadIdx.x] - top);
            shared_o[k * n + threadIdx.x] = pw;
            sum = fmaf(pw, ps, sum);
          }
          factors[threadIdx.x] = sum == 0.f ? blank(i) : 1.f / sum;
          if (p.lse) p.lse[place(i)] = lse(i, top, sum);
        }
        __syncwarp();
        named_bar(2, 256);
        constexpr uint32_t kBatch = 2;   // rows of a warp in flight
#pragma unroll 1
        for (uint32_t i0 = warp; i0 < n; i0 += 8 * kBatch) {
          float y[kBatch][N] = {};
#pragma unroll 4
          for (uint32_t k = 0; k < pieces; ++k) {
#pragma unroll
            for (uint32_t b = 0; b < kBatch; ++b) {
              const uint32_t i = min(i0 + 8 * b, n - 1);
              const V z = __ldcg((const V *)(piece(k) + (r0 + i) * D + lane * N));
              const float f = shared_o[k * n + i];
#pragma unroll
              for (uint32_t j = 0; j < N; ++j) y[b][j] = fmaf(f, ((const float *)&z)[j], y[b][j]);
            }
          }
#pragma unroll
          for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t i = i0 + 8 * b;
            if (i >= n) break;
            T *dst = (T *)p.out + place(r0 + i) * D + lane * N;
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) dst[j] = from_float<T>(y[b][j] * factors[i]);
          }
        }
        __syncwarp();
        named_bar(2, 256);
      }
    }
  }
  __syncwarp();
  named_bar(2, 256);   // Q's place and the shared words may change
}

// PAIR: blocks of 256 query rows, which 16-bit queries have room for.
template <int D, typename T, bool PAIR>
__global__ void __launch_bounds__(kTileThreads, 1) kv4_tile_kernel(const Kv4AttnParams p) {
  using S = TileSmem<D>;
  constexpr bool kSplit = sizeof(T) == 4;
  static_assert(!(kSplit && PAIR), "hi and lo take the second query tile's place");
  constexpr uint32_t kRows = PAIR ? 2 * kTileM : kTileM;      // query rows of a block
  constexpr uint32_t kPanel = kTileN * 128;                   // bytes of 64 channels of a tile
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t *smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ TileBars bars;
  __shared__ uint32_t tmem_base, aborted, last;
  __shared__ float factors[2 * kTileM], group_max[2][kTileM], group_sum[2][kTileM];
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const uint32_t rows = p.tokens * p.group;
  if (p.lse) pdl_launch_dependents();   // the weights kernel may take the SMs that this one leaves
  __shared__ TileDeal shared_deal;
  __shared__ TileWork shared_work;
  if (warp == 0) {
    const TilePlan<kRows> x(p);
    if (lane == 0) shared_deal = x;
    if (blockIdx.x < x.ctas) {
      const TileWork y = x.start();
      if (lane == 0) shared_work = y;
    }
  }
  if (threadIdx.x == 32) {
    mbar_init(&bars.q_full, 256);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_half[i], kTileM);
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
  if (warp == 12) tmem_alloc512(&tmem_base);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t *)&tmem_base;
  const TilePlan<kRows> plan(p, shared_deal);
  if (blockIdx.x >= plan.ctas) {   // nothing for this CTA
    if (warp == 12) tmem_free512(tmem);
    return;
  }
  // a wait that runs out makes every later one return at once: the roles then run to their ends on whatever is there
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity) || *(volatile uint32_t *)&aborted) return;
    if (!mbar_wait_bounded(bar, parity)) *(volatile uint32_t *)&aborted = 1;
  };
  // two query tiles, or one whose cache tiles the softmax groups share
  auto paired = [&](const TileWork &w) { return PAIR && rows - w.block * kRows > kTileM; };
  // f(work) for every piece of this CTA; whole warps
  const TileWork first_work = shared_work;
  auto each_work = [&](auto &&f) {
    TileWork w = first_work;
    do f(w);
    while (plan.advance(w));
  };

  if (warp >= 12) {
    fewer_registers<kOtherRegs>();
    // ---------------- products ----------------
    if (warp == 12) {
      const uint32_t q = operand_low(smem_u32(smem + S::kQ), 0), k = operand_low(smem_u32(smem + S::kK), 0);
      const uint32_t v = operand_low(smem_u32(smem + S::kV), kPanel);
      constexpr uint32_t kScoreDesc = tile_idesc(kTileN, false), kValueDesc = tile_idesc(D, true);
      constexpr uint32_t kTileOn = S::kOperand >> 4;   // from one operand to the next, in a descriptor
      uint32_t works = 0, tiles = 0, jobs0 = 0, jobs1 = 0;   // jobs: of each group
      each_work([&](const TileWork &w) {
        if (elect_one()) {
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
              const uint32_t d = tmem + x * 128, qa = q + (pair ? x * kTileOn : 0), ka = k + st * kTileOn;
#pragma unroll
              for (uint32_t c = 0; c < D / 16; ++c) {
                const uint32_t off = c / 4 * kPanel + c % 4 * 32;
                mma_ss(d, operand(qa, off), operand(ka, off), kScoreDesc, c > 0);
                if constexpr (kSplit) mma_ss(d, operand(qa, S::kOperand + off), operand(ka, off), kScoreDesc, true);
              }
              tc_commit(&bars.s_full[x]);
              if (!pair || x == 1) tc_commit(&bars.k_empty[st]);
            }
            if (j > 0) {   // values of job j - 1
              const uint32_t i = j - 1, x = i & 1, tile = tiles + (pair ? i >> 1 : i), st = tile & 1;
              const uint32_t parity = (x ? jobs1 : jobs0) & 1;
              const uint32_t d = tmem + 256 + x * 128, pa = tmem + x * 128, va = v + st * kTileOn;
              if (!pair || x == 0) wait(&bars.v_full[st], tile >> 1 & 1);
#pragma unroll
              for (uint32_t half = 0; half < 2; ++half) {
                wait(half ? &bars.p_full[x] : &bars.p_half[x], parity);
                tc_fence_after();
#pragma unroll
                for (uint32_t c = half * 4; c < half * 4 + 4; ++c) {
                  const uint64_t b = operand(va, c * 2048);
                  mma_ts(d, pa + c * 8, b, kValueDesc, c > 0 || (kSplit ? i / 2 % kFreshTiles != 0 : i > 1));
                  if constexpr (kSplit) mma_ts(d, pa + 64 + c * 8, b, kValueDesc, true);
                }
              }
              if (!pair || x == 1) tc_commit(&bars.v_empty[st]);
              if (i + 2 >= n) tc_commit(&bars.o_full[x]);
              if (x) ++jobs1;
              else ++jobs0;
            }
          }
          tiles += w.units;
        }
        __syncwarp();
      });
      if (elect_one()) {
        tc_commit(&bars.drained);   // tensor memory is freed after the last product, even when waits ran out
        mbar_wait_bounded(&bars.drained, 0);
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    fewer_registers<kOtherRegs>();
    // ---------------- unpacking ----------------
    const uint32_t tid = threadIdx.x - 256;
    const size_t run_bytes = (size_t)p.c.tiles * Kv4<D>::kTileBytes;
    // the first warp streams the cache's 64-row tiles; a stage is refilled once all have unpacked it
    TileWork ahead = first_work;
    uint32_t ahead_raw = 0;   // 64-row tile of the piece
    CopyRing<kRawStages> copies;   // `passed` and `stopped` are the loop's own: `used` below, and `aborted`
    bool ahead_on = true;
    auto fetch = [&]() {
      if (!ahead_on) return;
      const uint32_t raw = ahead.first * 2 + ahead_raw;
      if (raw < p.c.tiles && !*(volatile uint32_t *)&aborted) {
        copies.fetch([&](uint32_t st) {
          if (lane == 0) {
            mbar_arrive_expect_tx(&bars.raw_full[st], S::kRawStage);
            bulk_g2s(smem + S::kRaw + st * S::kRawStage,
                     p.c.data + ((size_t)ahead.seq * p.c.kv_heads + ahead.kv) * run_bytes + (size_t)raw * S::kRawStage,
                     S::kRawStage, &bars.raw_full[st]);
          }
        });
      }
      if (++ahead_raw == 2 * ahead.units) {
        ahead_raw = 0;
        ahead_on = plan.advance(ahead);
      }
    };
    if (warp == 8)
      for (uint32_t i = 0; i < kRawStages; ++i) fetch();
    // a thread unpacks 32 channels of a row, of kPasses rows of K and as many of V
    constexpr uint32_t kQuads = D / 32, kPassRows = kUnpackThreads / kQuads, kPasses = kKv4Tile / kPassRows;
    const uint32_t quad = tid % kQuads, r0 = tid / kQuads;
    // threads of the second panel write their chunks two on, which keeps a row pair's 8 threads off each other
    const bool turn = quad & 2;
    uint32_t off[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      off[k] = quad / 2 * kPanel + r0 * 128 + ((quad % 2 * 4 | ((turn ? 2 : 0) + k & 3)) ^ (r0 & 7)) * 16;
    uint32_t tiles = 0, used = 0;
    each_work([&](const TileWork &w) {
      const uint32_t held = kv4_held(p.c, w.seq);
#pragma unroll 1
      for (uint32_t u = 0; u < w.units; ++u, ++tiles) {
        const uint32_t st = tiles & 1;
        if (tiles >= 2) {
          wait(&bars.k_empty[st], (tiles >> 1) - 1 & 1);
          wait(&bars.v_empty[st], (tiles >> 1) - 1 & 1);
        }
        // one 64-row tile at a time, K and V, so that its stage is free for the third one after it
#pragma unroll 1
        for (uint32_t h = 0; h < 2; ++h) {
          const uint32_t raw = (w.first + u) * 2 + h;
          const bool have = raw < p.c.tiles;    // a run's last unit may have no second half: it is zeros
          const uint8_t *src = smem + S::kRaw + used % kRawStages * S::kRawStage;
          if (have) wait(&bars.raw_full[used % kRawStages], used / kRawStages & 1);
          uint8_t *dst = smem + S::kK + st * S::kOperand + h * (kKv4Tile * 128);
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            uint4 x[kPasses];
            __half d[kPasses];
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) {
              const uint32_t r = r0 + i * kPassRows;
              x[i] = *(const uint4 *)(src + Kv4<D>::codes(r, v) + quad * 16);
              d[i] = *(const __half *)(src + Kv4<D>::scales(r, v) + quad * 2);
              if (raw * kKv4Tile + r >= held) d[i] = __half(0.f);   // bytes past the rows held may be anything
            }
#pragma unroll
            for (uint32_t i = 0; i < kPasses; ++i) {
              const uint4 y = x[i];
              const uint32_t word[4] = {turn ? y.z : y.x, turn ? y.w : y.y, turn ? y.x : y.z, turn ? y.y : y.w};
              const __half2 d2 = __half2half2(d[i]), d72 = minus72(d2);
              uint8_t *out = dst + v * (S::kV - S::kK) + i * (kPassRows * 128);
#pragma unroll
              for (uint32_t k = 0; k < 4; ++k) {
                __align__(16) __half2 z[4];
                unpack8(word[k], d2, d72, z);
                *(uint4 *)(out + off[k]) = *(const uint4 *)z;
              }
            }
          }
          used += have;
          if (h == 1) {
            fence_async_smem();
            mbar_arrive(&bars.k_full[st]);
            mbar_arrive(&bars.v_full[st]);
          }
          __syncwarp();
          named_bar(1, kUnpackThreads);   // all have read the stage
          if (warp == 8) fetch();
        }
      }
    });
    // nothing is left in flight but after a wait that ran out, which passes over copies that have not landed
    if (tid == 0 && *(volatile uint32_t *)&aborted)
      copies.drain([&](uint32_t at, uint32_t parity) { mbar_wait_bounded(&bars.raw_full[at], parity); });
  } else {
    more_registers<kSoftmaxRegs>();
    // ---------------- softmax ----------------
    const uint32_t x = warp / 4, row = threadIdx.x % kTileM;       // group, and its row of the tile
    const uint32_t lanes = (warp % 4) << 21;                       // this warp's lanes of tensor memory
    const uint32_t s_addr = tmem + x * 128 + lanes, o_addr = tmem + 256 + x * 128 + lanes;
    uint32_t done = 0, works = 0;   // tiles of this group, pieces in which it had some
    each_work([&](const TileWork &w) {
      const bool pair = paired(w);
      const uint32_t row0 = w.block * kRows, held = kv4_held(p.c, w.seq);
      const int32_t count = kv4_count(p, w.seq);
      // ---- Q to shared memory, a warp a row: two tiles, or one (as hi and lo) that both groups load half of ----
      const uint32_t q_rows = pair ? 2 * kTileM : kTileM;
      constexpr uint32_t L = D / 8, kPer = 32 / L, kBatch = kTileM / (8 * kPer);   // lanes of a row, rows of a pass, passes in flight
      const uint32_t sub = lane % L, lane_row = lane / L;
#pragma unroll 1
      for (uint32_t r0 = warp * kPer; r0 < q_rows; r0 += 8 * kPer * kBatch) {
        float y[kBatch][8];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
          const uint32_t r = row0 + r0 + b * 8 * kPer + lane_row;
          const uint32_t tok = r / p.group, head = w.kv * p.group + r - tok * p.group;
          const T *src = (const T *)p.q + (int64_t)w.seq * p.qs.seq + (int64_t)tok * p.qs.token + (int64_t)head * p.qs.head + sub * 8;
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i) y[b][i] = 0.f;
          if (r < rows) {
            if (p.wide) load8<T, true>(src, y[b]);
            else load8<T, false>(src, y[b]);
          }
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
          const uint32_t r = r0 + b * 8 * kPer + lane_row;
          uint32_t top = 0;
#pragma unroll
          for (uint32_t i = 0; i < 8; ++i) top = max(top, __float_as_uint(y[b][i]) & 0x7FFFFFFFu);
#pragma unroll
          for (uint32_t o = 1; o < L; o <<= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
          float inverse;
          const float power = row_power(__uint_as_float(top), inverse);
          if (sub == 0) factors[r] = fmaxf(p.scale * inverse, 0x1p-126f);
          uint8_t *dst = smem + S::kQ + r / kTileM * S::kOperand + sub / 8 * kPanel + r % kTileM * 128 + ((sub % 8) ^ (r & 7)) * 16;
          __align__(16) uint32_t hi[4], lo[4];   // channels 0 4 1 5 2 6 3 7
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
            if constexpr (kSplit) split2(y[b][i] * power, y[b][i + 4] * power, hi[i], lo[i]);
            else hi[i] = half2_bits(__floats2half2_rn(y[b][i] * power, y[b][i + 4] * power));
          }
          *(uint4 *)dst = *(const uint4 *)hi;
          if constexpr (kSplit) *(uint4 *)(dst + S::kOperand) = *(const uint4 *)lo;
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
      float m = kNoScore, l = 0.f;   // m: of the products' sums, not yet scaled
      // fp32: the sum of earlier O, [channel][row] in the half of a partial result that 128-row blocks do not use, and the
      // maximum that it is relative to
      float *const kept = p.parts + (size_t)(blockIdx.x * 2 + x) * kTilePart<D> + kTileM * D;
      float kept_max = 0.f;
      bool keeping = false;
      const uint32_t step = pair ? 1 : 2;
#pragma unroll 1
      for (uint32_t u = pair ? 0 : x; u < w.units; u += step, ++done) {
        wait(&bars.s_full[x], done & 1);
        __syncwarp();
        tc_fence_after();
        const bool fresh = kSplit ? u / 2 % kFreshTiles == 0 : u < step;   // nothing in O counts
        if (kSplit && fresh && u >= step) {   // O is whole: the products before these scores are done
          const float r = exp2_fast((kept_max - m) * f);
#pragma unroll 1
          for (uint32_t c = 0; c < D; c += 32) {
            float o[32];
            tmem_load32(o_addr + c, o);
            tmem_wait_load();
            loaded(o);
            float *at = kept + c * kTileM + row;
            if (keeping) {
              float before[32];   // all loads before the first store: one latency, not 32
#pragma unroll
              for (uint32_t i = 0; i < 32; ++i) before[i] = at[i * kTileM];
#pragma unroll
              for (uint32_t i = 0; i < 32; ++i) o[i] = fmaf(before[i], r, o[i]);
            }
#pragma unroll
            for (uint32_t i = 0; i < 32; ++i) at[i * kTileM] = o[i];
          }
          kept_max = m;
          keeping = true;
        }
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
        for (int c = 4; c + 8 <= (int)kTileN; c += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) top[i] = max3(top[i], s[c + i], s[c + 4 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], s[kTileN - 4 + i]);
        const float best = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        if (__any_sync(~0u, (best - m) * f > kLead)) {
          const float up = fmaxf(m, best), r = exp2_fast((m - up) * f);
          m = up;
          l *= r;
          if (!fresh) {   // O has something: the products before these scores are done
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
        const float2 f2 = make_float2(f, f), base2 = make_float2(kTilePScale, kTilePScale), less = make_float2(-m, -m);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < (int)kTileN; c += 32) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float2 e = fma2(add2(make_float2(s[c + 2 * i], s[c + 2 * i + 1]), less), f2, base2);
            e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
            sum[i % 2] = add2(sum[i % 2], e);
            if constexpr (kSplit) split2(e.x, e.y, hi[i], lo[i]);
            else hi[i] = half2_bits(__floats2half2_rn(e.x, e.y));
          }
          tmem_store16(s_addr + c / 2, hi);
          if constexpr (kSplit) tmem_store16(s_addr + 64 + c / 2, lo);
          if (c == 32) {   // the products of the first 64 rows may start
            tmem_wait_store();
            tc_fence_before();
            mbar_arrive(&bars.p_half[x]);
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_wait_store();
        tc_fence_before();
        mbar_arrive(&bars.p_full[x]);
      }
      // ---- results ----
      const bool mine = pair || w.units > x;    // this group had a tile
      if (mine) wait(&bars.o_full[x], works++ & 1);
      __syncwarp();
      tc_fence_after();
      tile_results<D, T>(p, plan, w, pair, x, row, row0, l == 0.f ? kNoScore : m * f, l, mine, o_addr, keeping ? kept : nullptr,
                         exp2_fast((kept_max - m) * f), (float *)(smem + S::kQ), group_max, group_sum, factors, &last);
      tc_fence_before();
    });
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_free512(tmem);
  if (threadIdx.x == 0 && aborted) atomicOr(&p.c.state[0].status, kKv4Timeout);
}

}  // namespace vg
