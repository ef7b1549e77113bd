// A step of a paged cache's table: rows dropped, pages given back and handed out,
// and the slot map of the step's new tokens.
//
// For sequence s with rows r, keep k and count c: kept = min(k, r) rows stay (all
// of them for k < 0), its pages past ceil(kept / P) go onto the free stack, and it
// then needs ceil((kept + c) / P) - ceil(kept / P) pages. Frees are pushed in the
// order of sequences and table entries. The A pages of the sequences that fit are
// the topmost A of the stack, in stack order, so a step that takes back what the
// one before handed out gives every sequence the same pages again. A sequence fits
// when its demand and that of all before it do; one that needs none always fits.
//
// Everything is a prefix sum over the sequences (tokens, frees, demand, runs) and
// then one item a thread: a freed entry, a page handed out, four tokens, a run. An
// item finds its sequence by bisection of the prefix sums in shared memory. Every
// CTA forms the sums for itself; the frees are on the stack before a page is taken
// from it, which is the one place where CTAs wait for each other: a cluster barrier.
// Measured: 16 sequences 7.4 us, 1024 with 131,072 new tokens 19.6 us in 8 CTAs. A
// thread looks its first token's sequence up and walks on to those of the next three, so
// idle sequences cost a dependent read each: 16 busy ones of 4096 46 us, the first and the
// last alone 174.
#pragma once
#include "paged.cuh"

namespace vg {

constexpr uint32_t kStepThreads = 1024;
constexpr uint32_t kStepCtas = 8;       // of a large step
constexpr uint32_t kStepSeqs = 4096;    // their sums are held in shared memory

struct StepParams {
  PagedTable t;
  const int32_t *counts, *keep;
  int32_t *starts, *slots, *positions, *sequences;
  int4 *runs;      // first token, page, first row in the page, rows
  uint32_t tokens, most_runs;
};

// Sums of two numbers over the threads before this one, and over all. `part` is
// shared memory of 32 pairs that no other call uses.
struct Sums {
  uint64_t a, b;
};
__device__ __forceinline__ Sums sums_before(Sums x, Sums *part, Sums &all) {
  const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  Sums up = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t a = __shfl_up_sync(~0u, up.a, o), b = __shfl_up_sync(~0u, up.b, o);
    if (lane >= (uint32_t)o) up.a += a, up.b += b;
  }
  if (lane == 31) part[warp] = up;
  __syncthreads();
  Sums w = lane < warps ? part[lane] : Sums{0, 0};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t a = __shfl_up_sync(~0u, w.a, o), b = __shfl_up_sync(~0u, w.b, o);
    if (lane >= (uint32_t)o) w.a += a, w.b += b;
  }
  all = Sums{__shfl_sync(~0u, w.a, 31), __shfl_sync(~0u, w.b, 31)};
  const int before = (int)warp - 1;
  const uint64_t wa = __shfl_sync(~0u, w.a, max(before, 0)), wb = __shfl_sync(~0u, w.b, max(before, 0));
  return Sums{up.a - x.a + (warp ? wa : 0), up.b - x.b + (warp ? wb : 0)};
}

// The last sequence whose sum is at most i (before[0] is 0).
__device__ __forceinline__ uint32_t find_seq(const uint32_t *before, uint32_t n, uint32_t i) {
  uint32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (before[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct StepSeq {   // of each sequence, in shared memory: arrays of words, one after the other
  uint32_t *start, *kept, *fresh, *freed, *taken, *runs;
  __device__ __forceinline__ StepSeq(uint32_t *base, uint32_t n)
      : start(base), kept(base + n), fresh(base + 2 * n), freed(base + 3 * n), taken(base + 4 * n), runs(base + 5 * n) {}
};
constexpr uint32_t kStepWords = 6;

__global__ void __launch_bounds__(kStepThreads) paged_step_kernel(const StepParams p) {
  extern __shared__ __align__(16) uint32_t step_words[];
  __shared__ Sums parts[3][32];
  const PagedTable &t = p.t;
  const uint32_t n = t.seqs, tid = threadIdx.x, page = t.page_rows(), wide = t.seq_pages;
  const uint32_t each = (n + blockDim.x - 1) / blockDim.x, s0 = min(n, tid * each), s1 = min(n, s0 + each);
  const StepSeq q(step_words, n);
  const auto pages_of = [&](uint32_t rows) { return (rows + page - 1) >> t.shift; };
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t height = (uint32_t)min(max(__ldcg(&t.pool[0]), 0), (int32_t)t.pages);

  // ---- tokens and freed pages ----
  constexpr uint32_t kBad = 0x80000000u;
  Sums mine{0, 0}, all;
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t rows = (uint32_t)min(max(t.rows[s], 0), (int32_t)t.capacity());
    const int32_t k = p.keep ? p.keep[s] : -1, c = p.counts[s];
    const uint32_t kept = k < 0 ? rows : min((uint32_t)k, rows);
    const bool bad = c < 0 || (uint32_t)c > p.tokens;
    q.kept[s] = kept;
    q.fresh[s] = bad ? kBad : (uint32_t)c;
    q.freed[s] = pages_of(rows) - pages_of(kept);
    mine.a += bad ? 0 : c, mine.b += q.freed[s];
  }
  Sums sum = sums_before(mine, parts[0], all);
  const uint32_t total = (uint32_t)min(all.a, (uint64_t)p.tokens);
  const uint32_t freed = (uint32_t)min(all.b, (uint64_t)(t.pages - height));   // more only where a table is damaged
  const uint32_t high = height + freed;
  // ---- demand ----
  mine = Sums{0, 0};
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t was = q.fresh[s], c = was & ~kBad;
    q.start[s] = (uint32_t)min(sum.a, (uint64_t)p.tokens);
    sum.a += c;
    const uint32_t f = q.freed[s];
    q.freed[s] = (uint32_t)min(sum.b, (uint64_t)UINT32_MAX);
    sum.b += f;
    const bool bad = (was & kBad) || sum.a > p.tokens, full = (uint64_t)q.kept[s] + c > t.capacity();
    const uint32_t need = bad || full ? 0 : pages_of(q.kept[s] + c) - pages_of(q.kept[s]);
    q.fresh[s] = bad ? kBad : full ? kBad | 1 : c;
    q.runs[s] = need;
    mine.a += need;
  }
  sum = sums_before(mine, parts[1], all);
  // ---- who fits ----
  const bool first_cta = cluster_rank() == 0;
  uint64_t before = sum.a;
  mine = Sums{0, 0};
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t need = q.runs[s], was = q.fresh[s];
    const bool refused = was & kBad, shorted = need && before + need > high;
    q.taken[s] = (uint32_t)min(before, (uint64_t)UINT32_MAX);
    before += need;
    const uint32_t c = refused || shorted ? 0 : was, kept = q.kept[s];
    const uint32_t runs = c ? ((kept + c - 1) >> t.shift) - (kept >> t.shift) + 1 : 0;
    // the status is kept where a refused sequence has no new rows: bits 31 and below
    q.fresh[s] = shorted ? kBad | 2 : was;
    q.runs[s] = runs;
    mine.a += shorted ? 0 : need, mine.b += runs;
  }
  sum = sums_before(mine, parts[2], all);
  const uint32_t taken = (uint32_t)all.a, runs = (uint32_t)min(all.b, (uint64_t)p.most_runs), top = high - taken;
  for (uint32_t s = s0; s < s1; ++s) {
    const uint32_t r = q.runs[s];
    q.runs[s] = (uint32_t)sum.b;
    sum.b += r;
  }
  __syncthreads();

  // ---- freed pages onto the stack; their entries name no page ----
  const uint32_t threads = blockDim.x * cluster_size(), me = cluster_rank() * blockDim.x + tid;
  for (uint32_t i = me; i < freed; i += threads) {
    const uint32_t s = find_seq(q.freed, n, i), col = pages_of(q.kept[s]) + i - q.freed[s];
    int32_t *e = t.table + (size_t)s * wide + col;
    t.free[height + i] = *e;
    *e = -1;
  }
  cluster_sync();   // nobody reads what is written from here on, but for the stack
  // ---- pages off its top ----
  for (uint32_t i = me; i < taken; i += threads) {
    const uint32_t s = find_seq(q.taken, n, i), col = pages_of(q.kept[s]) + i - q.taken[s];
    t.table[(size_t)s * wide + col] = __ldcg(&t.free[top + i]);
  }
  if (first_cta) {
    for (uint32_t s = tid; s < n; s += blockDim.x) {
      const uint32_t f = q.fresh[s];
      t.rows[s] = (int32_t)(q.kept[s] + (f & kBad ? 0 : f));
      t.status[s] = !(f & kBad) ? 0 : (f & 3) == 0 ? kPagedBadCount : (f & 3) == 1 ? kPagedFull : kPagedNoPages;
      p.starts[s] = (int32_t)q.start[s];
    }
    if (tid == 0) {
      p.starts[n] = (int32_t)total;
      t.pool[0] = (int32_t)top;
    }
  }
  // the page of entry col of sequence s, kept or handed out just now
  const auto page_at = [&](uint32_t s, uint32_t col) {
    const uint32_t stay = pages_of(q.kept[s]);
    return col < stay ? t.table[(size_t)s * wide + col] : __ldcg(&t.free[top + q.taken[s] + col - stay]);
  };
  // ---- the tokens, four a thread ----
  for (uint32_t i = 4 * me; i < p.tokens; i += 4 * threads) {
    uint32_t s = i < total ? find_seq(q.start, n, i) : n - 1;
    int32_t slot[4], pos[4], seq[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
      slot[j] = pos[j] = seq[j] = -1;
      if (i + j >= total) continue;
      while (s + 1 < n && q.start[s + 1] <= i + j) ++s;
      if (q.fresh[s] & kBad) continue;
      const uint32_t at = q.kept[s] + i + j - q.start[s];
      pos[j] = (int32_t)at;
      seq[j] = (int32_t)s;
      slot[j] = (page_at(s, at >> t.shift) << t.shift) + (int32_t)(at & (page - 1));
    }
    if (i + 4 <= p.tokens) {
      *(int4 *)(p.slots + i) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *(int4 *)(p.positions + i) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      *(int4 *)(p.sequences + i) = make_int4(seq[0], seq[1], seq[2], seq[3]);
    } else {
      for (uint32_t j = 0; i + j < p.tokens; ++j) {
        p.slots[i + j] = slot[j];
        p.positions[i + j] = pos[j];
        p.sequences[i + j] = seq[j];
      }
    }
  }
  // ---- and the runs ----
  for (uint32_t i = me; i < p.most_runs; i += threads) {
    int4 r = make_int4(0, 0, 0, 0);
    if (i < runs) {
      const uint32_t s = find_seq(q.runs, n, i), kept = q.kept[s], end = kept + q.fresh[s];
      const uint32_t col = (kept >> t.shift) + i - q.runs[s];
      const uint32_t a = max(kept, col << t.shift), b = min(end, (col + 1) << t.shift);
      r = make_int4((int32_t)(q.start[s] + a - kept), page_at(s, col), (int32_t)(a & (page - 1)), (int32_t)(b - a));
    }
    p.runs[i] = r;
  }
}

}  // namespace vg
