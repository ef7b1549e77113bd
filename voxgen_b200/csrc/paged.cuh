// A paged KV cache: its layout, and what every kernel that touches it shares.
//
// Pool. [pages][kv_heads][K, V][page rows][head_dim] in fp16 or bf16: the K rows
// of a (page, KV head) are one run, its V rows the next. A page has 16 to 256
// rows, a power of two, so a block of 16 rows never leaves its page.
//
// Summaries. [pages][kv_heads][smallest, largest][head_dim] of the cache's type:
// per channel the extremes of K over the rows that the page held at its last append.
// NaN is passed over (a channel of NaN alone has 0 and 0), and append stores no
// infinity, so a summary of its rows is finite. A step that cuts rows of a page and adds
// none there leaves the summary: a bound for the rows left, until the next append.
//
// Table. table[seqs][seq_pages] names the pages of a sequence in order, rows[seqs]
// says how many rows it holds, free[pages] is a stack of free pages whose height
// is pool[0]. Only the step kernel moves pages. Kernels that read rows check every
// page number that they take from the table, so a damaged table gives wrong values
// and no bad address.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "kv4_rows.cuh"
#include "ptx.cuh"

namespace vg {

enum : int32_t {
  kPagedFull = 1,      // a step's new rows would pass seq_pages
  kPagedNoPages = 2,   // the pool has no pages left for them
  kPagedBadCount = 4,  // a count below 0, or past the step's tokens
};
enum : int32_t {          // in pool[1]
  kPagedTimeout = 8,     // a bounded wait inside attention ran out
  kPagedNonFinite = 16,  // an append met a NaN, or a value past the largest that the cache holds
};

struct PagedTable {
  int32_t *table, *rows, *status, *free, *pool;
  uint32_t seqs, seq_pages, pages, shift;   // shift: log2 of a page's rows
  __host__ __device__ __forceinline__ uint32_t page_rows() const { return 1u << shift; }
  __host__ __device__ __forceinline__ uint32_t capacity() const { return seq_pages << shift; }
};

struct PagedView {
  PagedTable t;
  void *data, *summaries;
  uint32_t kv_heads;
};

// Which rows a query attends: rows 0 .. seen - 1 of sequence seq.
struct PagedQueries {
  const int32_t *sequences;   // of each query, may be null: query i is sequence i's
  const int32_t *positions;   // last row that a query attends, may be null: all that are held
};
struct PagedSeen {
  uint32_t seq, seen;
};
__device__ __forceinline__ uint32_t paged_held(const PagedTable &t, uint32_t s) {
  return (uint32_t)min(max(t.rows[s], 0), (int32_t)t.capacity());
}
__device__ __forceinline__ PagedSeen paged_seen(const PagedTable &t, const PagedQueries &q, uint32_t i) {
  const int32_t s = q.sequences ? q.sequences[i] : (int32_t)i;
  if ((uint32_t)s >= t.seqs) return {0, 0};
  uint32_t n = paged_held(t, s);
  if (q.positions) n = min(n, (uint32_t)max(q.positions[i], -1) + 1u);
  return {(uint32_t)s, n};
}

// ---- cluster -----------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// Every thread of every CTA of the cluster; what was written before is seen after.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The two halves of that.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of a place of this CTA's shared memory in CTA `rank`'s, and a store there.
__device__ __forceinline__ uint32_t remote_smem(const void *p, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void st_remote(uint32_t address, uint64_t x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(address), "l"(x) : "memory");
}

}  // namespace vg
