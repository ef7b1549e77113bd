// C entry points of the paged KV cache (include/voxgen_cuda.h). They work on the
// caller's device buffers, enqueue on the caller's stream and return after the
// launch; no C++ exception is thrown.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../../include/voxgen_cuda.h"
#include "entry.cuh"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "paged_rows.cuh"
#include "paged_select.cuh"
#include "paged_table.cuh"

using namespace vg;

namespace {

bool page_size(uint32_t rows) { return rows >= 16 && rows <= 256 && (rows & (rows - 1)) == 0; }

int table_of(const vg_paged_table *t, PagedTable *v) {
  if (!t || !t->table || !t->rows || !t->status || !t->free || !t->pool) return VG_EINVAL;
  for (const void *p : {(const void *)t->table, (const void *)t->rows, (const void *)t->status, (const void *)t->free,
                        (const void *)t->pool})
    if (!aligned(p, 4)) return VG_EINVAL;
  if (!t->seqs || !t->seq_pages || !t->pages) return VG_EINVAL;
  if (!page_size(t->page_rows)) return VG_EUNSUPPORTED;
  if (t->seqs > kStepSeqs || (uint64_t)t->pages * t->page_rows > 0x7FFFFFFFu ||
      (uint64_t)t->seq_pages * t->page_rows > 0x40000000u)
    return VG_ERANGE;
  *v = PagedTable{t->table, t->rows, t->status, t->free, t->pool, t->seqs, t->seq_pages, t->pages,
                  (uint32_t)__builtin_ctz(t->page_rows)};
  return VG_OK;
}

int cache_of(const vg_paged_cache *c, PagedView *v) {
  if (!c || !c->data || !aligned(c->data, 16) || !aligned(c->summaries, 32) || !c->kv_heads) return VG_EINVAL;
  if (c->dtype != VG_DTYPE_F16 && c->dtype != VG_DTYPE_BF16) return VG_EUNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return VG_EUNSUPPORTED;
  const int rc = table_of(c->table, &v->t);
  if (rc) return rc;
  if ((uint64_t)v->t.pages * c->kv_heads > kMaxGrid) return VG_ERANGE;   // a coordinate of the copies
  v->data = c->data;
  v->summaries = c->summaries;
  v->kv_heads = c->kv_heads;
  return VG_OK;
}

uint32_t runs_of(const PagedTable &t, uint32_t tokens) {
  return (uint32_t)std::min<uint64_t>(tokens, (uint64_t)(tokens >> t.shift) + 2ull * t.seqs);
}

int step_of(const vg_paged_step *s) {
  if (!s || !s->starts || !s->slots || !s->positions || !s->sequences || !s->runs) return VG_EINVAL;
  for (const void *p : {(const void *)s->starts, (const void *)s->slots, (const void *)s->positions,
                        (const void *)s->sequences, (const void *)s->runs})
    if (!aligned(p, 16)) return VG_EINVAL;
  return s->tokens > 0x40000000u ? VG_ERANGE : VG_OK;
}

// Every launch may start while the kernel before it on the stream finishes: each of
// these kernels waits for that one before it reads or writes global memory.
template <typename... A>
int launch(void (*fn)(A...), uint32_t grid, uint32_t cluster, uint32_t threads, size_t smem, void *stream, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, args...);
  if (e != cudaSuccess) cudaGetLastError();   // reported here, and not by a later call
  return e == cudaSuccess ? VG_OK : e == cudaErrorMemoryAllocation ? VG_ENOMEM : VG_ECUDA;
}

template <typename F>
int by_cache_type(int dtype, F &&f) {
  return dtype == VG_DTYPE_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

// The pool as a tensor of {channel, row, K or V, (page, KV head)} and boxes of 64 channels, 16 rows, K and V.
int pool_map(const PagedView &c, int dtype, uint32_t head_dim, CUtensorMap *map) {
  typedef CUresult (*Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<void *> found{nullptr};
  void *fn = found.load(std::memory_order_acquire);
  if (!fn) {
    cudaDriverEntryPointQueryResult how;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &how) != cudaSuccess ||
        how != cudaDriverEntryPointSuccess || !fn) {
      cudaGetLastError();
      return VG_ECUDA;
    }
    found.store(fn, std::memory_order_release);
  }
  const uint64_t rows = c.t.page_rows(), row = (uint64_t)head_dim * 2;
  const cuuint64_t dims[4] = {head_dim, rows, 2, (uint64_t)c.t.pages * c.kv_heads};
  const cuuint64_t strides[3] = {row, rows * row, 2 * rows * row};
  const cuuint32_t box[4] = {64, kPagedBlock, 2, 1}, ones[4] = {1, 1, 1, 1};
  const CUresult r = ((Encode)fn)(
      map, dtype == VG_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, c.data, dims, strides,
      box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? VG_OK : VG_ECUDA;
}

// The arguments that select and attention share.
struct Queries {
  uint32_t group;
  int64_t query, head;   // strides
};
int queries_of(const PagedView &c, uint32_t head_dim, const void *q, int dtype, uint32_t queries, uint32_t heads,
               const int64_t *strides, const int32_t *sequences, const int32_t *positions, Queries *out) {
  const size_t size = type_size(dtype);
  if (!size) return VG_EUNSUPPORTED;
  if (!q || !aligned(q, size) || !queries || !heads || heads % c.kv_heads || !aligned(sequences, 4) || !aligned(positions, 4))
    return VG_EINVAL;
  if (!sequences && queries > c.t.seqs) return VG_EINVAL;   // query i would have no sequence
  out->group = heads / c.kv_heads;
  out->query = strides ? strides[0] : (int64_t)heads * head_dim;
  out->head = strides ? strides[1] : (int64_t)head_dim;
  return VG_OK;
}

constexpr uint64_t kPagedTicketBytes = kPagedTickets * 4;
// How the tiles of 8 heads of a KV head make segments.
struct Tiling {
  uint32_t tiles, lanes;               // of a segment (1, 2 or 4), segments of a query
  uint32_t warps;                      // consumer warps of a CTA
  bool share;                          // consecutive queries of a sequence may make one segment
};
Tiling tiling_of(uint32_t kv_heads, uint32_t heads, uint32_t queries, uint32_t budget) {
  Tiling x{};
  const uint32_t head_tiles = (heads / kv_heads + kPagedHeads - 1) / kPagedHeads;   // of a KV head
  x.share = head_tiles == 1 && !budget;   // lists of pages differ from query to query
  x.tiles = 1;
  while (x.tiles < kPagedTiles && x.tiles < head_tiles) x.tiles *= 2;
  x.lanes = kv_heads * ((head_tiles + kPagedTiles - 1) / kPagedTiles);
  x.warps = (uint64_t)queries * x.lanes < kPagedMany ? kPagedWarps : kPagedFew;
  return x;
}

uint64_t blocks_of(const PagedTable &t, uint32_t budget) {   // of a segment, at most
  return (uint64_t)(budget ? budget : t.seq_pages) << (t.shift - 4);
}

}  // namespace

extern "C" {

int vg_k_paged_bytes(uint32_t pages, uint32_t page_rows, uint32_t kv_heads, uint32_t head_dim, uint64_t *data_bytes,
                     uint64_t *summary_bytes) {
  if (!data_bytes || !summary_bytes || !pages || !kv_heads) return VG_EINVAL;
  if (!page_size(page_rows) || (head_dim != 64 && head_dim != 128)) return VG_EUNSUPPORTED;
  if ((uint64_t)pages * page_rows > 0x7FFFFFFFu || (uint64_t)pages * kv_heads > kMaxGrid) return VG_ERANGE;
  const uint64_t heads = (uint64_t)pages * kv_heads;
  *data_bytes = heads * 2 * page_rows * head_dim * 2;
  *summary_bytes = heads * 2 * head_dim * 2;
  return VG_OK;
}

int vg_k_paged_runs(const vg_paged_table *table, uint32_t tokens, uint32_t *runs) {
  PagedTable t;
  const int rc = table_of(table, &t);
  if (rc) return rc;
  if (!runs) return VG_EINVAL;
  if (tokens > 0x40000000u) return VG_ERANGE;
  *runs = runs_of(t, tokens);
  return VG_OK;
}

int vg_k_paged_step(const vg_paged_table *table, const int32_t *counts, const int32_t *keep, const vg_paged_step *step,
                    void *cuda_stream) {
  StepParams p{};
  int rc = table_of(table, &p.t);
  if (rc) return rc;
  if ((rc = step_of(step))) return rc;
  if (!counts || !aligned(counts, 4) || !aligned(keep, 4)) return VG_EINVAL;
  p.counts = counts;
  p.keep = keep;
  p.starts = step->starts;
  p.slots = step->slots;
  p.positions = step->positions;
  p.sequences = step->sequences;
  p.runs = (int4 *)step->runs;
  p.tokens = step->tokens;
  p.most_runs = runs_of(p.t, step->tokens);
  static std::atomic<uint64_t> done;
  if ((rc = allow_smem((const void *)paged_step_kernel, kStepSeqs * kStepWords * 4, done))) return rc;
  // 8192 new tokens of 256 sequences take 9.1 us in eight CTAs and 11.0 in one, 4096 take 8.4 and 7.9. Pages given back do not
  // count, though 131072 of them with few tokens take 116 us in one CTA and 24 in eight.
  const uint32_t ctas = step->tokens > 4 * kStepThreads ? kStepCtas : 1;
  return launch(paged_step_kernel, ctas, ctas, kStepThreads, (size_t)table->seqs * kStepWords * 4, cuda_stream, p);
}

int vg_k_paged_append(const vg_paged_cache *cache, const vg_paged_step *step, const void *k, const void *v, int dtype,
                      const int64_t *k_strides, const int64_t *v_strides, void *cuda_stream) {
  PagedAppendParams p{};
  int rc = cache_of(cache, &p.c);
  if (rc) return rc;
  if ((rc = step_of(step))) return rc;
  const size_t size = type_size(dtype);
  if (!size) return VG_EUNSUPPORTED;
  if (!step->tokens) return VG_OK;   // no rows to point at
  if (!k || !v || !aligned(k, size) || !aligned(v, size)) return VG_EINVAL;
  const int64_t row = (int64_t)cache->kv_heads * cache->head_dim, head = cache->head_dim, wide = (int64_t)(16 / size);
  p.ks = k_strides ? Strides{0, k_strides[0], k_strides[1]} : Strides{0, row, head};
  p.vs = v_strides ? Strides{0, v_strides[0], v_strides[1]} : Strides{0, row, head};
  p.k = k;
  p.v = v;
  p.runs = (const int4 *)step->runs;
  p.tokens = step->tokens;
  p.most_runs = runs_of(p.c.t, step->tokens);
  // 16-byte loads need the base and every row on a 16-byte boundary
  const bool vec = aligned(k, 16) && aligned(v, 16) && p.ks.token % wide == 0 && p.ks.head % wide == 0 &&
                   p.vs.token % wide == 0 && p.vs.head % wide == 0;
  const uint64_t items = (uint64_t)p.most_runs * cache->kv_heads;
  if (items > kMaxGrid / 2) return VG_ERANGE;
  // a block an item while all are resident at once, else a warp an item: 65,000 rows of 8 KV heads take 107 us with blocks
  const bool blocks = items <= 148 * kPagedRowBlocks;
  const uint32_t warps = kPagedRowThreads / 32;
  const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks ? items : (items + warps - 1) / warps, 148 * kPagedRowBlocks);
  return by_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      return by_cache_type(cache->dtype, [&](auto c) {
        using C = decltype(c);
        const auto go = [&](auto fn) { return launch(fn, grid, 1, kPagedRowThreads, 0, cuda_stream, p); };
        const auto pick = [&](auto w) {
          constexpr int W = decltype(w)::value;
          if (cache->summaries)
            return vec ? go(paged_append_kernel<D, T, C, true, true, W>) : go(paged_append_kernel<D, T, C, false, true, W>);
          return vec ? go(paged_append_kernel<D, T, C, true, false, W>) : go(paged_append_kernel<D, T, C, false, false, W>);
        };
        return blocks ? pick(Dim<8>{}) : pick(Dim<1>{});
      });
    });
  });
}

int vg_k_paged_select(const vg_paged_cache *cache, const void *q, int dtype, uint32_t queries, uint32_t heads,
                      const int64_t *q_strides, const int32_t *sequences, const int32_t *positions, uint32_t budget,
                      uint32_t sinks, uint32_t recent, int32_t *chosen, void *cuda_stream) {
  PagedSelectParams p{};
  int rc = cache_of(cache, &p.c);
  if (rc) return rc;
  Queries x;
  if ((rc = queries_of(p.c, cache->head_dim, q, dtype, queries, heads, q_strides, sequences, positions, &x))) return rc;
  if (!cache->summaries || !chosen || !aligned(chosen, 4) || !budget) return VG_EINVAL;
  if (p.c.t.seq_pages > kSelectPages || (uint64_t)sinks + recent > budget) return VG_ERANGE;
  const uint64_t items = (uint64_t)queries * cache->kv_heads;
  if (items > kMaxGrid / 8 || budget > 0x40000000u) return VG_ERANGE;
  p.q = q;
  p.q_query = x.query;
  p.q_head = x.head;
  p.which = PagedQueries{sequences, positions};
  p.chosen = chosen;
  p.group = x.group;
  p.budget = budget;
  p.sinks = sinks;
  p.recent = recent;
  // CTAs of a (query, KV head): no more than are resident at once, one an SM, and have pages to score
  uint32_t ctas = 8;
  while (ctas > 1 && (items * ctas > 148 || (ctas - 1) * kSelectWarps * 16 >= p.c.t.seq_pages)) ctas /= 2;
  const size_t smem = (size_t)p.c.t.seq_pages * 8;
  return by_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      return by_cache_type(cache->dtype, [&](auto c) {
        const auto fn = paged_select_kernel<D, T, decltype(c)>;
        static std::atomic<uint64_t> done;
        const int e = allow_smem((const void *)fn, kSelectPages * 8, done);
        return e ? e : launch(fn, (uint32_t)items * ctas, ctas, kSelectThreads, smem, cuda_stream, p);
      });
    });
  });
}

int vg_k_paged_attention_bytes(const vg_paged_cache *cache, uint32_t queries, uint32_t heads, uint32_t budget,
                               uint64_t *bytes) {
  PagedView c;
  const int rc = cache_of(cache, &c);
  if (rc) return rc;
  if (!bytes || !queries || !heads || heads % cache->kv_heads) return VG_EINVAL;
  const Tiling x = tiling_of(c.kv_heads, heads, queries, budget);
  const uint64_t segments = (uint64_t)queries * x.lanes;
  const uint64_t blocks = blocks_of(c.t, budget);
  const uint64_t cost = segments * blocks * x.tiles;
  if (x.lanes > 1u << 16 || segments > kMaxGrid || blocks > kPagedMost || cost > kMaxGrid)
    return VG_ERANGE;   // the plan counts in 32 bits
  const uint64_t parts = (uint64_t)paged_slots(segments, paged_ctas(x.warps)) * (x.share ? kPagedTiles : x.tiles);
  *bytes = kPagedTicketBytes + parts * kPagedHeads * (cache->head_dim + 2) * 4;
  return VG_OK;
}

int vg_k_paged_attention(const vg_paged_cache *cache, const void *q, int dtype, uint32_t queries, uint32_t heads,
                         const int64_t *q_strides, const int32_t *sequences, const int32_t *positions, const int32_t *chosen,
                         uint32_t budget, float scale, void *out, void *workspace, uint64_t workspace_bytes,
                         void *cuda_stream) {
  uint64_t need = 0;
  if ((chosen != nullptr) != (budget != 0)) return VG_EINVAL;
  int rc = vg_k_paged_attention_bytes(cache, queries, heads, budget, &need);
  if (rc) return rc;
  PagedView c;
  if ((rc = cache_of(cache, &c))) return rc;
  Queries x;
  if ((rc = queries_of(c, cache->head_dim, q, dtype, queries, heads, q_strides, sequences, positions, &x))) return rc;
  if (!out || !workspace || workspace_bytes < need || !aligned(out, 16) || !aligned(workspace, 16) || !aligned(chosen, 4) ||
      out == q || !(scale > 0.f) || !(scale < __builtin_huge_valf()))
    return VG_EINVAL;
  PagedAttnParams p{};
  p.t = c.t;
  p.kv_heads = c.kv_heads;
  p.q = q;
  p.out = out;
  p.q_query = x.query;
  p.q_head = x.head;
  p.which = PagedQueries{sequences, positions};
  p.chosen = chosen;
  p.budget = budget;
  p.queries = queries;
  p.heads = heads;
  p.group = x.group;
  const Tiling tiling = tiling_of(c.kv_heads, heads, queries, budget);
  p.share = tiling.share && sequences;   // else every query is of its own sequence
  p.tiles = p.share ? kPagedTiles : tiling.tiles;
  p.lanes = tiling.lanes;
  const uint64_t blocks = blocks_of(c.t, budget);
  p.scale = scale * 1.44269504088896340736f;
  p.tickets = (uint32_t *)workspace;
  p.parts = (float *)((uint8_t *)workspace + kPagedTicketBytes);
  CUtensorMap map;
  if ((rc = pool_map(c, cache->dtype, cache->head_dim, &map))) return rc;
  return by_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      return by_cache_type(cache->dtype, [&](auto ct) {
        using C = decltype(ct);
        const auto go = [&](auto w, auto fresh) {
          constexpr int W = decltype(w)::value;
          using S = PagedSmem<D, W, kQTerms<T, C>>;
          const auto fn = paged_attention_kernel<D, T, C, W, decltype(fresh)::value>;
          static std::atomic<uint64_t> done;
          const int e = allow_smem((const void *)fn, S::kBytes, done);
          return e ? e : launch(fn, paged_ctas(W), 1, (W + 1) * 32, S::kBytes, cuda_stream, p, map);
        };
        const auto sums = [&](auto w) {
          const uint32_t teams = (uint32_t)decltype(w)::value / p.tiles;   // warps that share a piece's blocks, at least
          if constexpr (sizeof(T) == 2) {
            if ((blocks + teams - 1) / teams * kPTerms<C> <= kPagedProducts) return go(w, std::false_type{});
          }
          return go(w, std::true_type{});
        };
        return tiling.warps == kPagedWarps ? sums(Dim<(int)kPagedWarps>{}) : sums(Dim<(int)kPagedFew>{});
      });
    });
  });
}

}  // extern "C"
