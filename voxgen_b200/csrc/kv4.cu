// C entry points of the 4-bit KV cache and of draft verification
// (include/voxgen_cuda.h). They work on the caller's device buffers, enqueue on
// the caller's stream and return after the launch; no C++ exception is thrown.
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/voxgen_cuda.h"
#include "entry.cuh"
#include "kv4_rows.cuh"
#include "kv4_rows_attention.cuh"
#include "kv4_tile_attention.cuh"
#include "kv4_weights.cuh"
#include "verify_kernel.cuh"

using namespace vg;

namespace {

int shape_status(uint64_t seqs, uint64_t kv_heads, uint32_t head_dim, uint32_t capacity) {
  if (!seqs || !kv_heads || !capacity) return VG_EINVAL;
  if (head_dim != 64 && head_dim != 128) return VG_EUNSUPPORTED;
  if (capacity > 0x40000000u || seqs * kv_heads > kMaxGrid) return VG_ERANGE;
  return VG_OK;
}

int view_of(const vg_kv4_cache *c, Kv4View *v) {
  if (!c || !c->data || !c->state) return VG_EINVAL;
  if (!aligned(c->data, 16) || !aligned(c->state, 16) || !aligned(c->weights, 4) || !aligned(c->positions, 4))
    return VG_EINVAL;
  const int rc = shape_status(c->seqs, c->kv_heads, c->head_dim, c->capacity);
  if (rc) return rc;
  *v = Kv4View{(uint8_t *)c->data, (Kv4Seq *)c->state, c->weights, c->positions,
               c->seqs,            c->kv_heads,        c->capacity, kv4_tiles(c->capacity)};
  return VG_OK;
}

// Strides in elements {sequence, token, head}; NULL: [seqs][tokens][heads][head_dim].
Strides strides_of(const int64_t *s, uint32_t tokens, uint32_t heads, uint32_t head_dim) {
  const int64_t row = (int64_t)heads * head_dim;
  return s ? Strides{s[0], s[1], s[2]} : Strides{row * tokens, row, (int64_t)head_dim};
}

// 16-byte loads need the base and every row on a 16-byte boundary.
bool wide(const void *p, const Strides &s, size_t size) {
  const int64_t n = (int64_t)(16 / size);
  return aligned(p, 16) && s.seq % n == 0 && s.token % n == 0 && s.head % n == 0;
}

// Blocks of a sequence for `items` (token, head) pairs: no more than have a pass to
// make, and no more in all than are resident at once (per_sm of them on each SM),
// so that no second wave runs with a few.
uint32_t row_blocks(uint64_t items, uint32_t per_block, uint32_t seqs, uint32_t per_sm) {
  const uint64_t most = (items + per_block - 1) / per_block;
  return (uint32_t)std::min<uint64_t>(most, std::max(1u, 148 * per_sm / seqs));
}

// Attention workspace: counters (zero between calls, at the same place for every
// shape), partial results, then the softmax denominators.
constexpr uint64_t kTicketBytes = kMostTickets * 4;
uint64_t segments_of(const vg_kv4_cache *c, uint32_t heads, uint32_t tokens) {
  const uint64_t rows = (uint64_t)tokens * (heads / c->kv_heads);
  return (rows + kTileRows - 1) / kTileRows * c->kv_heads * c->seqs;
}
// Query rows of a (sequence, KV head) from which on the 128-row kernel is taken: 16 ragged streams with 16 rows each take
// 14 us with two passes of the few-row kernel, with 24 rows 22 us with the other.
constexpr uint64_t kTileFrom = 17;
// Segments of 256 rows from which on they are worth it: with 32 of them a prompt of 512 tokens takes 40 us against 24 with
// twice as many of 128 rows; with 64, 1024 tokens over 8192 rows take 113 us against 137.
constexpr uint64_t kPairFrom = 48;
bool tiled(const vg_kv4_cache *c, uint32_t heads, uint32_t tokens) {
  return (uint64_t)tokens * (heads / c->kv_heads) >= kTileFrom;
}
// Whether 16-bit queries are taken 256 rows at a time: an unpacked tile then serves
// twice as many rows, but there are half as many segments to share out.
bool paired(const vg_kv4_cache *c, uint32_t heads, uint32_t tokens) {
  const uint64_t rows = (uint64_t)tokens * (heads / c->kv_heads);
  return (rows + 2 * kTileM - 1) / (2 * kTileM) * c->kv_heads * c->seqs >= kPairFrom;
}
// The most units of cache rows that a call can have over all its segments.
uint64_t units_of_call(const vg_kv4_cache *c, uint32_t heads, uint32_t tokens) {
  const uint64_t rows = (uint64_t)tokens * (heads / c->kv_heads), lanes = (uint64_t)c->kv_heads * c->seqs;
  if (tiled(c, heads, tokens)) return (rows + kTileM - 1) / kTileM * lanes * ((c->capacity + kTileN - 1) / kTileN);
  return segments_of(c, heads, tokens) * ((c->capacity + kUnit - 1) / kUnit);
}
uint64_t part_bytes(const vg_kv4_cache *c, uint32_t heads, uint32_t tokens) {
  if (tiled(c, heads, tokens)) return (uint64_t)kTileSlots * 2 * kTileM * (c->head_dim + 2) * 4;
  return most_pieces(segments_of(c, heads, tokens)) * kTileRows * (c->head_dim + 2) * 4;
}

}  // namespace

extern "C" {

int vg_k_kv4_bytes(uint32_t seqs, uint32_t kv_heads, uint32_t head_dim, uint32_t capacity, uint64_t *bytes) {
  if (!bytes) return VG_EINVAL;
  const int rc = shape_status(seqs, kv_heads, head_dim, capacity);
  if (rc) return rc;
  const uint64_t tile = head_dim == 64 ? Kv4<64>::kTileBytes : Kv4<128>::kTileBytes;
  *bytes = (uint64_t)seqs * kv_heads * kv4_tiles(capacity) * tile;
  return VG_OK;
}

int vg_k_kv4_append(const vg_kv4_cache *cache, const void *k, const void *v, int dtype, uint32_t tokens,
                    const int64_t *k_strides, const int64_t *v_strides, const int32_t *at, const int32_t *counts,
                    void *cuda_stream) {
  AppendParams p{};
  const int rc = view_of(cache, &p.c);
  if (rc) return rc;
  const size_t size = type_size(dtype);
  if (!size) return VG_EUNSUPPORTED;
  if (!k || !v || !tokens || !aligned(k, size) || !aligned(v, size) || !aligned(at, 4) || !aligned(counts, 4))
    return VG_EINVAL;
  if (tokens > cache->capacity) return VG_EFULL;
  p.k = k;
  p.v = v;
  p.ks = strides_of(k_strides, tokens, cache->kv_heads, cache->head_dim);
  p.vs = strides_of(v_strides, tokens, cache->kv_heads, cache->head_dim);
  p.at = at;
  p.counts = counts;
  p.tokens = tokens;
  const uint64_t items = (uint64_t)tokens * cache->kv_heads;
  const uint32_t per_block = kRowThreads / (cache->head_dim / 16);
  if (items > kMaxGrid) return VG_ERANGE;
  p.blocks = row_blocks(items, per_block, cache->seqs, kAppendBlocks);
  const bool vec = wide(k, p.ks, size) && wide(v, p.vs, size);
  const dim3 grid(p.blocks * cache->seqs);
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  return by_dim(cache->head_dim, [&](auto d) {
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (vec) kv4_append_kernel<decltype(d)::value, T, true><<<grid, kRowThreads, 0, st>>>(p);
      else kv4_append_kernel<decltype(d)::value, T, false><<<grid, kRowThreads, 0, st>>>(p);
      return launched();
    });
  });
}

int vg_k_kv4_read(const vg_kv4_cache *cache, const int32_t *first, uint32_t tokens, int dtype, void *k, void *v,
                  void *cuda_stream) {
  ReadParams p{};
  const int rc = view_of(cache, &p.c);
  if (rc) return rc;
  if (!type_size(dtype)) return VG_EUNSUPPORTED;
  if (!k || !v || !tokens || !aligned(k, 16) || !aligned(v, 16) || !aligned(first, 4)) return VG_EINVAL;
  p.k = k;
  p.v = v;
  p.first = first;
  p.tokens = tokens;
  const uint32_t per_block = kRowThreads / (cache->head_dim / 8);
  const uint64_t items = (uint64_t)tokens * cache->kv_heads;
  if (items > kMaxGrid) return VG_ERANGE;
  p.blocks = row_blocks(items, per_block, cache->seqs, 8);
  const dim3 grid(p.blocks * cache->seqs);
  return by_dim(cache->head_dim, [&](auto d) {
    return by_type(dtype, [&](auto t) {
      kv4_read_kernel<decltype(d)::value, decltype(t)><<<grid, kRowThreads, 0, (cudaStream_t)cuda_stream>>>(p);
      return launched();
    });
  });
}

int vg_k_kv4_attention_bytes(const vg_kv4_cache *cache, uint32_t heads, uint32_t tokens, uint64_t *bytes) {
  Kv4View v;
  const int rc = view_of(cache, &v);
  if (rc) return rc;
  if (!bytes || !heads || !tokens || heads % cache->kv_heads) return VG_EINVAL;
  if ((uint64_t)heads * tokens > kMaxGrid / cache->seqs) return VG_ERANGE;
  if (units_of_call(cache, heads, tokens) > kMaxGrid) return VG_ERANGE;   // counted in 32 bits
  *bytes = kTicketBytes + part_bytes(cache, heads, tokens) + (uint64_t)cache->seqs * tokens * heads * 4;
  return VG_OK;
}

int vg_k_kv4_attention(const vg_kv4_cache *cache, const void *q, int dtype, uint32_t heads, uint32_t tokens,
                       const int64_t *q_strides, const int32_t *counts, float scale, int track, void *out,
                       void *workspace, uint64_t workspace_bytes, void *cuda_stream) {
  Kv4AttnParams p{};
  uint64_t need = 0;
  int rc = vg_k_kv4_attention_bytes(cache, heads, tokens, &need);
  if (rc) return rc;
  if ((rc = view_of(cache, &p.c))) return rc;
  const size_t size = type_size(dtype);
  if (!size) return VG_EUNSUPPORTED;
  if (!q || !out || !workspace || workspace_bytes < need || !aligned(q, size) || !aligned(out, 16) ||
      !aligned(workspace, 16) || !aligned(counts, 4) || (track && !cache->weights) || !(scale > 0.f) ||
      !(scale < __builtin_huge_valf()) || (track && out == q))   // the tracking kernel reads q while out is written
    return VG_EINVAL;
  uint8_t *ws = (uint8_t *)workspace;
  p.q = q;
  p.out = out;
  p.tickets = (uint32_t *)ws;
  p.parts = (float *)(ws + kTicketBytes);
  p.lse = track ? (float *)(ws + kTicketBytes + part_bytes(cache, heads, tokens)) : nullptr;
  p.qs = strides_of(q_strides, tokens, heads, cache->head_dim);
  p.wide = wide(q, p.qs, size);
  p.counts = counts;
  p.tokens = tokens;
  p.heads = heads;
  p.group = heads / cache->kv_heads;
  p.scale = scale * 1.44269504088896340736f;
  const bool tile = tiled(cache, heads, tokens);
  const bool pair = tile && size == 2 && paired(cache, heads, tokens);
  const uint32_t block = !tile ? kTileRows : pair ? 2 * kTileM : kTileM;   // query rows that a CTA takes at a time
  p.row_tiles = (tokens * p.group + block - 1) / block;
  const uint64_t blocks = ((uint64_t)cache->capacity + kWeightRows - 1) / kWeightRows * cache->seqs * cache->kv_heads;
  if (track && blocks > kMaxGrid) return VG_ERANGE;
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  return by_dim(cache->head_dim, [&](auto d) {
    return by_type(dtype, [&](auto t) {
      using T = decltype(t);
      constexpr int D = decltype(d)::value;
      static std::atomic<uint64_t> done[3];
      if (tile) {
        const auto go = [&](auto fn, std::atomic<uint64_t> &set) {
          const int e = allow_smem((const void *)fn, TileSmem<D>::kBytes, set, (kSoftmaxRegs + kOtherRegs) / 2);
          if (!e) fn<<<kTileCtas, kTileThreads, TileSmem<D>::kBytes, st>>>(p);
          return e;
        };
        int e;
        if constexpr (sizeof(T) == 2) {
          e = pair ? go(kv4_tile_kernel<D, T, true>, done[2]) : go(kv4_tile_kernel<D, T, false>, done[0]);
        } else {
          e = go(kv4_tile_kernel<D, T, false>, done[0]);
        }
        if (e) return e;
      } else {
        const auto fn = kv4_rows_kernel<D, T>;
        const int e = allow_smem((const void *)fn, RowsSmem<D>::kBytes, done[1]);
        if (e) return e;
        fn<<<kRowsCtas, kRowsThreads, RowsSmem<D>::kBytes, st>>>(p);
      }
      if (track) {   // starts as the attention's CTAs leave, and waits for the last of them where it needs their sums
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((uint32_t)blocks);
        cfg.blockDim = dim3(kWeightThreads);
        cfg.dynamicSmemBytes = kWeightSmem<D, T>;
        cfg.stream = st;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        const cudaError_t err = cudaLaunchKernelEx(&cfg, kv4_weights_kernel<D, T>, p);
        if (err != cudaSuccess) return VG_ECUDA;
      }
      return launched();
    });
  });
}

int vg_k_kv4_evict(const vg_kv4_cache *cache, uint32_t budget, uint32_t recent, uint32_t sinks,
                   const vg_kv4_cache *into, void *cuda_stream) {
  EvictParams p{};
  int rc = view_of(cache, &p.c);
  if (rc) return rc;
  if (!cache->weights || !cache->positions || !budget) return VG_EINVAL;
  if (budget > cache->capacity || (uint64_t)recent + sinks > budget) return VG_ERANGE;
  if (cache->capacity > 65536) return VG_ERANGE;
  if (into) {
    Kv4View o;
    if ((rc = view_of(into, &o))) return rc;
    if (!into->weights || !into->positions || into->data != cache->data || into->seqs != cache->seqs ||
        into->kv_heads != cache->kv_heads || into->head_dim != cache->head_dim || into->capacity != cache->capacity)
      return VG_EINVAL;
    const int same = (into->state == cache->state) + (into->weights == cache->weights) + (into->positions == cache->positions);
    if (same != 0 && same != 3) return VG_EINVAL;
  }
  const vg_kv4_cache *o = into ? into : cache;
  p.state_out = (Kv4Seq *)o->state;
  p.weights_out = o->weights;
  p.positions_out = o->positions;
  p.budget = budget;
  p.recent = recent;
  p.sinks = sinks;
  p.list = std::min(budget, cache->capacity - budget);
  const size_t rest = kEvictBins * 4 + (size_t)p.list * 4, with_keys = rest + (size_t)cache->capacity * 4;
  const bool keys = with_keys <= kEvictSmem;
  return by_dim(cache->head_dim, [&](auto d) {
    constexpr int D = decltype(d)::value;
    const auto go = [&](auto fn, std::atomic<uint64_t> &done) {
      const int e = allow_smem((const void *)fn, kEvictSmem, done);
      if (e) return e;
      fn<<<cache->seqs * cache->kv_heads, kEvictThreads, keys ? with_keys : rest, (cudaStream_t)cuda_stream>>>(p);
      return launched();
    };
    static std::atomic<uint64_t> done[2];
    return keys ? go(kv4_evict_kernel<D, true>, done[0]) : go(kv4_evict_kernel<D, false>, done[1]);
  });
}

int vg_k_verify_draft(const int32_t *tokens, const float *draft, const float *target, const float *u_accept,
                      const float *u_sample, const int32_t *counts, uint32_t seqs, uint32_t drafted, uint32_t vocab,
                      int32_t *accepted, int32_t *next, void *cuda_stream) {
  if (!tokens || !draft || !target || !u_accept || !u_sample || !accepted || !next || !seqs || !drafted || !vocab)
    return VG_EINVAL;
  for (const void *q : {(const void *)tokens, (const void *)draft, (const void *)target, (const void *)u_accept,
                        (const void *)u_sample, (const void *)counts, (const void *)accepted, (const void *)next})
    if (!aligned(q, 4)) return VG_EINVAL;
  if (seqs > kMaxGrid / kVerifyCtas || vocab > kVerifyVocab || drafted > 0x100000u) return VG_ERANGE;
  const VerifyParams p{tokens, draft, target, u_accept, u_sample, counts, accepted, next, drafted, vocab};
  const cudaStream_t st = (cudaStream_t)cuda_stream;
  if (vocab % 4 == 0 && aligned(draft, 16) && aligned(target, 16))
    verify_draft_kernel<true><<<seqs * kVerifyCtas, kVerifyThreads, 0, st>>>(p);
  else
    verify_draft_kernel<false><<<seqs * kVerifyCtas, kVerifyThreads, 0, st>>>(p);
  return launched();
}

}  // extern "C"
