// Append to a paged cache: the step's new rows into their pages, and the summaries
// of the pages that got rows.
//
// A run is what a step adds to one page. A block, or where there are many a warp,
// takes a (run, KV head): lanes of 16 bytes of a cache row, K and V side by side. The
// extremes of K are taken in the cache's own type, two channels an instruction, on
// the values as they are stored; rows that the page held before are read back for
// it. Values past the largest finite number of the cache's type are held as that one:
// attention multiplies rows by the terms of split numbers, and an infinity times a
// term of 0 would be NaN. 65,000 rows of 8 KV heads, bf16, with summaries (489 MB): 90 us,
// 83% of the measured copy rate; a row for each of 16 streams: 2.2 us, the launch.
#pragma once
#include <type_traits>

#include "kv4_rows.cuh"
#include "paged.cuh"

namespace vg {

struct PagedAppendParams {
  PagedView c;
  const void *k, *v;
  Strides ks, vs;         // token and head
  const int4 *runs;
  uint32_t tokens, most_runs;
};

constexpr uint32_t kPagedRowThreads = 256, kPagedRowBlocks = 4;   // blocks: resident on an SM

template <typename C>
using Pair = typename std::conditional<std::is_same<C, __half>::value, __half2, __nv_bfloat162>::type;
template <typename P>
__device__ __forceinline__ P pair_of(uint32_t bits) { return *reinterpret_cast<P *>(&bits); }
template <typename P>
__device__ __forceinline__ uint32_t pair_bits(P x) { return *reinterpret_cast<uint32_t *>(&x); }

template <typename C>
constexpr uint32_t kLargestBits = std::is_same<C, __half>::value ? 0x7BFF7BFFu : 0x7F7F7F7Fu;   // finite, twice
template <typename C>
constexpr uint32_t kInfBits = std::is_same<C, __half>::value ? 0x7C007C00u : 0x7F807F80u;

// Eight values of type T as eight of the cache's, rounded to nearest; what is past its largest finite number is held as
// that, NaN as NaN, and `odd` says that there were such.
__device__ __forceinline__ uint32_t round_pair(float x, float y, __half) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t round_pair(float x, float y, __nv_bfloat16) {
  uint32_t r;
  asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  return r;
}
template <typename T, typename C, bool VEC>
__device__ __forceinline__ uint4 load_rounded(const T *p, bool &odd) {
  using P = Pair<C>;
  uint32_t w[4];
  if constexpr (std::is_same<T, C>::value) {
    uint4 x;
    if constexpr (VEC) {
      x = __ldg((const uint4 *)p);
    } else {
      __align__(16) C h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = p[i];
      x = *(const uint4 *)h;
    }
    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
    const P top = pair_of<P>(kLargestBits<C>), bottom = pair_of<P>(kLargestBits<C> | 0x80008000u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pair_bits(__hmin2_nan(__hmax2_nan(pair_of<P>(y[i]), bottom), top));
      odd |= __heq2_mask(pair_of<P>(w[i]), pair_of<P>(y[i])) != ~0u;   // NaN equals nothing
    }
  } else {
    float x[8];
    load8<T, VEC>(p, x);
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7FFFFFFFu);   // NaN and infinities are the largest
    odd |= most > (std::is_same<C, __half>::value ? 0x477FE000u : 0x7F7F0000u);          // the largest of C
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = round_pair(x[2 * i], x[2 * i + 1], C{});
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// W: warps of a (run, KV head), 8 or 1. With one there are no block barriers, and a warp has four rows of K and of V in
// flight (90 us for the prompts above; with blocks 107); with 8 a single token's page is read back by a whole block.
template <int D, typename T, typename C, bool VEC, bool SUM, int W>
__global__ void __launch_bounds__(kPagedRowThreads, kPagedRowBlocks) paged_append_kernel(const PagedAppendParams p) {
  constexpr uint32_t L = D / 8;                       // lanes of a row
  constexpr uint32_t kRows = W * 32 / L;              // rows a pass
  constexpr uint32_t kGroups = kPagedRowThreads / 32 / W;
  using P = Pair<C>;
  __shared__ uint4 ends[SUM && W > 1 ? W : 1][2][L];
  const PagedTable &t = p.c.t;
  const uint32_t lane = threadIdx.x % L, slot = threadIdx.x % (W * 32) / L, page_rows = t.page_rows();
  const uint32_t items = p.most_runs * p.c.kv_heads, stride = gridDim.x * kGroups;   // the host keeps items below 2^31
  bool odd = false;   // met a NaN, or a value past the largest that the cache holds
  pdl_launch_dependents();
  pdl_wait();
  uint32_t item = blockIdx.x * kGroups + threadIdx.x / (W * 32);
  int4 next = item < items ? p.runs[item / p.c.kv_heads] : make_int4(0, 0, 0, 0);
  for (; item < items; item += stride) {
    const int4 r = next;
    if (item + stride < items) next = p.runs[(item + stride) / p.c.kv_heads];
    const uint32_t head = item % p.c.kv_heads;
    const uint32_t first = (uint32_t)r.x, page = (uint32_t)r.y, at = (uint32_t)r.z, rows = (uint32_t)r.w;
    if (!rows) break;   // runs past the last are empty
    if (page >= t.pages || at >= page_rows || rows > page_rows - at || first >= p.tokens || rows > p.tokens - first) continue;
    const size_t place = (size_t)page * p.c.kv_heads + head;
    C *k_page = (C *)p.c.data + place * 2 * page_rows * D + lane * 8, *v_page = k_page + (size_t)page_rows * D;
    P low[4], high[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) low[i] = pair_of<P>(kInfBits<C>), high[i] = pair_of<P>(kInfBits<C> | 0x80008000u);
    const auto widen = [&](const uint4 &x) {
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) low[i] = __hmin2(low[i], pair_of<P>(w[i])), high[i] = __hmax2(high[i], pair_of<P>(w[i]));
    };
    const T *k = (const T *)p.k + (int64_t)first * p.ks.token + (int64_t)head * p.ks.head + lane * 8;
    const T *v = (const T *)p.v + (int64_t)first * p.vs.token + (int64_t)head * p.vs.head + lane * 8;
#pragma unroll(W == 1 && sizeof(T) == 2 ? 4 : 2)
    for (uint32_t i = slot; i < rows; i += kRows) {
      const uint4 a = load_rounded<T, C, VEC>(k + (int64_t)i * p.ks.token, odd);
      const uint4 b = load_rounded<T, C, VEC>(v + (int64_t)i * p.vs.token, odd);
      *(uint4 *)(k_page + (size_t)(at + i) * D) = a;
      *(uint4 *)(v_page + (size_t)(at + i) * D) = b;
      if constexpr (SUM) widen(a);
    }
    if constexpr (SUM) {
#pragma unroll 4
      for (uint32_t i = slot; i < at; i += kRows) widen(*(const uint4 *)(k_page + (size_t)i * D));   // rows that it had
      // over the rows of a warp, then over the warps
#pragma unroll
      for (uint32_t o = L; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          low[i] = __hmin2(low[i], pair_of<P>(__shfl_xor_sync(~0u, pair_bits(low[i]), o)));
          high[i] = __hmax2(high[i], pair_of<P>(__shfl_xor_sync(~0u, pair_bits(high[i]), o)));
        }
      }
      uint4 *out = (uint4 *)((C *)p.c.summaries + place * 2 * D);
      // a channel whose rows are all NaN has kept +inf and -inf: 0 and 0
      const auto pack = [&](const P(&x)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pair_bits(x[i]) & ~__hgt2_mask(low[i], high[i]);
        return make_uint4(w[0], w[1], w[2], w[3]);
      };
      if constexpr (W == 1) {
        if (threadIdx.x % 32 < L) out[lane] = pack(low), out[L + lane] = pack(high);
      } else {
        const uint32_t warp = threadIdx.x / 32;
        if (threadIdx.x % 32 < L) {
          ends[warp][0][lane] = make_uint4(pair_bits(low[0]), pair_bits(low[1]), pair_bits(low[2]), pair_bits(low[3]));
          ends[warp][1][lane] = make_uint4(pair_bits(high[0]), pair_bits(high[1]), pair_bits(high[2]), pair_bits(high[3]));
        }
        __syncthreads();
        if (threadIdx.x < D / 2) {   // two channels a thread
          const uint32_t c = threadIdx.x;
          P a = pair_of<P>(((const uint32_t *)ends[0][0])[c]), b = pair_of<P>(((const uint32_t *)ends[0][1])[c]);
#pragma unroll
          for (uint32_t w = 1; w < W; ++w) {
            a = __hmin2(a, pair_of<P>(((const uint32_t *)ends[w][0])[c]));
            b = __hmax2(b, pair_of<P>(((const uint32_t *)ends[w][1])[c]));
          }
          const uint32_t none = __hgt2_mask(a, b);
          ((uint32_t *)out)[c] = pair_bits(a) & ~none;
          ((uint32_t *)out)[D / 2 + c] = pair_bits(b) & ~none;
        }
        __syncthreads();
      }
    }
  }
  if (odd) atomicOr(&t.pool[1], kPagedNonFinite);
}

}  // namespace vg
