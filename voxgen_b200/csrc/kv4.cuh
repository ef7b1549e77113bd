// A KV cache held in 4 bits: its layout, and the arithmetic every kernel that
// touches it shares.
//
// Values. A block is 32 consecutive channels of one row. It holds 32 codes n in
// [-8, 7] and one scale d, and stands for n*d. With x the block's values (NaN
// as 0, clamped to +-7168) and b its value of largest magnitude (the positive
// one where two tie),
//   d = -b/8 rounded to 7 significant bits, 0 when |d| < 2^-18
//   n = clamp(rint(x * (1/d)), -8, 7), 0 when d = 0.
// Mapping b to -8 uses the one code that has no opposite, so the step is 1/8 of
// the largest magnitude and not 1/7. The 7 bits are what makes n*d (3 + 7 bits)
// and 72*d (4 + 7 bits) exact fp16 numbers: tensor-core operands carry the
// cache's values without a rounding, and one fused multiply-add unpacks a pair
// of codes (unpack8). The clamp keeps 72*d finite in fp16.
//
// Layout. Per (sequence, KV head): tiles of 64 rows, each tile
//   K codes  64 x D/2 bytes   channel 2j in the low nibble of byte j, nibble = n + 8
//   V codes  64 x D/2 bytes
//   K scales 64 x D/32 fp16
//   V scales 64 x D/32 fp16
// so a tile is one contiguous copy of 72*D bytes (9,216 at head_dim 128, against
// 32,768 in fp16), and any range of whole rows is four.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace vg {

constexpr uint32_t kKv4Tile = 64;    // rows of a tile
constexpr uint32_t kKv4Block = 32;   // channels that share a scale
constexpr float kKv4Largest = 7168.f;
constexpr float kKv4Smallest = 0x1p-18f;

template <int D>
struct Kv4 {
  static constexpr uint32_t kRow = D / 2;         // code bytes of a row
  static constexpr uint32_t kScale = D / 16;      // scale bytes of a row
  static constexpr uint32_t kVCodes = kKv4Tile * kRow;
  static constexpr uint32_t kKScales = 2 * kKv4Tile * kRow;
  static constexpr uint32_t kVScales = kKScales + kKv4Tile * kScale;
  static constexpr uint32_t kTileBytes = kVScales + kKv4Tile * kScale;

  // byte offsets of a row's codes and scales within its (sequence, head) run
  static __host__ __device__ __forceinline__ size_t codes(uint32_t row, int v) {
    return (size_t)(row / kKv4Tile) * kTileBytes + (v ? kVCodes : 0) + (row % kKv4Tile) * kRow;
  }
  static __host__ __device__ __forceinline__ size_t scales(uint32_t row, int v) {
    return (size_t)(row / kKv4Tile) * kTileBytes + (v ? kVScales : kKScales) + (row % kKv4Tile) * kScale;
  }
};

__host__ __device__ __forceinline__ uint32_t kv4_tiles(uint32_t capacity) {
  return (capacity + kKv4Tile - 1) / kKv4Tile;
}

// One sequence's words in vg_kv4_cache.state.
struct Kv4Seq {
  int32_t rows, next, status, ticket;
};

enum : int32_t {
  kKv4Full = 1,       // an append went past the capacity
  kKv4BadRow = 2,     // an append started past the rows held, or its count is out of range
  kKv4NonFinite = 4,  // an append met a NaN, or a value past +-kKv4Largest
  kKv4Timeout = 8,    // a bounded wait inside attention ran out (sequence 0's word)
};

// Two fp32 operations in one instruction, and the extremes of three.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*(const uint64_t *)&a), "l"(*(const uint64_t *)&b), "l"(*(const uint64_t *)&c));
  return *(const float2 *)&d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(const uint64_t *)&a), "l"(*(const uint64_t *)&b));
  return *(const float2 *)&d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*(const uint64_t *)&a), "l"(*(const uint64_t *)&b));
  return *(const float2 *)&d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// d of a block from its extremes.
__device__ __forceinline__ float kv4_scale(float high, float low) {
  const float d = (high >= -low ? high : low) * -0.125f;
  uint32_t b = __float_as_uint(d);
  b = (b + 0xFFFFu + ((b >> 17) & 1u)) & ~0x1FFFFu;  // 7 significant bits, ties to even
  const float r = __uint_as_float(b);
  return fabsf(r) < kKv4Smallest ? 0.f : r;
}

// Eight codes (a word of the cache) times their scale, as four fp16 pairs
// (channels i and i + 4). Setting 0x5400 under a nibble at bits 4..7 of a half
// makes the number 64 + (n + 8); (72 + n) * d - 72 * d is one fused
// multiply-add whose two products and result are exact.
__device__ __forceinline__ void unpack8(uint32_t w, __half2 d, __half2 d72, __half2 (&out)[4]) {
  const uint32_t x[4] = {w << 4, w, w >> 4, w >> 8};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h;
    asm("lop3.b32 %0, %1, 0x00F000F0, 0x54005400, 0xEA;" : "=r"(h) : "r"(x[i]));  // (x & mask) | magic
    out[i] = __hfma2(reinterpret_cast<__half2 &>(h), d, d72);
  }
}
__device__ __forceinline__ __half2 minus72(__half2 d) { return __hmul2(d, __float2half2_rn(-72.f)); }

// Eight consecutive values of a row in any of the three types, as fp32. VEC: the
// address is a multiple of the 8 values' size (16 or 32 bytes).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (VEC && sizeof(T) == 4) {
    const float4 a = __ldg((const float4 *)p), b = __ldg((const float4 *)p + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (VEC) {
    const uint4 a = __ldg((const uint4 *)p);
    const T *h = (const T *)&a;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)h[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
  }
}

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    ((float4 *)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    ((float4 *)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    __align__(16) T h[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = from_float<T>(x[i]);
    *(uint4 *)p = *(const uint4 *)h;
  }
}

}  // namespace vg
