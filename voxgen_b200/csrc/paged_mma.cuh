// MMA operands of a paged cache's types, fp16 and bf16.
#pragma once
#include "kv4_rows_attention.cuh"

namespace vg {

__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __half) { mma_f16(c, a, b); }
__device__ __forceinline__ void mma_16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2], __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// Two values rounded to a pair of type C, and what is left of them.
__device__ __forceinline__ uint32_t take_pair(float &x, float &y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  x -= f.x, y -= f.y;
  return half2_bits(h);
}
__device__ __forceinline__ uint32_t take_pair(float &x, float &y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  const float2 f = __bfloat1622float2(h);
  x -= f.x, y -= f.y;
  return *reinterpret_cast<const uint32_t *>(&h);
}

}  // namespace vg
