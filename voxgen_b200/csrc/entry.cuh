// What C entry points share: checks of their arguments, launches, and the choice of a
// kernel's template by type and head size.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/voxgen_cuda.h"

namespace vg {

constexpr uint64_t kMaxGrid = 0x7FFFFFFFu;

inline bool aligned(const void *p, size_t a) { return (uintptr_t)p % a == 0; }

inline int launched() {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? VG_OK : e == cudaErrorMemoryAllocation ? VG_ENOMEM : VG_ECUDA;
}

inline size_t type_size(int dtype) {
  return dtype == VG_DTYPE_F32 ? 4 : dtype == VG_DTYPE_F16 || dtype == VG_DTYPE_BF16 ? 2 : 0;
}

template <typename F>
int by_type(int dtype, F &&f) {
  switch (dtype) {
    case VG_DTYPE_F32: return f(float{});
    case VG_DTYPE_F16: return f(__half{});
    case VG_DTYPE_BF16: return f(__nv_bfloat16{});
  }
  return VG_EUNSUPPORTED;
}

template <int D>
struct Dim {
  static constexpr int value = D;
};
template <typename F>
int by_dim(uint32_t head_dim, F &&f) {
  return head_dim == 64 ? f(Dim<64>{}) : f(Dim<128>{});
}

// Lets fn use up to `bytes` of dynamic shared memory on the current device. `done`
// belongs to fn: the devices (up to 64) on which that has been set. `registers`: the
// fewest registers of a thread that fn may have been compiled to; the tile kernel's
// warpgroups trade theirs, and if they took more in all than the launch brings, the
// takers would wait for good.
inline int allow_smem(const void *fn, size_t bytes, std::atomic<uint64_t> &done, int registers = 0) {
  if (bytes <= 48 * 1024) return VG_OK;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return VG_ECUDA;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && done.load(std::memory_order_acquire) & bit) return VG_OK;
  cudaFuncAttributes a;
  if (cudaFuncGetAttributes(&a, fn) != cudaSuccess) return VG_ECUDA;
  if (a.numRegs < registers) return VG_EUNSUPPORTED;
  if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) return VG_ECUDA;
  done.fetch_or(bit, std::memory_order_release);
  return VG_OK;
}

}  // namespace vg
