// What the token kernels share: the capped score of attention, and launch attributes.
#pragma once

#include "tokens.h"

#include <atomic>

#include <cuda_runtime.h>

namespace ah {

constexpr float kSeriesCap = 256.f;

// cap * tanh(s / cap) in powers of two: cap (1 - 2 / (1 + exp(2 s / cap))), good to a few units
// of 2^-24 cap. Beyond a cap of 256, where that is no longer small beside the score, small
// arguments take the odd series of tanh instead.
__device__ __forceinline__ float attn_capped(float s, const AttnArgs& a) {
  const float u = s * a.cap_arg;
  if (a.cap_log2 > kSeriesCap * 1.44269504f && fabsf(u) < 0.3f) {
    // tanh u = u - u^3/3 + 2u^5/15 - 17u^7/315 + 62u^9/2835; the next term is below 2^-24 u
    const float z = u * u;
    return a.cap_log2 * u * (1.f + z * (-1.f / 3 + z * (2.f / 15 + z * (-17.f / 315 + z * (62.f / 2835)))));
  }
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(u * 2.88539008f));
  return a.cap_log2 - __fdividef(2.f * a.cap_log2, 1.f + e);
}

// A kernel's function attributes, set once per device.
struct AttrOnce {
  std::atomic<uint64_t> done{0};
  cudaError_t set(const void* fn, int smem_bytes, bool wide_clusters = false) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes);
    if (e == cudaSuccess && wide_clusters)
      e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
    return e;
  }
};

}  // namespace ah
