// What the token kernels share: conversions of the two element types, the exponential and the capped
// score of attention, asynchronous copies of vectors and of rows of any alignment, and launch
// attributes.
#pragma once

#include "ptx.cuh"
#include "tokens.h"

#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace ah {

// fp16 and bf16, one at a time and in pairs.
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void from_f(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f2(float a, float b, __half2* o) { *o = __floats2half2_rn(a, b); }
__device__ __forceinline__ void from_f2(float a, float b, __nv_bfloat162* o) { *o = __floats2bfloat162_rn(a, b); }

template <typename T>
struct Two;
template <>
struct Two<__half> {
  using type = __half2;
};
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// Two values rounded to T, the first in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typename Two<T>::type v;
  from_f2(lo, hi, &v);
  return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// How scores are capped, cap * tanh(s / cap), in powers of two:
//   kCapExp     cap (1 - 2 / (1 + exp(2 s / cap))), good to a few units of 2^-24 cap
//   kCapSeries  for a cap beyond 256, where that is no longer small beside the score: small
//               arguments take the odd series of tanh instead
enum CapForm : int { kCapNone = 0, kCapExp = 1, kCapSeries = 2 };
constexpr float kSeriesCap = 256.f;

inline CapForm cap_form(const AttnArgs& a) {
  return a.cap_log2 > kSeriesCap * 1.44269504f ? kCapSeries : (a.cap_log2 > 0.f ? kCapExp : kCapNone);
}

__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Of two scores.
template <int FORM>
__device__ __forceinline__ uint64_t attn_capped2(uint64_t s, const AttnArgs& a) {
  auto both = [](float v) { return ptx::pack_f2(v, v); };
  const float2 e = ptx::unpack_f2(ptx::mul_f2(s, both(a.cap_exp)));
  const float2 d = ptx::unpack_f2(ptx::add_f2(ptx::pack_f2(exp2_fast(e.x), exp2_fast(e.y)), both(1.f)));
  const uint64_t x =
      ptx::fma_f2(ptx::pack_f2(rcp_fast(d.x), rcp_fast(d.y)), both(-2.f * a.cap_log2), both(a.cap_log2));
  if constexpr (FORM == kCapSeries) {
    // tanh u = u - u^3/3 + 2u^5/15 - 17u^7/315 + 62u^9/2835; the next term is below 2^-24 u
    const float2 sv = ptx::unpack_f2(s), xv = ptx::unpack_f2(x);
    auto one = [&](float v, float big) {
      const float u = v * a.cap_arg, z = u * u;
      const float t =
          a.cap_log2 * u * (1.f + z * (-1.f / 3 + z * (2.f / 15 + z * (-17.f / 315 + z * (62.f / 2835)))));
      return fabsf(u) < 0.3f ? t : big;
    };
    return ptx::pack_f2(one(sv.x, xv.x), one(sv.y, xv.y));
  }
  return x;
}

// Asynchronous copies of a vector into shared memory, and their groups.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Rows of 2-byte elements between global memory and shared memory, by a group of GROUP threads,
// in 16-byte pieces whatever their alignment; the elements before the first and behind the last
// 16-byte boundary go one by one.
// Elements [0, n) of `src` to where `dst` + (src % 16 bytes) starts. Waits for nothing.
template <typename T, int GROUP>
__device__ __forceinline__ void copy_in(uint8_t* dst, const T* src, int n, int t) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(src);
  const int head = min(n, static_cast<int>((16 - at % 16) % 16 / 2)), body = (n - head) / 8;
  T* d = reinterpret_cast<T*>(dst + at % 16);
  if (t < head) d[t] = src[t];
  for (int i = t; i < body; i += GROUP)
    copy_async<16>(d + head + 8 * i, src + head + 8 * i);
  const int tail = head + body * 8 + t;
  if (tail < n) d[tail] = src[tail];
}

// The way back: elements [0, n) from `src` + (dst % 16 bytes).
template <typename T, int GROUP>
__device__ __forceinline__ void copy_out(T* dst, const uint8_t* src, int n, int t) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(dst);
  const int head = min(n, static_cast<int>((16 - at % 16) % 16 / 2)), body = (n - head) / 8;
  const T* from = reinterpret_cast<const T*>(src + at % 16);
  if (t < head) dst[t] = from[t];
  for (int i = t; i < body; i += GROUP)
    *reinterpret_cast<uint4*>(dst + head + 8 * i) = *reinterpret_cast<const uint4*>(from + head + 8 * i);
  const int tail = head + body * 8 + t;
  if (tail < n) dst[tail] = from[tail];
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
