// Choice of the norm kernel (token_norm_kernel.cuh).
#include "token_norm_kernel.cuh"

namespace ah {

cudaError_t norm_launch(const NormArgs& a, int dtype, int num_sms, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  // The widest vectors that divide the rows, and that every pointer and stride is aligned to.
  // (Vectors of 4 bytes are no faster than the staged kernel anywhere: 90 channels 205 us against
  // 148, 510 channels 385 against 149, for 64 Mi elements.)
  uintptr_t bits = static_cast<uintptr_t>(a.C) * 2;
  const void* ptrs[] = {a.x, a.y, a.gate, a.mscale, a.mshift, a.out, a.norm};
  const long long strides[] = {a.xs, a.ys, a.gs, a.ms, a.ms, a.os, a.ns};
  for (int i = 0; i < 7; ++i)
    if (ptrs[i]) bits |= reinterpret_cast<uintptr_t>(ptrs[i]) | static_cast<uintptr_t>(strides[i] * 2);
  const bool bf16 = dtype == kTokenBf16;
  for (int vec = 8; vec >= 4; vec /= 2)
    if (bits % (vec * 2) == 0)
      return bf16 ? token_norm::vectors_bf16(a, vec, num_sms, s) : token_norm::vectors_f16(a, vec, num_sms, s);
  return bf16 ? token_norm::elements_bf16(a, num_sms, s) : token_norm::elements_f16(a, num_sms, s);
}

}  // namespace ah
