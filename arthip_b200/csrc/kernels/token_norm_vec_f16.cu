// Norms of f16 rows of vectors.
#include "token_norm_kernel.cuh"

namespace ah {
namespace token_norm {

cudaError_t vectors_f16(const NormArgs& a, int vec, int num_sms, cudaStream_t s) {
  return vec == 8 ? by_width<__half, 8>(a, num_sms, s) : by_width<__half, 4>(a, num_sms, s);
}

}  // namespace token_norm
}  // namespace ah
