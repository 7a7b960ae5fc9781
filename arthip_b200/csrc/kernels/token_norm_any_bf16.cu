// Norms of bf16 rows of any width, stride and alignment.
#include "token_norm_kernel.cuh"

namespace ah {
namespace token_norm {

cudaError_t elements_bf16(const NormArgs& a, int num_sms, cudaStream_t s) { return by_elements<__nv_bfloat16>(a, num_sms, s); }

}  // namespace token_norm
}  // namespace ah
