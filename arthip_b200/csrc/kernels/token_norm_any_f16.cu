// Norms of f16 rows of any width, stride and alignment.
#include "token_norm_kernel.cuh"

namespace ah {
namespace token_norm {

cudaError_t elements_f16(const NormArgs& a, int num_sms, cudaStream_t s) { return by_elements<__half>(a, num_sms, s); }

}  // namespace token_norm
}  // namespace ah
