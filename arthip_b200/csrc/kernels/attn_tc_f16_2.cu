// attn_tc_kernel for f16, heads of up to 128 elements.
#include "attn_tc_kernel.cuh"

namespace ah {
namespace attn_tc {

cudaError_t launch_f16_2(const AttnTcArgs& args, cudaStream_t s) {
  return launch_variant<__half, 2>(args, s);
}

}  // namespace attn_tc
}  // namespace ah
