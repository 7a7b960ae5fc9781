// attn_tc_kernel for bf16, heads of up to 64 elements.
#include "attn_tc_kernel.cuh"

namespace ah {
namespace attn_tc {

cudaError_t launch_bf16_1(const AttnTcArgs& args, cudaStream_t s) {
  return launch_variant<__nv_bfloat16, 1>(args, s);
}

}  // namespace attn_tc
}  // namespace ah
