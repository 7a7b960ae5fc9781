// Host side of the tcgen05 attention kernel (attn_tc_kernel.cuh): tensor maps of q, k and v.
// They are encoded for each call, as they hold its addresses, and travel as a kernel
// parameter, so a captured launch keeps its own.
#include "attn_tc_kernel.cuh"

#include <atomic>

#include <cuda.h>

namespace ah {

namespace {

// Failure-path test hook (ah_test_set_attn_fault_hook): 0 = off.
std::atomic<int> g_test_wait_ms{0};
std::atomic<int> g_test_stall_load{-1};

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

bool encode(EncodeTiledFn fn, CUtensorMap* map, int dtype, const void* p, int dim, long long tokens, long long tok,
            int heads, long long head, std::string* err) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(tokens),
                              static_cast<cuuint64_t>(heads)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(tok) * 2, static_cast<cuuint64_t>(head) * 2};
  const cuuint32_t box[3] = {64, 128, 1}, elem[3] = {1, 1, 1};
  const CUresult r = fn(map, dtype == kTokenBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        3, const_cast<void*>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return true;
  if (err) *err = "cuTensorMapEncodeTiled failed (code " + std::to_string(static_cast<int>(r)) + ")";
  return false;
}

}  // namespace

void attn_tc_set_test_hook(int wait_limit_ms, int stall_load) {
  const bool on = wait_limit_ms > 0 && wait_limit_ms <= 4000 && stall_load >= 0;
  g_test_stall_load.store(on ? stall_load : -1, std::memory_order_relaxed);
  g_test_wait_ms.store(on ? wait_limit_ms : 0, std::memory_order_relaxed);
}

cudaError_t attn_tc_launch(const AttnArgs& a, int dtype, cudaStream_t s, std::string* err) {
  const EncodeTiledFn fn = encode_fn();
  if (!fn) {
    if (err) *err = "cuTensorMapEncodeTiled is unavailable from the CUDA driver";
    return cudaErrorNotSupported;
  }
  AttnTcArgs args;
  args.a = a;
  const int hook_ms = g_test_wait_ms.load(std::memory_order_relaxed);
  args.wait_limit_ns = hook_ms > 0 ? static_cast<unsigned long long>(hook_ms) * 1000000ull : ptx::kWaitLimitNs;
  args.stall_load = hook_ms > 0 ? g_test_stall_load.load(std::memory_order_relaxed) : -1;
  if (!encode(fn, &args.q, dtype, a.q, a.head_dim, a.q_total, a.q_tok, a.q_heads, a.q_head, err) ||
      !encode(fn, &args.k, dtype, a.k, a.head_dim, a.k_total, a.k_tok, a.kv_heads, a.k_head, err) ||
      !encode(fn, &args.v, dtype, a.v, a.head_dim, a.k_total, a.v_tok, a.kv_heads, a.v_head, err))
    return cudaErrorInvalidValue;
  const bool two = a.head_dim > 64;
  if (dtype == kTokenBf16) return two ? attn_tc::launch_bf16_2(args, s) : attn_tc::launch_bf16_1(args, s);
  return two ? attn_tc::launch_f16_2(args, s) : attn_tc::launch_f16_1(args, s);
}

}  // namespace ah
