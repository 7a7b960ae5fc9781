// Host-side launch interface of the token operators (sm_100a): norms around a block with
// its gate and residual scale, rotary positions over several axes, and attention. Tensors
// are fp16 or bf16 with their rows (tokens) at a caller-given stride in elements; the C ABI
// (tokens_capi.cc) has checked every argument before it calls these.
#pragma once

#include <cstdint>
#include <string>

#include <cuda_runtime.h>

namespace ah {

enum TokenType : int { kTokenF16 = 0, kTokenBf16 = 1 };

// ---------------------------------------------------------------------------
// token_norm.cu
// ---------------------------------------------------------------------------
enum NormKind : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum GateAct : int { kGateLinear = 0, kGateSigmoid = 1, kGateTanh = 2, kGateSilu = 3 };

constexpr int kNormMaxChannels = 8192;

struct NormArgs {
  const void* x = nullptr;      // residual stream
  const void* y = nullptr;      // block output, or null
  const void* gate = nullptr;   // [rows / rows_per_gate][C], or null
  const void* mscale = nullptr; // [rows / rows_per_mod][C], or null
  const void* mshift = nullptr;
  void* out = nullptr;          // x + scaled block, or null
  void* norm = nullptr;         // pre-norm of it, or null
  long long xs = 0, ys = 0, gs = 0, ms = 0, os = 0, ns = 0;  // row strides, elements
  long long rows = 0, rows_per_gate = 1, rows_per_mod = 1;
  const float* a = nullptr;   // post weight * layer scale * residual scale, or null (= 1)
  const float* b = nullptr;   // post bias times the same, or null
  const float* w = nullptr;   // pre weight / bias, or null
  const float* wb = nullptr;
  float post_eps = 0.f, pre_eps = 0.f;
  int C = 0, post = 0, pre = 0, act = 0;
};
cudaError_t norm_launch(const NormArgs& a, int dtype, int num_sms, cudaStream_t s);

// ---------------------------------------------------------------------------
// token_rope.cu
// ---------------------------------------------------------------------------
enum RopeLayout : int { kRopeHalves = 0, kRopePairs = 1, kRopeShared = 2 };

struct RopePair {
  double turns;  // signed turns per unit of position: frequency / 2 pi
  int axis;
  int e0, e1;    // the pair's elements within a head
  int pad;
};

struct RopeTable {
  RopePair* pairs = nullptr;  // device, npairs
  int npairs = 0;
  int rot = 0;                // rotated elements of a head (2 * npairs)
  int head_dim = 0;
  int axes = 0;
  int layout = 0;
  int halves8 = 0;            // every run of 8 pairs is two runs of 8 elements, each at a multiple of 8
};

struct RopeArgs {
  const float* pos = nullptr;  // [axes][tokens]
  const void* in[2] = {};      // q, k
  void* out[2] = {};
  long long in_tok[2] = {}, in_head[2] = {}, out_tok[2] = {}, out_head[2] = {};
  int heads[2] = {};
  long long tokens = 0;
};
cudaError_t rope_launch(const RopeTable& t, const RopeArgs& a, int dtype, int num_sms, cudaStream_t s);

// ---------------------------------------------------------------------------
// Attention: attn_mma.cu
// ---------------------------------------------------------------------------
constexpr int kAttnMaxHeadDim = 128;
constexpr int kAttnMaxAxes = 3;

// A document: its query and key ranges and the keys that every query of it may see.
struct AttnDoc {
  int q0, nq, k0, nk, prefix;
};
// A block of rows of one document, from row row0. A row is a query token and one of the query
// heads that share a key head: row = token * group + head in group.
struct AttnItem {
  int doc, row0;
};

struct AttnArgs {
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  void* out = nullptr;
  long long q_tok = 0, q_head = 0, k_tok = 0, k_head = 0, v_tok = 0, v_head = 0, o_tok = 0, o_head = 0;
  const float* q_pos = nullptr;  // [axes][total queries]
  const float* k_pos = nullptr;  // [axes][total keys]
  long long q_total = 0, k_total = 0;
  const int* k_lens = nullptr;  // keys in use of each document, or null
  const AttnDoc* docs = nullptr;
  const AttnItem* items = nullptr;
  const float* slopes = nullptr;  // [q heads][axes], in the scores' units
  uint32_t* status = nullptr;
  int num_items = 0, num_sms = 148;
  int heads_per_block = 1;  // set by the launch that uses it
  int q_heads = 0, kv_heads = 0, group = 1, head_dim = 0, axes = 0, causal = 0;
  // Scores: q.k less the bias, and times score_mul in powers of two; or with a cap, in powers of
  // two before the bias, cap_log2 * tanh(cap_arg * (q.k)), with cap_exp = 2 log2(e) cap_arg.
  float score_mul = 0.f, cap_log2 = 0.f, cap_arg = 0.f, cap_exp = 0.f;
};

// Rows per block of the two forms of the mma.sync kernel.
constexpr int kMmaRowsWide = 64;  // four warps of 16 rows
constexpr int kMmaRowsFew = 16;   // 16 rows, the keys shared out over the warps
constexpr int kMmaKeys = 64;      // keys per tile
// `tiles`: the most key tiles of any block.
cudaError_t attn_mma_launch(const AttnArgs& a, int dtype, bool few_rows, int cluster, int tiles, cudaStream_t s);

// attn_tc.cu: tcgen05 form. Its items are not rows but query tokens: two tiles of 128, one
// after the other of one query head, or, for an even group, of the same tokens for two heads.
constexpr int kTcRows = 128;
constexpr int kTcKeys = 128;
inline bool attn_tc_head_pairs(int group) { return group % 2 == 0; }
inline int attn_tc_item_tokens(int group) { return attn_tc_head_pairs(group) ? kTcRows : 2 * kTcRows; }
cudaError_t attn_tc_launch(const AttnArgs& a, int dtype, cudaStream_t s, std::string* err);
// Bounds every wait of later launches by wait_limit_ms and leaves out load `stall_load` of each CTA.
void attn_tc_set_test_hook(int wait_limit_ms, int stall_load);

}  // namespace ah
