// Attention for blocks of a few rows: one CTA takes 64 rows (or 16) of one document and one
// key head, runs over the keys that any of its rows sees, and keeps the running maximum and
// sum of each row's softmax in fp32 registers. Products are mma.sync m16n8k16 with fp32 sums.
//
// A row is a query token together with one of the `group` query heads that share the key
// head, so a key tile is read once for all of them. What a row sees is always one interval of
// keys: its document's keys in use, cut at its own position where the mask is causal, but
// never below the prefix. So a mask is two comparisons, made only in tiles that some row's
// interval ends in, and tiles that no row sees are not loaded.
//
// Scores are kept as powers of two (x = score * log2 e), capped and biased in fp32. The weights 2^(x - max) are rounded to the tensors' type for the second product, as the
// matrix instructions take no wider operand; their sum is taken before that rounding.
//
// Keys and values beyond a document's keys in use are filled with zeros as they are staged,
// whatever the memory holds, so a NaN there cannot reach a sum through a weight of zero.
//
// Two forms: 64 rows, each warp 16 of them with all keys of a tile; or 16 rows, for a few
// query tokens, where each warp takes 16 of a tile's 64 keys and the four partial results are
// joined at the end. Either may share its keys out over a cluster of CTAs, whose partial
// results are joined through distributed shared memory, so no workspace is needed and the
// order of the sums is fixed.
#include "token_common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ah {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 128;
constexpr int kStages = 3;

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// 16 bytes into shared memory, or zeros.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DP, bool FEW>
struct Layout {
  static constexpr int kRow = DP * 2 + 16;  // bytes of a staged row: 16 more than it holds, for the banks
  static constexpr int kTile = kMmaKeys * kRow;
  static constexpr int kStage = 2 * kTile + kAttnMaxAxes * kMmaKeys * 4;
  static constexpr int kQ = (FEW ? kMmaRowsFew : kMmaRowsWide) * kRow;
  static constexpr int kBytes = kQ + kStages * kStage;
  // partial results, in the place of the stages
  static constexpr int kPartRow = DP + 4;  // floats
  static_assert(kStages * kStage >= 4 * 16 * kPartRow * 4 + 4 * 16 * 2 * 4, "partial results do not fit");
};

template <typename T, int DP, bool FEW>
__global__ void __launch_bounds__(kThreads) attn_mma_kernel(const __grid_constant__ AttnArgs a) {
  using L = Layout<DP, FEW>;
  constexpr int kRows = FEW ? kMmaRowsFew : kMmaRowsWide;
  constexpr int kWarpKeys = FEW ? kMmaKeys / 4 : kMmaKeys;  // of a tile
  constexpr int kNT = kWarpKeys / 8;
  constexpr int kKD = DP / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sStage = smem + L::kQ;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const AttnItem item = a.items[blockIdx.x / ranks];
  const AttnDoc doc = a.docs[item.doc];
  const int kvh = blockIdx.y;
  int klen = doc.nk;
  if (a.k_lens) klen = min(max(a.k_lens[item.doc], 0), doc.nk);
  const int rows = min(kRows, doc.nq * a.group - item.row0);
  const int prefix = min(doc.prefix, klen);
  // Row r sees the document's keys [0, hi(r)).
  auto hi_of = [&](int r) {
    if (!a.causal) return klen;
    const int tok = (item.row0 + r) / a.group;
    return min(klen, max(prefix, tok + klen - doc.nq + 1));
  };
  const int hi_last = max(hi_of(rows - 1), 0);   // the largest
  const int hi_first = hi_of(0);                 // the smallest
  const int tiles = (hi_last + kMmaKeys - 1) / kMmaKeys;
  const int tile0 = static_cast<int>(static_cast<long long>(tiles) * rank / ranks);
  const int tile1 = static_cast<int>(static_cast<long long>(tiles) * (rank + 1) / ranks);

  const T* kbase = static_cast<const T*>(a.k) + doc.k0 * a.k_tok + kvh * a.k_head;
  const T* vbase = static_cast<const T*>(a.v) + doc.k0 * a.v_tok + kvh * a.v_head;
  const int chunks = a.head_dim / 8;

  auto load_tile = [&](int tile) {
    uint8_t* st = sStage + (tile - tile0) % kStages * L::kStage;
    const uint32_t sk = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    constexpr int kC = DP / 8;
    for (int i = threadIdx.x; i < kMmaKeys * kC; i += kThreads) {
      const int r = i / kC, c = i % kC;
      const int key = tile * kMmaKeys + r;
      const bool take = key < klen && c < chunks;
      const long long kk = take ? key : 0;
      const int cc = take ? c * 8 : 0;
      cp_async16(sk + r * L::kRow + c * 16, kbase + kk * a.k_tok + cc, take);
      cp_async16(sk + L::kTile + r * L::kRow + c * 16, vbase + kk * a.v_tok + cc, take);
    }
    if (a.axes) {
      float* sp = reinterpret_cast<float*>(st + 2 * L::kTile);
      for (int i = threadIdx.x; i < a.axes * kMmaKeys; i += kThreads) {
        const int ax = i / kMmaKeys, key = tile * kMmaKeys + i % kMmaKeys;
        sp[i] = key < klen ? a.k_pos[ax * a.k_total + doc.k0 + key] : 0.f;
      }
    }
  };

  // Queries of the block, rows past its end as zeros.
  {
    const uint32_t sq = static_cast<uint32_t>(__cvta_generic_to_shared(sQ));
    constexpr int kC = DP / 8;
    for (int i = threadIdx.x; i < kRows * kC; i += kThreads) {
      const int r = i / kC, c = i % kC;
      const bool take = r < rows && c < chunks;
      const int row = item.row0 + (take ? r : 0);
      const T* src = static_cast<const T*>(a.q) + (static_cast<long long>(doc.q0) + row / a.group) * a.q_tok +
                     (kvh * a.group + row % a.group) * a.q_head + (take ? c * 8 : 0);
      cp_async16(sq + r * L::kRow + c * 16, src, take);
    }
  }
#pragma unroll
  for (int p = 0; p < kStages - 1; ++p) {
    if (tile0 + p < tile1) load_tile(tile0 + p);
    cp_async_commit();
  }

  // This thread's two rows.
  const int wrow = FEW ? 0 : warp * 16;
  int hi[2];
  float slope[2][kAttnMaxAxes], qpos[2][kAttnMaxAxes];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = min(wrow + g + 8 * e, rows - 1);
    hi[e] = hi_of(r);
    const int row = item.row0 + r;
    const int h = kvh * a.group + row % a.group;
#pragma unroll
    for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
      slope[e][ax] = ax < a.axes ? a.slopes[h * a.axes + ax] : 0.f;
      qpos[e][ax] = ax < a.axes ? a.q_pos[ax * a.q_total + doc.q0 + row / a.group] : 0.f;
    }
  }

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  uint32_t qf[kKD][4];
  for (int tile = tile0; tile < tile1; ++tile) {
    cp_async_wait<kStages - 2>();
    __syncthreads();
    if (tile + kStages - 1 < tile1) load_tile(tile + kStages - 1);
    cp_async_commit();
    if (tile == tile0) {
      const uint32_t sq = static_cast<uint32_t>(__cvta_generic_to_shared(sQ));
#pragma unroll
      for (int kd = 0; kd < kKD; ++kd)
        ldmatrix4(qf[kd], sq + (wrow + (lane & 15)) * L::kRow + kd * 32 + (lane >> 4) * 16);
    }
    const uint8_t* st = sStage + (tile - tile0) % kStages * L::kStage;
    const uint32_t sk = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    const uint32_t sv = sk + L::kTile;
    const float* sp = reinterpret_cast<const float*>(st + 2 * L::kTile);
    const int wk0 = FEW ? warp * kWarpKeys : 0;  // this warp's first key within the tile
    const int key0 = tile * kMmaKeys + wk0;

    float s[kNT][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int kd = 0; kd < kKD; ++kd)
#pragma unroll
      for (int n = 0; n < kNT; n += 2) {
        uint32_t b[4];  // keys n*8 .. +7 (b0, b1) and +8 .. +15 (b2, b3)
        const int kr = wk0 + n * 8 + (lane & 7) + (lane >> 4) * 8;
        ldmatrix4(b, sk + kr * L::kRow + kd * 32 + ((lane >> 3) & 1) * 16);
        mma<T>(s[n], qf[kd], b[0], b[1]);
        mma<T>(s[n + 1], qf[kd], b[2], b[3]);
      }
    if (a.cap_log2 > 0.f) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = attn_capped(s[n][e], a);
    } else {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] *= a.score_mul;
    }
    if (a.axes) {
#pragma unroll
      for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
        if (ax >= a.axes) break;
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const float2 kp = *reinterpret_cast<const float2*>(sp + ax * kMmaKeys + wk0 + n * 8 + t4 * 2);
          s[n][0] -= slope[0][ax] * fabsf(qpos[0][ax] - kp.x);
          s[n][1] -= slope[0][ax] * fabsf(qpos[0][ax] - kp.y);
          s[n][2] -= slope[1][ax] * fabsf(qpos[1][ax] - kp.x);
          s[n][3] -= slope[1][ax] * fabsf(qpos[1][ax] - kp.y);
        }
      }
    }
    if (key0 + kWarpKeys > hi_first) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (key0 + n * 8 + t4 * 2 + (e & 1) >= hi[e >> 1]) s[n][e] = -INFINITY;
    }
    uint32_t pf[kNT][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top = m[e];
#pragma unroll
      for (int n = 0; n < kNT; ++n) top = fmaxf(top, fmaxf(s[n][2 * e], s[n][2 * e + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float base = top == -INFINITY ? 0.f : top;  // a row that has seen nothing yet
      const float shrink = exp2_fast(m[e] - base);
      m[e] = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float p0 = exp2_fast(s[n][2 * e] - base), p1 = exp2_fast(s[n][2 * e + 1] - base);
        sum += p0 + p1;
        pf[n][e] = pack2<T>(p0, p1);
      }
      l[e] = l[e] * shrink + sum;
#pragma unroll
      for (int i = 0; i < DP / 8; ++i) {
        o[i][2 * e] *= shrink;
        o[i][2 * e + 1] *= shrink;
      }
    }
#pragma unroll
    for (int kk = 0; kk < kNT / 2; ++kk) {
      const uint32_t pa[4] = {pf[2 * kk][0], pf[2 * kk][1], pf[2 * kk + 1][0], pf[2 * kk + 1][1]};
#pragma unroll
      for (int i = 0; i < DP / 8; i += 2) {
        uint32_t b[4];
        const int kr = wk0 + kk * 16 + (lane & 15);
        ldmatrix4_trans(b, sv + kr * L::kRow + i * 16 + (lane >> 4) * 16);
        mma<T>(o[i], pa, b[0], b[1]);
        mma<T>(o[i + 1], pa, b[2], b[3]);
      }
    }
  }
  cp_async_wait<0>();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
    l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
  }

  auto store8 = [&](int r, int c, const float (&f)[8]) {
    const int row = item.row0 + r;
    T* dst = static_cast<T*>(a.out) + (static_cast<long long>(doc.q0) + row / a.group) * a.o_tok +
             (kvh * a.group + row % a.group) * a.o_head + c * 8;
    uint4 u;
    u.x = pack2<T>(f[0], f[1]);
    u.y = pack2<T>(f[2], f[3]);
    u.z = pack2<T>(f[4], f[5]);
    u.w = pack2<T>(f[6], f[7]);
    *reinterpret_cast<uint4*>(dst) = u;
  };

  // Partial results of the warps, 16 rows each, in the place of the stages.
  __syncthreads();
  float* part = reinterpret_cast<float*>(sStage);
  float2* ml = reinterpret_cast<float2*>(part + 4 * 16 * L::kPartRow);
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = warp * 16 + g + 8 * e;
    if (t4 == 0) ml[r] = make_float2(m[e], l[e]);
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
      *reinterpret_cast<float2*>(part + r * L::kPartRow + i * 8 + t4 * 2) = make_float2(o[i][2 * e], o[i][2 * e + 1]);
  }
  __syncthreads();
  if constexpr (FEW) {  // the four warps hold the same rows: join them into the first 16
    constexpr int kPer = (16 * (DP / 8) + kThreads - 1) / kThreads;
    float f[kPer][8];
    float2 mj[kPer];
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = threadIdx.x + p * kThreads;
      const int r = i / (DP / 8), c = i % (DP / 8);
      if (i >= 16 * (DP / 8)) continue;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) top = fmaxf(top, ml[w * 16 + r].x);
      mj[p] = make_float2(top, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[p][j] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 v = ml[w * 16 + r];
        const float k = v.x == -INFINITY ? 0.f : exp2_fast(v.x - top);
        mj[p].y += k * v.y;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[p][j] += k * part[(w * 16 + r) * L::kPartRow + c * 8 + j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int i = threadIdx.x + p * kThreads;
      const int r = i / (DP / 8), c = i % (DP / 8);
      if (i >= 16 * (DP / 8)) continue;
      if (c == 0) ml[r] = mj[p];
#pragma unroll
      for (int j = 0; j < 8; ++j) part[r * L::kPartRow + c * 8 + j] = f[p][j];
    }
  }
  if (ranks > 1)
    cluster.sync();
  else
    __syncthreads();
  // Each CTA of the cluster joins and writes its share of the (row, 8 elements) pieces.
  for (int i = threadIdx.x * ranks + rank; i < rows * chunks; i += kThreads * ranks) {
    const int r = i / chunks, c = i - r * chunks;
    float f[8], sum = 0.f, top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    for (int w = 0; w < ranks; ++w) top = fmaxf(top, cluster.map_shared_rank(ml, w)[r].x);
    for (int w = 0; w < ranks; ++w) {
      const float2 v = cluster.map_shared_rank(ml, w)[r];
      const float k = v.x == -INFINITY ? 0.f : exp2_fast(v.x - top);
      const float4* src =
          reinterpret_cast<const float4*>(cluster.map_shared_rank(part, w) + r * L::kPartRow + c * 8);
      const float4 x = src[0], y = src[1];
      sum += k * v.y;
      f[0] += k * x.x, f[1] += k * x.y, f[2] += k * x.z, f[3] += k * x.w;
      f[4] += k * y.x, f[5] += k * y.y, f[6] += k * y.z, f[7] += k * y.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zeros
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= inv;
    store8(r, c, f);
  }
  if (ranks > 1) cluster.sync();  // no CTA leaves while another reads its shared memory
}

template <typename T, int DP, bool FEW>
cudaError_t launch(const AttnArgs& a, int cluster, cudaStream_t s) {
  auto fn = attn_mma_kernel<T, DP, FEW>;
  static AttrOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(fn), Layout<DP, FEW>::kBytes, true);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.num_items) * cluster, a.kv_heads);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<DP, FEW>::kBytes;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, a);
}

template <typename T, bool FEW>
cudaError_t by_dim(const AttnArgs& a, int cluster, cudaStream_t s) {
  if (a.head_dim <= 32) return launch<T, 32, FEW>(a, cluster, s);
  if (a.head_dim <= 64) return launch<T, 64, FEW>(a, cluster, s);
  if (a.head_dim <= 96) return launch<T, 96, FEW>(a, cluster, s);
  return launch<T, 128, FEW>(a, cluster, s);
}

}  // namespace

cudaError_t attn_mma_launch(const AttnArgs& a, int dtype, bool few_rows, int cluster, cudaStream_t s) {
  if (dtype == kTokenBf16)
    return few_rows ? by_dim<__nv_bfloat16, true>(a, cluster, s) : by_dim<__nv_bfloat16, false>(a, cluster, s);
  return few_rows ? by_dim<__half, true>(a, cluster, s) : by_dim<__half, false>(a, cluster, s);
}

}  // namespace ah
