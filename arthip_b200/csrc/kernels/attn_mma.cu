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
// Scores are capped and biased in fp32. Their weights are rounded to the tensors' type for the
// second product, whose matrix instructions take both operands in that type (a wider form would
// want the values widened too, at twice the shared memory and half the rate); the sum of the
// weights is taken before that rounding. It adds an error of about the output's own rounding: of
// fp16 outputs, relative to 64 bits, 2.1e-4 without it and 2.4e-4 to 2.9e-4 with it, of bf16 ones
// 1.65e-3 and 2.0e-3.
//
// Keys and values beyond a document's keys in use are filled with zeros as they are staged,
// whatever the memory holds, so a NaN there cannot reach a sum through a weight of zero.
//
// Three forms: 64 rows, each warp 16 of them with all keys of a tile; or 16 rows, for a few
// query tokens, where each warp takes 16 of a tile's 64 keys and the four partial results are
// joined at the end; each of them with its keys shared out over a cluster of CTAs, whose
// partial results are joined through distributed shared memory, so that no workspace is needed
// and the order of the sums is fixed; and 64 rows with all their keys in one CTA, which takes
// some key heads one after another, the next one's loads under way, and writes its rows itself.
#include "token_common.cuh"
#include "tokens.h"

#include <algorithm>

#include <cooperative_groups.h>

namespace ah {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 128;
constexpr int kStages = 3;
constexpr float kWeightShift = 6.f;  // weights are 2^(x - max + 6): a wider range above fp16's smallest

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

enum Form : int { kFew = 0, kWideShared = 1, kWideAlone = 2 };

template <int DP, int FORM>
struct Layout {
  static constexpr bool FEW = FORM == kFew;
  static constexpr int kRow = DP * 2 + 16;  // bytes of a staged row: 16 more than it holds, for the banks
  static constexpr int kTile = kMmaKeys * kRow;
  static constexpr int kPos = 2 * kTile;  // in a stage: keys, values, key positions, queries
  static constexpr int kStageQ = kPos + kAttnMaxAxes * kMmaKeys * 4;
  static constexpr int kStage = kStageQ + (FORM == kWideAlone ? kMmaRowsWide * kRow : 0);
  static constexpr int kQ = FORM == kWideAlone ? 0 : (FEW ? kMmaRowsFew : kMmaRowsWide) * kRow;
  static constexpr int bytes(int stages) { return kQ + stages * kStage; }
  // partial results, in the place of the stages
  static constexpr int kPartRow = DP + 4;  // floats
  static_assert(kStages * kStage >= 4 * 16 * kPartRow * 4 + 4 * 16 * 2 * 4, "partial results do not fit");
};

// Heads of up to 32, whole keys in a CTA: four CTAs to an SM by their shared memory, so the
// registers are held to 128 (2040 windows of 64 tokens, 6 heads of 32, two axes: 75 us; left at 218
// registers, two CTAs, 99 us). Wider heads hold the SM to two CTAs or one by their shared memory as
// soon as they have keys for three stages, and do not gain where they have not (the same windows, 6
// heads of 64: 132 us as it is, 134 us with three CTAs of 168 registers).
template <typename T, int DP, int FORM>
__global__ void __launch_bounds__(kThreads, FORM == kWideAlone && DP == 32 ? 4 : 1)
    attn_mma_kernel(const __grid_constant__ AttnArgs a) {
  using L = Layout<DP, FORM>;
  constexpr bool FEW = L::FEW;
  constexpr int kRows = FEW ? kMmaRowsFew : kMmaRowsWide;
  constexpr int kWarpKeys = FEW ? kMmaKeys / 4 : kMmaKeys;  // of a tile
  constexpr int kNT = kWarpKeys / 8;
  constexpr int kKD = DP / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  uint8_t* sQ = smem;
  uint8_t* sStage = smem + L::kQ;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = FORM == kWideAlone ? 1 : static_cast<int>(cluster.num_blocks());
  const int rank = FORM == kWideAlone ? 0 : static_cast<int>(cluster.block_rank());

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const AttnItem item = a.items[blockIdx.x / ranks];
  const AttnDoc doc = a.docs[item.doc];
  const int kvh0 = blockIdx.y * (FORM == kWideAlone ? a.heads_per_block : 1);
  const int heads = FORM == kWideAlone ? min(a.heads_per_block, a.kv_heads - kvh0) : 1;  // one after another
  int klen = doc.nk;
  if (a.k_lens) klen = min(max(a.k_lens[item.doc], 0), doc.nk);
  const int rows = min(kRows, doc.nq * a.group - item.row0);
  const int prefix = min(doc.prefix, klen);
  // A row's token within the document, and its head within the group. (Divisions by a number
  // not known when compiling were a third of the instructions of a 64-token window.)
  auto token_of = [&](int r) { return a.group == 1 ? item.row0 + r : (item.row0 + r) / a.group; };
  auto member_of = [&](int r) { return a.group == 1 ? 0 : (item.row0 + r) % a.group; };
  // Row r sees the document's keys [0, hi(r)).
  auto hi_of = [&](int r) {
    if (!a.causal) return klen;
    const int tok = token_of(r);
    return min(klen, max(prefix, klen - (doc.nq - tok) + 1));
  };
  const int hi_last = max(hi_of(rows - 1), 0);   // the largest
  const int hi_first = hi_of(0);                 // the smallest
  const int tiles = (hi_last + kMmaKeys - 1) / kMmaKeys;
  const int tile0 = static_cast<int>(static_cast<long long>(tiles) * rank / ranks);
  const int tile1 = static_cast<int>(static_cast<long long>(tiles) * (rank + 1) / ranks);

  const int tiles_here = tile1 - tile0, steps = tiles_here * heads;
  const int chunks = a.head_dim / 8;

  // Queries of the block for one key head, rows past its end as zeros.
  auto load_queries = [&](uint8_t* to, int kvh) {
    const uint32_t sq = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    constexpr int kC = DP / 8;
    for (int i = threadIdx.x; i < kRows * kC; i += kThreads) {
      const int r = i / kC, c = i % kC;
      const bool take = r < rows && c < chunks;
      const int row = take ? r : 0;
      const T* src = static_cast<const T*>(a.q) + (static_cast<long long>(doc.q0) + token_of(row)) * a.q_tok +
                     (kvh * a.group + member_of(row)) * a.q_head + (take ? c * 8 : 0);
      cp_async16(sq + r * L::kRow + c * 16, src, take);
    }
  };
  // Step s is tile tile0 + s % tiles_here of head s / tiles_here.
  auto load_step = [&](int s) {
    const int h = FORM == kWideAlone ? s / tiles_here : 0, tile = tile0 + s - h * tiles_here;
    const T* kbase = static_cast<const T*>(a.k) + doc.k0 * a.k_tok + (kvh0 + h) * a.k_head;
    const T* vbase = static_cast<const T*>(a.v) + doc.k0 * a.v_tok + (kvh0 + h) * a.v_head;
    uint8_t* st = sStage + s % kStages * L::kStage;
    const uint32_t sk = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    constexpr int kC = DP / 8;
    if constexpr (kThreads % kC == 0) {  // a thread's pieces are a column: one pointer each to step on
      constexpr int kStep = kThreads / kC;
      const int r = threadIdx.x / kC, c = threadIdx.x % kC;
      const int left = c < chunks ? klen - tile * kMmaKeys - r : 0;
      const T* kp = kbase + (static_cast<long long>(tile) * kMmaKeys + r) * a.k_tok + c * 8;
      const T* vp = vbase + (static_cast<long long>(tile) * kMmaKeys + r) * a.v_tok + c * 8;
      const long long k_step = kStep * a.k_tok, v_step = kStep * a.v_tok;
      const uint32_t to = sk + r * L::kRow + c * 16;
#pragma unroll
      for (int j = 0; j < kMmaKeys / kStep; ++j) {
        const bool take = j * kStep < left;
        cp_async16(to + j * kStep * L::kRow, take ? kp : kbase, take);
        cp_async16(to + j * kStep * L::kRow + L::kTile, take ? vp : vbase, take);
        kp += k_step, vp += v_step;
      }
    } else {
      for (int i = threadIdx.x; i < kMmaKeys * kC; i += kThreads) {
        const int r = i / kC, c = i % kC;
        const int key = tile * kMmaKeys + r;
        const bool take = key < klen && c < chunks;
        const long long kk = take ? key : 0;
        const int cc = take ? c * 8 : 0;
        cp_async16(sk + r * L::kRow + c * 16, kbase + kk * a.k_tok + cc, take);
        cp_async16(sk + L::kTile + r * L::kRow + c * 16, vbase + kk * a.v_tok + cc, take);
      }
    }
    if (FORM == kWideAlone && tile == tile0) load_queries(st + L::kStageQ, kvh0 + h);
    if (a.axes) {
      float* sp = reinterpret_cast<float*>(st + L::kPos);
      for (int i = threadIdx.x; i < a.axes * kMmaKeys; i += kThreads) {
        const int ax = i / kMmaKeys, key = tile * kMmaKeys + i % kMmaKeys;
        sp[i] = key < klen ? -a.k_pos[ax * a.k_total + doc.k0 + key] : 0.f;
      }
    }
  };

  if constexpr (FORM != kWideAlone) load_queries(sQ, kvh0);
#pragma unroll
  for (int p = 0; p < kStages - 1; ++p) {
    if (p < steps) load_step(p);
    copies_commit();
  }

  // This thread's two rows.
  const int wrow = FEW ? 0 : warp * 16;
  int hi[2];
  float slope[2][kAttnMaxAxes], qpos[2][kAttnMaxAxes];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = min(wrow + g + 8 * e, rows - 1);
    hi[e] = hi_of(r);
#pragma unroll
    for (int ax = 0; ax < kAttnMaxAxes; ++ax)
      qpos[e][ax] = ax < a.axes ? a.q_pos[ax * a.q_total + doc.q0 + token_of(r)] : 0.f;
  }
  auto load_slopes = [&](int kvh) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int h = kvh * a.group + member_of(min(wrow + g + 8 * e, rows - 1));
#pragma unroll
      for (int ax = 0; ax < kAttnMaxAxes; ++ax) slope[e][ax] = ax < a.axes ? a.slopes[h * a.axes + ax] : 0.f;
    }
  };
  load_slopes(kvh0);

  float o[DP / 8][4], m[2], l[2];
  auto reset = [&] {
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    m[0] = m[1] = -INFINITY, l[0] = l[1] = 0.f;
  };
  reset();
  auto place = [&](int kvh, int r, int c) {  // of 8 elements of the output
    return reinterpret_cast<uint4*>(static_cast<T*>(a.out) +
                                    (static_cast<long long>(doc.q0) + token_of(r)) * a.o_tok +
                                    (kvh * a.group + member_of(r)) * a.o_head + c * 8);
  };
  auto join_lanes = [&] {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
    }
  };
  if (FORM == kWideAlone && steps == 0) {  // no row sees a key: zeros
    for (int i = threadIdx.x; i < heads * rows * chunks; i += kThreads)
      *place(kvh0 + i / (rows * chunks), i / chunks % rows, i % chunks) = make_uint4(0, 0, 0, 0);
    return;
  }

  const float mul = a.cap_log2 > 0.f ? 1.f : a.score_mul;  // from the scores' units to powers of two
  uint32_t qf[kKD][4];
  int tile = tile0;
  for (int step = 0; step < steps; ++step) {
    copies_wait<kStages - 2>();
    __syncthreads();
    if (step + kStages - 1 < steps) load_step(step + kStages - 1);
    copies_commit();
    uint8_t* st = sStage + step % kStages * L::kStage;
    if (tile == tile0) {
      const uint32_t sq =
          static_cast<uint32_t>(__cvta_generic_to_shared(FORM == kWideAlone ? st + L::kStageQ : sQ));
#pragma unroll
      for (int kd = 0; kd < kKD; ++kd)
        ldmatrix4(qf[kd], sq + (wrow + (lane & 15)) * L::kRow + kd * 32 + (lane >> 4) * 16);
    }
    const uint32_t sk = static_cast<uint32_t>(__cvta_generic_to_shared(st));
    const uint32_t sv = sk + L::kTile;
    const float* sp = reinterpret_cast<const float*>(st + L::kPos);
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
    if (a.cap_log2 > kSeriesCap * 1.44269504f) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 v = ptx::unpack_f2(attn_capped2<kCapSeries>(ptx::pack_f2(s[n][e], s[n][e + 1]), a));
          s[n][e] = v.x, s[n][e + 1] = v.y;
        }
    } else if (a.cap_log2 > 0.f) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float2 v = ptx::unpack_f2(attn_capped2<kCapExp>(ptx::pack_f2(s[n][e], s[n][e + 1]), a));
          s[n][e] = v.x, s[n][e + 1] = v.y;
        }
    }
    if (a.axes) {
#pragma unroll
      for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
        if (ax >= a.axes) break;
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          const uint64_t away = *reinterpret_cast<const uint64_t*>(sp + ax * kMmaKeys + wk0 + n * 8 + t4 * 2);  // negated
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float2 far = ptx::unpack_f2(ptx::add_f2(ptx::pack_f2(qpos[e][ax], qpos[e][ax]), away));
            const float2 z =
                ptx::unpack_f2(ptx::fma_f2(ptx::pack_f2(fabsf(far.x), fabsf(far.y)),
                                           ptx::pack_f2(-slope[e][ax], -slope[e][ax]),
                                           ptx::pack_f2(s[n][2 * e], s[n][2 * e + 1])));
            s[n][2 * e] = z.x, s[n][2 * e + 1] = z.y;
          }
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
      for (int n = 0; n < kNT; ++n) top = ptx::max3_nan(top, s[n][2 * e], s[n][2 * e + 1]);
      top = ptx::max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = ptx::max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // A row that has seen nothing yet weighs nothing; an infinite score makes a NaN, as the
      // formula does.
      const float base = top == -INFINITY ? 0.f : top;
      const float shrink = exp2_fast((m[e] - base) * mul), lift = kWeightShift - base * mul;
      m[e] = top;
      const uint64_t mul2 = ptx::pack_f2(mul, mul), lift2 = ptx::pack_f2(lift, lift);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        const float2 x = ptx::unpack_f2(ptx::fma_f2(ptx::pack_f2(s[n][2 * e], s[n][2 * e + 1]), mul2, lift2));
        const float p0 = exp2_fast(x.x), p1 = exp2_fast(x.y);
        sum[n & 1] = ptx::add_f2(sum[n & 1], ptx::pack_f2(p0, p1));
        pf[n][e] = pack2<T>(p0, p1);
      }
      const float2 total = ptx::unpack_f2(ptx::add_f2(sum[0], sum[1]));
      l[e] = l[e] * shrink + (total.x + total.y);
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
    ++tile;
    if (FORM == kWideAlone && tile == tile1) {
      // A head's last tile. A warp's rows go out through the places of its own queries, which
      // it has in registers (those of the first tile's stage, or the unused ones of this).
      const int h = kvh0 + step / tiles_here;
      join_lanes();
      __syncwarp();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];  // a row that sees nothing is zeros
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
          *reinterpret_cast<uint32_t*>(st + L::kStageQ + (wrow + g + 8 * e) * L::kRow + i * 16 + t4 * 4) =
              pack2<T>(o[i][2 * e] * inv, o[i][2 * e + 1] * inv);
      }
      __syncwarp();
      for (int i = lane; i < 16 * (DP / 8); i += 32) {
        const int r = wrow + i / (DP / 8), c = i % (DP / 8);
        if (r < rows && c < chunks) *place(h, r, c) = *reinterpret_cast<const uint4*>(st + L::kStageQ + r * L::kRow + c * 16);
      }
      tile = tile0;
      if (step + 1 < steps) {
        load_slopes(h + 1);
        reset();
      }
    }
  }
  copies_wait<0>();
  if constexpr (FORM == kWideAlone) return;
  const int kvh = kvh0;
  join_lanes();

  auto store8 = [&](int r, int c, const float (&f)[8]) {
    uint4 u;
    u.x = pack2<T>(f[0], f[1]);
    u.y = pack2<T>(f[2], f[3]);
    u.z = pack2<T>(f[4], f[5]);
    u.w = pack2<T>(f[6], f[7]);
    *place(kvh, r, c) = u;
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
      for (int w = 0; w < 4; ++w) top = ptx::max_nan(top, ml[w * 16 + r].x);
      mj[p] = make_float2(top, 0.f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[p][j] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 v = ml[w * 16 + r];
        const float k = v.x == -INFINITY ? 0.f : exp2_fast((v.x - top) * mul);
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
    for (int w = 0; w < ranks; ++w) top = ptx::max_nan(top, cluster.map_shared_rank(ml, w)[r].x);
    for (int w = 0; w < ranks; ++w) {
      const float2 v = cluster.map_shared_rank(ml, w)[r];
      const float k = v.x == -INFINITY ? 0.f : exp2_fast((v.x - top) * mul);
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

template <typename T, int DP, int FORM>
cudaError_t launch(const AttnArgs& a, int cluster, int tiles, cudaStream_t s) {
  auto fn = attn_mma_kernel<T, DP, FORM>;
  static AttrOnce once;
  cudaError_t e = once.set(reinterpret_cast<const void*>(fn), Layout<DP, FORM>::bytes(kStages), true);
  if (e != cudaSuccess) return e;
  if constexpr (FORM == kWideAlone) {
    // Several heads to a CTA, so that one's loads run under another's work, while that leaves
    // some CTAs for every place; and no more stages than it has steps.
    AttnArgs b = a;
    b.heads_per_block = static_cast<int>(
        std::clamp<long long>(static_cast<long long>(a.num_items) * a.kv_heads / (12LL * a.num_sms), 1, a.kv_heads));
    const long long steps = static_cast<long long>(tiles) * b.heads_per_block;
    const int smem = Layout<DP, FORM>::bytes(static_cast<int>(std::clamp<long long>(steps, 1, kStages)));
    const dim3 grid(a.num_items, (a.kv_heads + b.heads_per_block - 1) / b.heads_per_block);
    fn<<<grid, kThreads, smem, s>>>(b);
    return cudaGetLastError();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.num_items) * cluster, a.kv_heads);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Layout<DP, FORM>::bytes(kStages);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, fn, a);
}

template <typename T, int FORM>
cudaError_t by_dim(const AttnArgs& a, int cluster, int tiles, cudaStream_t s) {
  if (a.head_dim <= 32) return launch<T, 32, FORM>(a, cluster, tiles, s);
  if (a.head_dim <= 64) return launch<T, 64, FORM>(a, cluster, tiles, s);
  if (a.head_dim <= 96) return launch<T, 96, FORM>(a, cluster, tiles, s);
  return launch<T, 128, FORM>(a, cluster, tiles, s);
}

template <typename T>
cudaError_t by_form(const AttnArgs& a, bool few_rows, int cluster, int tiles, cudaStream_t s) {
  if (few_rows) return by_dim<T, kFew>(a, cluster, tiles, s);
  return cluster > 1 ? by_dim<T, kWideShared>(a, cluster, tiles, s) : by_dim<T, kWideAlone>(a, cluster, tiles, s);
}

}  // namespace

cudaError_t attn_mma_launch(const AttnArgs& a, int dtype, bool few_rows, int cluster, int tiles, cudaStream_t s) {
  return dtype == kTokenBf16 ? by_form<__nv_bfloat16>(a, few_rows, cluster, tiles, s)
                             : by_form<__half>(a, few_rows, cluster, tiles, s);
}

}  // namespace ah
