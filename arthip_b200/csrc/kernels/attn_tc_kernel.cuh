// Attention on the tcgen05 tensor cores for blocks of many rows. One CTA per SM takes two
// tiles of 128 queries that read the same keys: two tiles of one head, or, where an even
// number of query heads share a key head, the same 128 tokens of two heads.
//
//   S = Q K^T    A, B from shared memory (TMA, 128B swizzle, K-major), S in tensor memory
//   P = 2^(x - m)  one thread per row; rounded to 16 bits into the columns S was in
//   O += P V     A from tensor memory, B = V as TMA brought it (MN-major)
//
// Two warpgroups work on the two tiles' softmax in turn with the tensor cores: while one
// tile's S and O products run, the other's exponentials do. A thread holds a whole row of S,
// so its maximum and sum need no exchange. Warp 8 issues the TMA loads of the key and value
// tiles into a ring, warp 9 the products; its issue order (O += P V of a tile, then S of the
// same tile's next keys) makes S's completion stand for O's: a warpgroup that sees S may
// rescale O. It does so only where a row's maximum has grown by more than 2^8, so in most
// tiles O stays where it is; weights reach 2^14 at most, which fp16 holds.
//
// Masks, caps and biases are as in attn_mma.cu. Values behind a document's keys in use are
// written over with zeros in shared memory before the product that reads them, and whole
// steps of 16 keys that no row of a tile sees are left out.
//
// Every wait is bounded; one that runs out ends the CTA and sets the status word.
#pragma once

#include "attn_common.cuh"
#include "ptx.cuh"
#include "tokens.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ah {

struct AttnTcArgs {
  CUtensorMap q, k, v;  // {head_dim, tokens, heads}, box {64, 128, 1}, 128B swizzle
  AttnArgs a;
};

namespace attn_tc {

constexpr int kThreads = 320;
constexpr int kChunkBytes = 128 * 128;  // 128 rows of 64 elements
constexpr float kWeightShift = 6.f;     // weights are 2^(x - m + 6): a wider range above fp16's smallest
constexpr float kRescaleAt = 8.f;

// NCH: chunks of 64 elements in a head.
template <int NCH>
struct Smem {
  static constexpr int kSlots = NCH == 1 ? 6 : 4;
  static constexpr int kTile = NCH * kChunkBytes;
  static constexpr int kQ = 0;
  static constexpr int kRing = kQ + 2 * kTile;
  static constexpr int kPos = kRing + kSlots * kTile;  // key positions: [2 tiles][2 buffers][axes][128]
  static constexpr int kBars = kPos + 2 * 2 * kAttnMaxAxes * kTcKeys * 4;
  static constexpr int kBytes = kBars + 256 + 1024;    // and room to align to 1024
};

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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

template <typename T, int NCH, bool CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ AttnTcArgs args) {
  using L = Smem<NCH>;
  const AttnArgs& a = args.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full = bars;                 // [kSlots] a K or V tile has landed
  uint64_t* empty = full + L::kSlots;    // [kSlots] the products that read it are done
  uint64_t* s_full = empty + L::kSlots;  // [2] S of a tile (and the O before it) is complete
  uint64_t* p_ready = s_full + 2;        // [2] its weights are in tensor memory (a count of 4 warps)
  uint64_t* q_full = p_ready + 2;
  uint64_t* drained = q_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool pairs = a.group % 2 == 0;
  const AttnItem item = a.items[blockIdx.x];
  const AttnDoc doc = a.docs[item.doc];
  int klen = doc.nk;
  if (a.k_lens) klen = min(max(a.k_lens[item.doc], 0), doc.nk);
  const int prefix = min(doc.prefix, klen);
  auto hi_of = [&](int tok) {  // the document's keys [0, hi) are what token tok sees
    return a.causal ? min(klen, max(prefix, tok + klen - doc.nq + 1)) : klen;
  };
  int head[2], tok0[2], ntok[2], hi_top[2], tiles[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    head[g] = pairs ? 2 * blockIdx.y + g : blockIdx.y;
    tok0[g] = item.row0 + (pairs ? 0 : g * kTcRows);
    ntok[g] = min(kTcRows, max(0, doc.nq - tok0[g]));
    hi_top[g] = ntok[g] ? max(0, hi_of(tok0[g] + ntok[g] - 1)) : 0;
    tiles[g] = (hi_top[g] + kTcKeys - 1) / kTcKeys;
  }
  const int ntiles = max(tiles[0], tiles[1]);
  const int kvh = head[0] / a.group;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      ptx::mbar_init(ptx::smem_u32(full + i), 1);
      ptx::mbar_init(ptx::smem_u32(empty + i), 1);
    }
    for (int g = 0; g < 2; ++g) {
      ptx::mbar_init(ptx::smem_u32(s_full + g), 1);
      ptx::mbar_init(ptx::smem_u32(p_ready + g), 4);
    }
    ptx::mbar_init(ptx::smem_u32(q_full), 1);
    ptx::mbar_init(ptx::smem_u32(drained), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 9) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int never_abort = 0;

  if (warp == 8) {
    // ------------------------------------------------------------------ loads
    if (lane == 0) {
      ptx::prefetch_tensormap(&args.q);
      ptx::prefetch_tensormap(&args.k);
      ptx::prefetch_tensormap(&args.v);
      int issued = 0;
      if (ntiles > 0) {
        const uint32_t qb = ptx::smem_u32(q_full);
        ptx::mbar_arrive_expect_tx(qb, ((tiles[0] > 0) + (tiles[1] > 0)) * L::kTile);
        for (int g = 0; g < 2; ++g)
          for (int c = 0; c < NCH && tiles[g] > 0; ++c)
            ptx::tma_load_3d(ptx::smem_u32(smem + L::kQ + g * L::kTile + c * kChunkBytes), &args.q, qb, c * 64,
                             doc.q0 + tok0[g], head[g]);
      }
      for (; issued < 2 * ntiles; ++issued) {  // K and V of each tile in turn
        const int slot = issued % L::kSlots, use = issued / L::kSlots;
        if (!ptx::mbar_wait(ptx::smem_u32(empty + slot), (use & 1) ^ 1, abort_flag)) break;
        const uint32_t fb = ptx::smem_u32(full + slot);
        ptx::mbar_arrive_expect_tx(fb, L::kTile);
        const CUtensorMap* map = issued & 1 ? &args.v : &args.k;
        for (int c = 0; c < NCH; ++c)
          ptx::tma_load_3d(ptx::smem_u32(smem + L::kRing + slot * L::kTile + c * kChunkBytes), map, fb, c * 64,
                           doc.k0 + (issued >> 1) * kTcKeys, kvh);
      }
      // Nothing may be in flight when the CTA ends, which after a wait that ran out it might.
      if (ntiles > 0) ptx::mbar_wait(ptx::smem_u32(q_full), 0, &never_abort);
      for (int i = max(0, issued - L::kSlots); i < issued; ++i)
        ptx::mbar_wait(ptx::smem_u32(full + i % L::kSlots), (i / L::kSlots) & 1, &never_abort);
    }
    __syncwarp();
  } else if (warp == 9) {
    // --------------------------------------------------------------- products
    const int ksteps_q = (a.head_dim + 15) / 16;
    const uint32_t n_out = ksteps_q * 16;
    auto ring = [&](int seq) { return ptx::smem_u32(smem + L::kRing + seq % L::kSlots * L::kTile); };
    auto await = [&](uint64_t* bar, int parity) {  // the same answer in all lanes
      return __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(bar), parity, abort_flag)) != 0;
    };
    auto wait_full = [&](int seq) { return await(full + seq % L::kSlots, (seq / L::kSlots) & 1); };
    auto seen = [&](int g, int j) { return min(kTcKeys, hi_top[g] - j * kTcKeys); };  // keys of tile j
    auto issue_s = [&](int g, int j) {
      const uint32_t q = ptx::smem_u32(smem + L::kQ + g * L::kTile), k = ring(2 * j);
      const uint32_t idesc = ptx::idesc_16_f32(kIsBf16<T>, false, kTcRows, (seen(g, j) + 15) / 16 * 16);
      for (int s = 0; s < ksteps_q; ++s) {
        const uint32_t off = (s >> 2) * kChunkBytes + (s & 3) * 32;
        ptx::mma_f16_ss(tmem + g * 128, ptx::smem_desc(q + off, 2, 1024), ptx::smem_desc(k + off, 2, 1024), idesc,
                        s > 0);
      }
    };
    auto issue_o = [&](int g, int j) {
      const uint32_t v = ring(2 * j + 1);
      const uint32_t idesc = ptx::idesc_16_f32(kIsBf16<T>, true, kTcRows, n_out);
      const int steps = (seen(g, j) + 15) / 16;
      for (int s = 0; s < steps; ++s)
        ptx::mma_f16_ts(tmem + 256 + g * 128, tmem + g * 128 + s * 8,
                        ptx::smem_desc_mn128(v + s * 2048, kChunkBytes, 1024), idesc, j > 0 || s > 0);
    };
    bool ok = true;
    if (ntiles > 0) {
      ok = await(q_full, 0) && wait_full(0);
      ptx::tc_fence_after();
      if (ok && lane == 0) {
        for (int g = 0; g < 2; ++g)
          if (tiles[g] > 0) {
            issue_s(g, 0);
            ptx::mma_commit(ptx::smem_u32(s_full + g));
          }
        ptx::mma_commit(ptx::smem_u32(empty + 0));
      }
      __syncwarp();
    }
    for (int j = 0; j < ntiles && ok; ++j) {
      bool have_v = false, have_k = false;
      for (int g = 0; g < 2 && ok; ++g) {
        if (j >= tiles[g]) continue;
        if (!have_v) {
          ok = wait_full(2 * j + 1);
          have_v = true;
          const int used = klen - j * kTcKeys;
          if (ok && used < kTcKeys && used % 16) {  // zeros behind the keys in use, to the end of their step
            uint8_t* v = smem + L::kRing + (2 * j + 1) % L::kSlots * L::kTile;
            const int words = (16 - used % 16) * 8;  // of 16 bytes, per chunk
            for (int i = lane; i < NCH * words; i += 32)
              *reinterpret_cast<uint4*>(v + i / words * kChunkBytes + used * 128 + i % words * 16) =
                  make_uint4(0, 0, 0, 0);
            ptx::fence_proxy_async_smem();
            __syncwarp();
          }
        }
        ok = ok && await(p_ready + g, j & 1);
        const bool more = j + 1 < tiles[g];
        if (ok && more && !have_k) {
          ok = wait_full(2 * j + 2);
          have_k = true;
        }
        if (!ok) break;
        ptx::tc_fence_after();
        if (lane == 0) {
          issue_o(g, j);
          if (more) issue_s(g, j + 1);
          ptx::mma_commit(ptx::smem_u32(s_full + g));
        }
        __syncwarp();
      }
      if (ok && lane == 0) {
        ptx::mma_commit(ptx::smem_u32(empty + (2 * j + 1) % L::kSlots));
        if (j + 1 < ntiles) ptx::mma_commit(ptx::smem_u32(empty + (2 * j + 2) % L::kSlots));
      }
      __syncwarp();
    }
    // No product may be running when tensor memory is freed.
    if (lane == 0 && ntiles > 0) {
      ptx::mma_commit(ptx::smem_u32(drained));
      ptx::mbar_wait(ptx::smem_u32(drained), 0, &never_abort);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 2;
    const int r = threadIdx.x & 127;  // row of the tile = lane of tensor memory
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    const uint32_t ts = tmem + lanes + g * 128, to = tmem + lanes + 256 + g * 128;
    const int n = tiles[g];
    const bool mine = r < ntok[g];
    const int tok = tok0[g] + min(r, max(ntok[g] - 1, 0));
    const int hi = n ? hi_of(tok) : 0;
    const int hi_low = n ? hi_of(tok0[g]) : 0;
    float* pos_all = reinterpret_cast<float*>(smem + L::kPos) + g * 2 * kAttnMaxAxes * kTcKeys;
    float slope[kAttnMaxAxes], qpos[kAttnMaxAxes], kpos[kAttnMaxAxes];
    auto fetch_pos = [&](int j) {  // one key of tile j per thread
      const int key = j * kTcKeys + r;
#pragma unroll
      for (int ax = 0; ax < kAttnMaxAxes; ++ax)
        if (ax < a.axes) kpos[ax] = key < klen ? a.k_pos[ax * a.k_total + doc.k0 + key] : 0.f;
    };
    if constexpr (BIAS) {
#pragma unroll
      for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
        slope[ax] = ax < a.axes && n ? a.slopes[head[g] * a.axes + ax] : 0.f;
        qpos[ax] = ax < a.axes && n ? a.q_pos[ax * a.q_total + doc.q0 + tok] : 0.f;
      }
      if (n) fetch_pos(0);
    }
    const float mul = CAP || BIAS ? 1.f : a.score_mul;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      float* pos = pos_all + (j & 1) * kAttnMaxAxes * kTcKeys;
      if constexpr (BIAS) {
#pragma unroll
        for (int ax = 0; ax < kAttnMaxAxes; ++ax)
          if (ax < a.axes) pos[ax * kTcKeys + r] = kpos[ax];
        asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
        if (j + 1 < n) fetch_pos(j + 1);
      }
      // After a wait that ran out, only the group's barrier is still met.
      if (ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(s_full + g), j & 1, abort_flag));
      if (!ok) continue;
      ptx::tc_fence_after();
      uint32_t u[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(ts + c * 32, u[c]);
      ptx::tmem_wait_ld();
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if constexpr (CAP || BIAS) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float x = __uint_as_float(u[c][i]);
            if constexpr (CAP)
              x = attn_capped(x, a);
            else
              x *= a.score_mul;
            u[c][i] = __float_as_uint(x);
          }
          if constexpr (BIAS) {
#pragma unroll
            for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
              if (ax >= a.axes) break;
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 kp = *reinterpret_cast<const float4*>(pos + ax * kTcKeys + c * 32 + i);
                u[c][i] = __float_as_uint(__uint_as_float(u[c][i]) - slope[ax] * fabsf(qpos[ax] - kp.x));
                u[c][i + 1] = __float_as_uint(__uint_as_float(u[c][i + 1]) - slope[ax] * fabsf(qpos[ax] - kp.y));
                u[c][i + 2] = __float_as_uint(__uint_as_float(u[c][i + 2]) - slope[ax] * fabsf(qpos[ax] - kp.z));
                u[c][i + 3] = __float_as_uint(__uint_as_float(u[c][i + 3]) - slope[ax] * fabsf(qpos[ax] - kp.w));
              }
            }
          }
        }
        if ((j + 1) * kTcKeys > hi_low) {
          const int lim = hi - j * kTcKeys - c * 32;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (i >= lim) u[c][i] = 0xff800000u;
        }
        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          t0 = fmaxf(t0, __uint_as_float(u[c][i]));
          t1 = fmaxf(t1, __uint_as_float(u[c][i + 1]));
        }
        top = fmaxf(top, fmaxf(t0, t1));
      }
      const float m_new = fmaxf(m, top);
      if (j == 0) {
        m = m_new;
      } else {
        const bool grow = (m_new - m) * mul > kRescaleAt;
        if (__any_sync(0xffffffffu, grow)) {
          const float shrink = grow ? exp2_fast((m - m_new) * mul) : 1.f;
          if (grow) m = m_new;
          l *= shrink;
          for (int c = 0; c < a.head_dim; c += 16) {
            uint32_t o[32];
            ptx::tmem_ld_32x32b_x16(to + c, o);
            ptx::tmem_wait_ld();
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
            ptx::tmem_st_32x32b_x16(to + c, w);
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : kWeightShift - m * mul;
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p0 = exp2_fast(__uint_as_float(u[c][2 * i]) * mul + base);
          const float p1 = exp2_fast(__uint_as_float(u[c][2 * i + 1]) * mul + base);
          sum += p0 + p1;
          w[i] = pack2<T>(p0, p1);
        }
        ptx::tmem_st_32x32b_x16(ts + c * 16, w);
      }
      l += sum;
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(p_ready + g));
    }
    if (n > 0 && ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(s_full + g), n & 1, abort_flag));
    if (ok) {
      ptx::tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing is zeros
      T* dst = static_cast<T*>(a.out) + static_cast<long long>(doc.q0 + tok) * a.o_tok + head[g] * a.o_head;
      for (int c = 0; c < a.head_dim; c += 16) {
        uint32_t o[32];
        if (n > 0) {
          ptx::tmem_ld_32x32b_x16(to + c, o);
          ptx::tmem_wait_ld();
        }
        if (!mine) continue;
        uint4 w[2];
        uint32_t* p = reinterpret_cast<uint32_t*>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          p[i] = n > 0 ? pack2<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv) : 0u;
        *reinterpret_cast<uint4*>(dst + c) = w[0];
        if (c + 8 < a.head_dim) *reinterpret_cast<uint4*>(dst + c + 8) = w[1];
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 9) ptx::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) atomicOr(a.status, 1u);
}

template <typename T, int NCH, bool CAP, bool BIAS>
cudaError_t launch(const AttnTcArgs& args, cudaStream_t s) {
  auto fn = attn_tc_kernel<T, NCH, CAP, BIAS>;
  static AttrOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(fn), Smem<NCH>::kBytes);
  if (e != cudaSuccess) return e;
  const AttnArgs& a = args.a;
  const int heads = attn_tc_head_pairs(a.group) ? a.q_heads / 2 : a.q_heads;
  fn<<<dim3(a.num_items, heads), kThreads, Smem<NCH>::kBytes, s>>>(args);
  return cudaGetLastError();
}

template <typename T, int NCH>
cudaError_t launch_variant(const AttnTcArgs& args, cudaStream_t s) {
  const bool cap = args.a.cap_log2 > 0.f, bias = args.a.axes > 0;
  if (cap) return bias ? launch<T, NCH, true, true>(args, s) : launch<T, NCH, true, false>(args, s);
  return bias ? launch<T, NCH, false, true>(args, s) : launch<T, NCH, false, false>(args, s);
}

// One translation unit each (attn_tc_*.cu).
cudaError_t launch_f16_1(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_f16_2(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_bf16_1(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_bf16_2(const AttnTcArgs& args, cudaStream_t s);

}  // namespace attn_tc
}  // namespace ah
