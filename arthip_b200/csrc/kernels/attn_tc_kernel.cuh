// Attention on the tcgen05 tensor cores for blocks of many rows. One CTA per SM takes two
// tiles of 128 queries that read the same keys: two tiles of one head, or, where an even
// number of query heads share a key head, the same 128 tokens of two heads.
//
//   S = Q K^T    A, B from shared memory (TMA, 128B swizzle, K-major), S in tensor memory
//   P = 2^(x - m)  rounded to 16 bits, in tensor memory
//   O += P V     A from tensor memory, B = V as TMA brought it (MN-major)
//
// Keys are taken 128 at a time. Eight warps work on each tile's softmax, 16 rows each, so that
// each of the SM's four schedulers has four of them: some have exponentials to do while others
// wait for S, load it or look for its maximum. Four threads share a row (the 16-lane loads of
// tensor memory give each of them every fourth pair of columns) and find its maximum with two
// shuffles. Half of the scores are loaded a second time rather than kept, which holds a thread
// to the 96 registers that 19 warps leave it; with a cap or a bias it is not quite enough, and 32
// to 132 bytes a thread are spilled (1.4% of the instructions of a capped and biased run). Warp 16
// issues the TMA loads of key and value tiles into a ring, warps 17 and 18 the products of one tile
// each.
//
// Heads of up to 64 have room for P beside S: S of the next keys is computed as soon as this
// one has been loaded into registers, and a softmax warp never waits for the round trip
// through the tensor cores. For wider heads P takes the place of S, and S of the next keys
// follows O += P V; there the two tiles' warps work in turn.
//
// O is rescaled only where a row's maximum has grown by more than 2^8, so in most steps it
// stays where it is; weights reach 2^14 at most, which fp16 holds.
//
// Masks, caps and biases are as in attn_mma.cu. Values behind a document's keys in use are
// written over with zeros in shared memory before the product that reads them, and whole
// steps of 16 keys that no row of a tile sees are left out.
//
// Every wait is bounded; one that runs out ends the CTA and sets the status word.
//
// Bound: latency, with the special function unit (one exponential a score at 16 per clock) and the
// issue of the 5.9 instructions that a score takes nearest to full. 32400 tokens, 8 heads of 64: 2.77
// to 3.03 ms (exponentials alone 1.92 ms at 1.85 GHz, products 1.27 ms); counted at 2.94 ms, the unit
// is 73% busy and issue 0.54. Capped and biased, 128 elements a head: unit 60%, issue 0.42. Tried
// beside this: issue by lane 0 instead of an elected thread 4.0 ms; two softmax warps per scheduler,
// whole rows, 3.1; keys 64 at a time with two buffers of S 3.5; a quarter of the exponentials as
// polynomials on the FMA pipe 2.93.
#pragma once

#include "token_common.cuh"
#include "tokens.h"

namespace ah {

struct AttnTcArgs {
  CUtensorMap q, k, v;  // {head_dim, tokens, heads}, box {64, 128, 1}, 128B swizzle
  AttnArgs a;
  unsigned long long wait_limit_ns;  // bound of every pipeline wait (4 s)
  int stall_load;  // failure-path test: the load (K and V of each tile in turn) that never comes, or -1
};

namespace attn_tc {

constexpr int kThreads = 608;
constexpr int kLoadWarp = 16, kProductWarp = 17;  // and the next; softmax: 0-15
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
  static constexpr int kSums = kPos + 2 * 2 * kAttnMaxAxes * kTcKeys * 4;  // [2 tiles][128]
  static constexpr int kBars = kSums + 2 * kTcRows * 4;
  // tensor memory columns
  static constexpr bool kOwnP = NCH == 1;  // P has columns of its own
  static constexpr int kCols = NCH * 64;   // of O
  static constexpr int kColO = 256, kColP = kOwnP ? 384 : 0, kStrideP = kOwnP ? 64 : 128;
  static constexpr int kBytes = kBars + 256 + 1024;    // and room to align to 1024
};

template <typename T>
constexpr bool kIsBf16 = false;
template <>
constexpr bool kIsBf16<__nv_bfloat16> = true;

// The weights 2^(u * mul + base) of a thread's share of 64 columns (16-lane layout: registers
// 4k, 4k + 1 are of its first row, 4k + 2, 4k + 3 of its second), packed to 16 bits, and their
// sums added to `sum`.
template <typename T>
__device__ __forceinline__ void weights32(const uint32_t (&u)[32], uint64_t mul, const uint64_t (&base)[2],
                                          uint32_t (&w)[16], uint64_t (&sum)[2]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint64_t x =
        ptx::fma_f2(ptx::pack_f2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1])), mul, base[i & 1]);
    const float2 v = ptx::unpack_f2(x);
    const float p0 = exp2_fast(v.x), p1 = exp2_fast(v.y);
    sum[i & 1] = ptx::add_f2(sum[i & 1], ptx::pack_f2(p0, p1));
    w[i] = pack2<T>(p0, p1);
  }
}

template <typename T, int NCH, int CAP, bool BIAS>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ AttnTcArgs args) {
  using L = Smem<NCH>;
  const AttnArgs& a = args.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* full = bars;                 // [kSlots] a K or V tile has landed
  uint64_t* empty = full + L::kSlots;    // [kSlots] the products that read it are done
  uint64_t* s_full = empty + L::kSlots;  // [2 tiles] S of a step is complete (wide heads: and O before it)
  uint64_t* s_free = s_full + 2;         // [2] it has been loaded (a count of 8 warps)
  uint64_t* p_ready = s_free + 2;        // [2] its weights are in tensor memory (8 warps)
  uint64_t* o_done = p_ready + 2;        // [2] and have been added to O
  uint64_t* q_full = o_done + 2;
  uint64_t* drained = q_full + 1;        // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool pairs = a.group % 2 == 0;
  const AttnItem item = a.items[blockIdx.x];
  const AttnDoc doc = a.docs[item.doc];
  int klen = doc.nk;
  if (a.k_lens) klen = min(max(a.k_lens[item.doc], 0), doc.nk);
  const int prefix = min(doc.prefix, klen);
  auto hi_of = [&](int tok) {  // the document's keys [0, hi) are what token tok sees
    return a.causal ? min(klen, max(prefix, klen - (doc.nq - tok) + 1)) : klen;
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
      ptx::mbar_init(ptx::smem_u32(empty + i), 2);
    }
    for (int g = 0; g < 2; ++g) {
      ptx::mbar_init(ptx::smem_u32(s_full + g), 1);
      ptx::mbar_init(ptx::smem_u32(s_free + g), 8);
      ptx::mbar_init(ptx::smem_u32(p_ready + g), 8);
      ptx::mbar_init(ptx::smem_u32(o_done + g), 1);
    }
    ptx::mbar_init(ptx::smem_u32(q_full), 1);
    ptx::mbar_init(ptx::smem_u32(drained), 1);
    ptx::mbar_init(ptx::smem_u32(drained + 1), 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == kProductWarp) {
    ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int never_abort = 0;

  if (warp == kLoadWarp) {
    // ------------------------------------------------------------------ loads
    if (ptx::elect_one()) {
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
        if (!ptx::mbar_wait_short(ptx::smem_u32(empty + slot), (use & 1) ^ 1, abort_flag, args.wait_limit_ns)) break;
        const uint32_t fb = ptx::smem_u32(full + slot);
        ptx::mbar_arrive_expect_tx(fb, L::kTile);
        if (issued == args.stall_load) continue;
        const CUtensorMap* map = issued & 1 ? &args.v : &args.k;
        for (int c = 0; c < NCH; ++c)
          ptx::tma_load_3d(ptx::smem_u32(smem + L::kRing + slot * L::kTile + c * kChunkBytes), map, fb, c * 64,
                           doc.k0 + (issued >> 1) * kTcKeys, kvh);
      }
      // Nothing may be in flight when the CTA ends, which after a wait that ran out it might.
      if (ntiles > 0) ptx::mbar_wait_short(ptx::smem_u32(q_full), 0, &never_abort, args.wait_limit_ns);
      for (int i = max(0, issued - L::kSlots); i < issued; ++i)
        ptx::mbar_wait_short(ptx::smem_u32(full + i % L::kSlots), (i / L::kSlots) & 1, &never_abort, args.wait_limit_ns);
    }
    __syncwarp();
  } else if (warp >= kProductWarp) {
    // --------------------------------------------------------------- products
    // The issue loops hold nothing but additions of constants: descriptors and counts are made
    // once, as one thread's instructions between two products are what would bound them.
    const int g = warp - kProductWarp;
    const int ksteps = (a.head_dim + 15) / 16;
    const uint32_t idesc_s = ptx::idesc_16_f32(kIsBf16<T>, false, kTcRows, 0);
    const uint32_t idesc_o = ptx::idesc_16_f32(kIsBf16<T>, true, kTcRows, ksteps * 16);
    constexpr uint32_t kHi = ptx::desc_hi(1024, 2);
    const uint32_t ring0 = ptx::smem_u32(smem + L::kRing);
    const uint32_t q_lo = ptx::desc_lo(ptx::smem_u32(smem + L::kQ)) + g * (L::kTile >> 4);
    const uint32_t k_lo = ptx::desc_lo(ring0), v_lo = ptx::desc_lo_mn(ring0, kChunkBytes);
    const uint32_t ts = tmem + g * 128, to = tmem + L::kColO + g * L::kCols;
    const uint32_t tp = tmem + L::kColP + g * L::kStrideP;
    const int n = tiles[g];
    auto slot_words = [&](int seq) { return static_cast<uint32_t>(seq % L::kSlots * (L::kTile >> 4)); };
    auto await = [&](uint64_t* bar, int parity) {
      return ptx::mbar_wait_short(ptx::smem_u32(bar), parity, abort_flag, args.wait_limit_ns);
    };
    auto wait_full = [&](int seq) { return await(full + seq % L::kSlots, (seq / L::kSlots) & 1); };
    auto release = [&](int seq) { ptx::mma_commit(ptx::smem_u32(empty + seq % L::kSlots)); };
    auto key_steps = [&](int j) {  // 16s of keys of tile j that some row sees
      return (min(kTcKeys, hi_top[g] - j * kTcKeys) + 15) / 16;
    };
    auto issue_s = [&](int j) {
      const uint32_t k = k_lo + slot_words(2 * j);
      const uint32_t idesc = idesc_s | static_cast<uint32_t>(key_steps(j)) << 18;  // N / 8
#pragma unroll
      for (int s = 0; s < 4 * NCH; ++s) {
        const uint32_t off = ((s >> 2) * kChunkBytes + (s & 3) * 32) >> 4;
        if (s < ksteps) ptx::mma_f16_ss2(ts, q_lo + off, kHi, k + off, kHi, idesc, s > 0);
      }
    };
    auto issue_o = [&](int j) {
      const uint32_t v = v_lo + slot_words(2 * j + 1), more = j > 0;
      const int steps = key_steps(j);
#pragma unroll
      for (int s = 0; s < 8; ++s)
        if (s < steps) ptx::mma_f16_ts(to, tp + s * 8, v + s * 128, kHi, idesc_o, s > 0 ? 1u : more);
    };
    auto clear_values = [&](int j) {  // zeros behind the keys in use, to the end of their 16
      const int used = klen - j * kTcKeys;
      if (used >= kTcKeys || used % 16 == 0) return;
      uint8_t* v = smem + L::kRing + (2 * j + 1) % L::kSlots * L::kTile;
      const int words = (16 - used % 16) * 8;  // of 16 bytes, per chunk
      for (int i = 0; i < NCH * words; ++i)
        *reinterpret_cast<uint4*>(v + i / words * kChunkBytes + used * 128 + i % words * 16) = make_uint4(0, 0, 0, 0);
      ptx::fence_proxy_async_smem();
    };
    if (ntiles > 0 && ptx::elect_one()) {
      bool ok = (n == 0 || await(q_full, 0)) && wait_full(0);
      if (ok) {
        ptx::tc_fence_after();
        if (n > 0) issue_s(0);
        ptx::mma_commit(ptx::smem_u32(s_full + g));
        release(0);
      }
      for (int j = 0; j < ntiles && ok; ++j) {
        const bool last = j + 1 == ntiles;
        if constexpr (L::kOwnP) {
          if (!last) {
            ok = wait_full(2 * j + 2) && (j + 1 >= n || await(s_free + g, j & 1));
            if (!ok) break;
            ptx::tc_fence_after();
            if (j + 1 < n) {
              issue_s(j + 1);
              ptx::mma_commit(ptx::smem_u32(s_full + g));
            }
            release(2 * j + 2);
          }
          ok = wait_full(2 * j + 1);
          if (!ok) break;
          clear_values(j);
          if (j < n) {
            ok = await(p_ready + g, j & 1);
            if (!ok) break;
            ptx::tc_fence_after();
            issue_o(j);
            ptx::mma_commit(ptx::smem_u32(o_done + g));
          }
          release(2 * j + 1);
        } else {
          ok = wait_full(2 * j + 1) && (last || wait_full(2 * j + 2));
          if (!ok) break;
          clear_values(j);
          if (j < n) {
            ok = await(p_ready + g, j & 1);
            if (!ok) break;
            ptx::tc_fence_after();
            issue_o(j);
            if (j + 1 < n) issue_s(j + 1);
            ptx::mma_commit(ptx::smem_u32(s_full + g));
          }
          release(2 * j + 1);
          if (!last) release(2 * j + 2);
        }
      }
      // No product may be running when tensor memory is freed.
      ptx::mma_commit(ptx::smem_u32(drained + g));
      ptx::mbar_wait_short(ptx::smem_u32(drained + g), 0, &never_abort, args.wait_limit_ns);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 3;
    const int row16 = (warp & 3) * 32 + (warp >> 2 & 1) * 16;  // this warp's rows of the tile
    const int t4 = lane & 3;
    const uint32_t lanes = static_cast<uint32_t>(row16) << 16;
    const uint32_t ts = tmem + lanes + g * 128;
    const uint32_t to = tmem + lanes + L::kColO + g * L::kCols;
    const uint32_t tp = tmem + lanes + L::kColP + g * L::kStrideP;
    const int n = tiles[g];
    const int hi_low = n ? hi_of(tok0[g]) : 0;
    int hi[2];
    float slope[kAttnMaxAxes], qpos[2][kAttnMaxAxes];
#pragma unroll
    for (int e = 0; e < 2; ++e) {  // this thread's two rows, row16 + lane / 4 and + 8
      const int tok = tok0[g] + min(row16 + (lane >> 2) + 8 * e, max(ntok[g] - 1, 0));
      hi[e] = n ? hi_of(tok) : 0;
      if constexpr (BIAS) {
#pragma unroll
        for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
          slope[ax] = ax < a.axes && n ? a.slopes[head[g] * a.axes + ax] : 0.f;
          qpos[e][ax] = ax < a.axes && n ? a.q_pos[ax * a.q_total + doc.q0 + tok] : 0.f;
        }
      }
    }
    bool ok = true;
    auto await = [&](uint64_t* bar, int parity) {  // the same answer in all lanes
      ok = ok && __all_sync(0xffffffffu, ptx::mbar_wait_short(ptx::smem_u32(bar), parity, abort_flag, args.wait_limit_ns));
    };
    auto arrive = [&](uint64_t* bar) {
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(bar));
    };
    auto meet = [&] { asm volatile("bar.sync %0, 256;" ::"r"(1 + g) : "memory"); };  // the tile's eight warps
    float* poss = reinterpret_cast<float*>(smem + L::kPos) + g * 2 * kAttnMaxAxes * kTcKeys;
    // The negated positions of the keys of tile j, into the buffer of j: written before the
    // meeting of tile j, read after it.
    auto stage_positions = [&](int j) {
      const int t = threadIdx.x & 255, key = j * kTcKeys + (t & 127);
      float* put = poss + (j & 1) * kAttnMaxAxes * kTcKeys;
      for (int ax = t >> 7; ax < a.axes; ax += 2)
        put[ax * kTcKeys + (t & 127)] = key < klen ? -a.k_pos[ax * a.k_total + doc.k0 + key] : 0.f;
    };
    const float mul = CAP ? 1.f : a.score_mul;  // from the scores' units to powers of two
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, top[2];
    // Caps, biases and masks 64 columns of tile j and takes the rows' largest into `top`.
    auto prepare = [&](int j, int c, uint32_t(&x)[32], bool masked) {
      if constexpr (CAP || BIAS) {
        if constexpr (CAP != kCapNone) {
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 v = ptx::unpack_f2(
                attn_capped2<CAP>(ptx::pack_f2(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), a));
            x[e] = __float_as_uint(v.x), x[e + 1] = __float_as_uint(v.y);
          }
        }
        if constexpr (BIAS) {
          const float* pos = poss + (j & 1) * kAttnMaxAxes * kTcKeys + c * 64 + 2 * t4;
#pragma unroll
          for (int ax = 0; ax < kAttnMaxAxes; ++ax) {
            if (ax >= a.axes) break;
            const uint64_t fall = ptx::pack_f2(-slope[ax], -slope[ax]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint64_t away = *reinterpret_cast<const uint64_t*>(pos + ax * kTcKeys + k * 8);  // negated
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t* y = x + 4 * k + 2 * e;
                const float2 far = ptx::unpack_f2(ptx::add_f2(ptx::pack_f2(qpos[e][ax], qpos[e][ax]), away));
                const float2 z = ptx::unpack_f2(
                    ptx::fma_f2(ptx::pack_f2(fabsf(far.x), fabsf(far.y)), fall,
                                ptx::pack_f2(__uint_as_float(y[0]), __uint_as_float(y[1]))));
                y[0] = __float_as_uint(z.x), y[1] = __float_as_uint(z.y);
              }
            }
          }
        }
      }
      if (masked) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (8 * (e >> 2) + (e & 1) >= hi[e >> 1 & 1] - (j * kTcKeys + c * 64 + 2 * t4)) x[e] = 0xff800000u;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          top[e] = ptx::max3_nan(top[e], __uint_as_float(x[4 * k + 2 * e]), __uint_as_float(x[4 * k + 2 * e + 1]));
    };
    for (int j = 0; j < n; ++j) {
      const bool masked = (j + 1) * kTcKeys > hi_low;
      if constexpr (BIAS) {
        stage_positions(j);
        meet();  // after a wait that ran out, only this is still done
      }
      await(s_full + g, j & 1);
      if (!ok) continue;
      ptx::tc_fence_after();
      uint32_t u[32], v[32], w[16];
      top[0] = top[1] = -INFINITY;
      ptx::tmem_ld_16x256b_x8(ts + 64, v);
      ptx::tmem_wait_ld(v);
      ptx::tmem_ld_16x256b_x8(ts, u);
      prepare(j, 1, v, masked);
      if constexpr (CAP || BIAS) ptx::tmem_st_16x256b_x8(ts + 64, v);  // for the second loading
      ptx::tmem_wait_ld(u);
      prepare(j, 0, u, masked);
      float m_new[2];
      bool grow = false;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = ptx::max_nan(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
        top[e] = ptx::max_nan(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
        m_new[e] = ptx::max_nan(m[e], top[e]);
        grow |= !((m_new[e] - m[e]) * mul <= kRescaleAt) && m_new[e] != m[e];  // NaN grows
      }
      if (L::kOwnP && j > 0) {  // P's columns are free, and O is at rest
        await(o_done + g, (j - 1) & 1);
        if (!ok) continue;
        ptx::tc_fence_after();
      }
      if (j == 0) {
        m[0] = m_new[0], m[1] = m_new[1];
      } else if (__any_sync(0xffffffffu, grow)) {
        float shrink[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          shrink[e] = m_new[e] == m[e] ? 1.f : exp2_fast((m[e] - m_new[e]) * mul);
          m[e] = m_new[e];
          l[e] *= shrink[e];
        }
        for (int c = 0; c < a.head_dim; c += 16) {
          uint32_t o[8];
          ptx::tmem_ld_16x256b_x2(to + c, o);
          ptx::tmem_wait_ld(o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink[e >> 1 & 1]);
          ptx::tmem_st_16x256b_x2(to + c, o);
        }
      }
      uint64_t base[2], sum[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // A row that has seen nothing yet weighs nothing; an infinite score makes a NaN, as the
        // formula does.
        const float shift = m[e] == -INFINITY ? 0.f : kWeightShift - m[e] * mul;
        const float b = m[e] == INFINITY ? NAN : shift;
        base[e] = ptx::pack_f2(b, b);
      }
      const uint64_t mul2 = ptx::pack_f2(mul, mul);
      if constexpr (CAP || BIAS) ptx::tmem_wait_st();
      ptx::tmem_ld_16x256b_x8(ts + 64, v);
      weights32<T>(u, mul2, base, w, sum);
      ptx::tmem_st_16x128b_x8(tp, w);
      ptx::tmem_wait_ld(v);
      if constexpr (L::kOwnP) arrive(s_free + g);
      if (!CAP && !BIAS && masked) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (8 * (e >> 2) + (e & 1) >= hi[e >> 1 & 1] - (j * kTcKeys + 64 + 2 * t4)) v[e] = 0xff800000u;
      }
      weights32<T>(v, mul2, base, w, sum);
      ptx::tmem_st_16x128b_x8(tp + 32, w);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 s2 = ptx::unpack_f2(sum[e]);
        l[e] += s2.x + s2.y;
      }
      ptx::tmem_wait_st();
      arrive(p_ready + g);
    }
    ptx::tmem_wait_st();  // a step that a wait ended early may have left stores under way
    if (n > 0) {
      if constexpr (L::kOwnP)
        await(o_done + g, (n - 1) & 1);
      else
        await(s_full + g, n & 1);
    }
    float* sums = reinterpret_cast<float*>(smem + L::kSums) + g * kTcRows;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if (t4 == 0) sums[row16 + (lane >> 2) + 8 * e] = l[e];
    }
    meet();
    if (ok) {  // two warps to 32 rows, a thread to a row: every other 16 columns each
      ptx::tc_fence_after();
      const int r = (warp & 3) * 32 + lane;
      const float sum = sums[r];
      const float inv = sum == 0.f ? 0.f : 1.f / sum;  // a row that sees nothing is zeros
      T* dst = static_cast<T*>(a.out) + static_cast<long long>(doc.q0 + tok0[g] + r) * a.o_tok + head[g] * a.o_head;
      const uint32_t from = tmem + (static_cast<uint32_t>(warp & 3) << 21) + L::kColO + g * L::kCols;
      for (int c = (warp >> 2 & 1) * 16; c < a.head_dim; c += 32) {
        uint32_t o[32];
        if (n > 0) {
          ptx::tmem_ld_32x32b_x16(from + c, o);
          ptx::tmem_wait_ld_x16(o);
        }
        if (r < ntok[g]) {
          uint4 q[2];
          uint32_t* p = reinterpret_cast<uint32_t*>(q);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            p[i] = n > 0 ? pack2<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv) : 0u;
          *reinterpret_cast<uint4*>(dst + c) = q[0];
          if (c + 8 < a.head_dim) *reinterpret_cast<uint4*>(dst + c + 8) = q[1];
        }
        __syncwarp();  // the next load wants the whole warp together, lanes behind the last query too
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == kProductWarp) ptx::tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) atomicOr(a.status, 1u);
}

template <typename T, int NCH, int CAP, bool BIAS>
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

template <typename T, int NCH, int CAP>
cudaError_t launch_biased(const AttnTcArgs& args, cudaStream_t s) {
  return args.a.axes > 0 ? launch<T, NCH, CAP, true>(args, s) : launch<T, NCH, CAP, false>(args, s);
}

template <typename T, int NCH>
cudaError_t launch_variant(const AttnTcArgs& args, cudaStream_t s) {
  switch (cap_form(args.a)) {
    case kCapExp: return launch_biased<T, NCH, kCapExp>(args, s);
    case kCapSeries: return launch_biased<T, NCH, kCapSeries>(args, s);
    default: return launch_biased<T, NCH, kCapNone>(args, s);
  }
}

// One translation unit each (attn_tc_*.cu).
cudaError_t launch_f16_1(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_f16_2(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_bf16_1(const AttnTcArgs& args, cudaStream_t s);
cudaError_t launch_bf16_2(const AttnTcArgs& args, cudaStream_t s);

}  // namespace attn_tc
}  // namespace ah
