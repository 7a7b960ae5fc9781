// Rotary positions over several axes: the pair (a, b) of a head that belongs to axis s turns
// by pos[s] * frequency,
//
//   (a cos - b sin, a sin + b cos).
//
// The angle is counted in turns: position * (frequency / 2 pi) in fp64, minus the nearest
// whole number, so that a far position loses nothing before it is rounded to fp32. One block
// takes a few tokens and puts their cosines and sines in shared memory once. A thread keeps one
// place within the head: it takes that place's cosines and sines of a token into registers and
// turns it in one head after another of q and k. Vectors to come are on their way into the
// thread's own places in shared memory meanwhile (asynchronous copies, some deep).
//
// Bound: HBM, 4 bytes per element (read, write).
#include "token_common.cuh"
#include "tokens.h"

#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ah {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTableBytes = 16384;  // cosines and sines of a block's tokens

__device__ __forceinline__ float2 unpack(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 unpack(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void pack(float2 f, __half2* o) { *o = __float22half2_rn(f); }
__device__ __forceinline__ void pack(float2 f, __nv_bfloat162* o) { *o = __float22bfloat162_rn(f); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }

template <typename T>
struct Two;
template <>
struct Two<__half> {
  using type = __half2;
};
template <>
struct Two<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// How a head is cut into the units that one thread turns:
//   kUnitPairs   8 elements, four adjacent pairs
//   kUnitHalves  8 pairs: 8 elements and the 8 elements that turn with them
//   kUnitOne     one pair, element by element
// Elements behind the rotated part are copied, 8 (or 1) at a time.
enum Unit : int { kUnitPairs = 0, kUnitHalves = 1, kUnitOne = 2 };

// How a block's threads are laid out over a pass: `width` places of a head, `heads` heads,
// `tokens` tokens.
struct RopeGrid {
  int tok_per_block;
  int turn_units, units;  // places of a head that turn, and all
  int width, heads, tokens;
};

constexpr int kRopeDepth = 4;  // items of a thread in flight

template <typename T, int UNIT>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeTable t, const RopeArgs a, const RopeGrid g) {
  constexpr int kVecs = UNIT == kUnitHalves ? 2 : 1;  // 16-byte vectors of an item
  constexpr int kPairs = UNIT == kUnitPairs ? 4 : (UNIT == kUnitHalves ? 8 : 1);
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;  // [depth][vector][thread]
  float2* cs = reinterpret_cast<float2*>(smem + (UNIT == kUnitOne ? 0 : kRopeDepth * kVecs * kRopeThreads * 16));
  using T2 = typename Two<T>::type;
  const long long tok0 = static_cast<long long>(blockIdx.x) * g.tok_per_block;
  const int ntok = static_cast<int>(min(static_cast<long long>(g.tok_per_block), a.tokens - tok0));
  const int all = a.heads[0] + a.heads[1];
  const int u0 = threadIdx.x % g.width, slot = threadIdx.x / g.width;
  const int h0 = slot % g.heads, first = slot / g.heads < g.tokens ? slot / g.heads : ntok;
  // Heads of k follow those of q. (The parameters are chosen from by value: an index into them
  // that is not known when compiling copies them to local memory, which cost a third.)
  auto source = [&](int tok, int h) {
    const bool k = h >= a.heads[0];
    return static_cast<const T*>(k ? a.in[1] : a.in[0]) + (tok0 + tok) * (k ? a.in_tok[1] : a.in_tok[0]) +
           (k ? (h - a.heads[0]) * a.in_head[1] : h * a.in_head[0]);
  };
  auto target = [&](int tok, int h) {
    const bool k = h >= a.heads[0];
    return static_cast<T*>(k ? a.out[1] : a.out[0]) + (tok0 + tok) * (k ? a.out_tok[1] : a.out_tok[0]) +
           (k ? (h - a.heads[0]) * a.out_head[1] : h * a.out_head[0]);
  };
  auto advance = [&](int* tok, int* h) {
    *h += g.heads;
    if (*h >= all) *h = h0, *tok += g.tokens;
  };
  const bool turn = u0 < g.turn_units;
  int e0 = u0 * 8, e1 = 0;  // the place's elements
  if constexpr (UNIT == kUnitHalves) {
    e0 = turn ? t.pairs[u0 * 8].e0 : t.rot + (u0 - g.turn_units) * 8;
    e1 = turn ? t.pairs[u0 * 8].e1 : e0;
  }
  int next_tok = first, next_h = h0;
  auto issue = [&](int at) {
    if (next_tok < ntok) {
      const T* in = source(next_tok, next_h);
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(
                         __cvta_generic_to_shared(ring + (at * kVecs + v) * kRopeThreads))),
                     "l"(in + (v ? e1 : e0))
                     : "memory");
      advance(&next_tok, &next_h);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (UNIT != kUnitOne) {
#pragma unroll
    for (int d = 0; d < kRopeDepth; ++d) issue(d);
  }
  for (int i = threadIdx.x; i < ntok * t.npairs; i += kRopeThreads) {
    const int tok = i / t.npairs;
    const RopePair p = t.pairs[i - tok * t.npairs];
    const double turns = static_cast<double>(a.pos[p.axis * a.tokens + tok0 + tok]) * p.turns;
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();
  if constexpr (UNIT == kUnitOne) {  // heads whose parts are no vectors: element by element
    for (int u = u0; u < g.units; u += g.width) {
      const bool turns = u < g.turn_units;
      const int i0 = turns ? t.pairs[u].e0 : t.rot + u - g.turn_units, i1 = turns ? t.pairs[u].e1 : i0;
      for (int tok = first, h = h0; tok < ntok; advance(&tok, &h)) {
        const T* in = source(tok, h);
        T* out = target(tok, h);
        if (!turns) {
          out[i0] = in[i0];
          continue;
        }
        const float2 c = cs[tok * t.npairs + u];
        const float x = to_f(in[i0]), y = to_f(in[i1]);
        from_f(x * c.x - y * c.y, out + i0);
        from_f(x * c.y + y * c.x, out + i1);
      }
    }
  } else {
    float2 c[kPairs];
    int have = -1;  // the token that c is of
    for (int tok = first, h = h0, at = 0; tok < ntok; advance(&tok, &h), at = (at + 1) % kRopeDepth) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRopeDepth - 1) : "memory");
      uint4 v[kVecs];
#pragma unroll
      for (int i = 0; i < kVecs; ++i) v[i] = ring[(at * kVecs + i) * kRopeThreads];
      issue(at);
      T* out = target(tok, h);
      if (turn) {
        if (tok != have) {
#pragma unroll
          for (int j = 0; j < kPairs; ++j) c[j] = cs[tok * t.npairs + u0 * kPairs + j];
          have = tok;
        }
        T2* pa = reinterpret_cast<T2*>(v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = unpack(pa[j]);
          if constexpr (UNIT == kUnitPairs) {
            pack(make_float2(x.x * c[j].x - x.y * c[j].y, x.x * c[j].y + x.y * c[j].x), pa + j);
          } else {
            const float2 c0 = c[2 * j], c1 = c[2 * j + 1], y = unpack(pa[4 + j]);
            pack(make_float2(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y), pa + j);
            pack(make_float2(x.x * c0.y + y.x * c0.x, x.y * c1.y + y.y * c1.x), pa + 4 + j);
          }
        }
        if constexpr (UNIT == kUnitHalves) *reinterpret_cast<uint4*>(out + e1) = v[1];
      }
      *reinterpret_cast<uint4*>(out + e0) = v[0];
    }
  }
}

template <typename T, int UNIT>
cudaError_t launch(const RopeTable& t, const RopeArgs& a, int num_sms, cudaStream_t s) {
  const int tail = t.head_dim - t.rot, all = a.heads[0] + a.heads[1];
  RopeGrid g;
  g.turn_units = UNIT == kUnitPairs ? t.rot / 8 : (UNIT == kUnitHalves ? t.npairs / 8 : t.npairs);
  g.units = g.turn_units + (UNIT == kUnitOne ? tail : tail / 8);
  g.width = std::min(g.units, kRopeThreads);
  // Neighbouring threads on neighbouring heads, up to 1 KB of a token.
  g.heads = std::min({std::max(1, 64 / g.width), all, kRopeThreads / g.width});
  g.tokens = kRopeThreads / (g.width * g.heads);
  // Several passes' tokens to a block while that leaves every SM some blocks.
  const int most = std::clamp(kRopeTableBytes / static_cast<int>(t.npairs * sizeof(float2)), 1, 256);
  const long long spread = a.tokens / (num_sms * 16LL);
  const long long passes = std::min<long long>(spread, most) / g.tokens;
  g.tok_per_block = static_cast<int>(passes > 0 ? passes * g.tokens : std::clamp<long long>(spread, 1, most));
  const long long blocks = (a.tokens + g.tok_per_block - 1) / g.tok_per_block;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  constexpr int kRing = UNIT == kUnitOne ? 0 : kRopeDepth * (UNIT == kUnitHalves ? 2 : 1) * kRopeThreads * 16;
  auto fn = rope_kernel<T, UNIT>;
  static AttrOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(fn), kRing + kRopeTableBytes + 4096);
  if (e != cudaSuccess) return e;
  fn<<<static_cast<unsigned>(blocks), kRopeThreads, kRing + g.tok_per_block * t.npairs * sizeof(float2), s>>>(t, a, g);
  return cudaGetLastError();
}

template <typename T>
cudaError_t by_unit(const RopeTable& t, const RopeArgs& a, int num_sms, cudaStream_t s) {
  // 16-byte units where the rotated part, the tail and every address allow them.
  uintptr_t bits = static_cast<uintptr_t>(t.rot | t.head_dim) * 2;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] <= 0) continue;
    bits |= reinterpret_cast<uintptr_t>(a.in[w]) | reinterpret_cast<uintptr_t>(a.out[w]);
    bits |= static_cast<uintptr_t>((a.in_tok[w] | a.out_tok[w]) * 2);
    if (a.heads[w] > 1) bits |= static_cast<uintptr_t>((a.in_head[w] | a.out_head[w]) * 2);
  }
  if (bits % 16 == 0) {
    if (t.layout == kRopePairs) return launch<T, kUnitPairs>(t, a, num_sms, s);
    if (t.halves8) return launch<T, kUnitHalves>(t, a, num_sms, s);
  }
  return launch<T, kUnitOne>(t, a, num_sms, s);
}

}  // namespace

cudaError_t rope_launch(const RopeTable& t, const RopeArgs& a, int dtype, int num_sms, cudaStream_t s) {
  if (a.tokens <= 0 || a.heads[0] + a.heads[1] <= 0) return cudaSuccess;
  return dtype == kTokenBf16 ? by_unit<__nv_bfloat16>(t, a, num_sms, s) : by_unit<__half>(t, a, num_sms, s);
}

}  // namespace ah
