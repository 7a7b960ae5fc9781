// Rotary positions over several axes: the pair (a, b) of a head that belongs to axis s turns
// by pos[s] * frequency,
//
//   (a cos - b sin, a sin + b cos).
//
// The angle is counted in turns: position * (frequency / 2 pi) in fp64, minus the nearest
// whole number, so that a far position loses nothing before it is rounded to fp32. One block
// takes a few tokens, puts their cosines and sines in shared memory once and applies them to
// every head of q and k, in memory order.
//
// Bound: HBM, 4 bytes per element (read, write).
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

template <typename T, int UNIT>
__global__ void __launch_bounds__(kRopeThreads)
    rope_kernel(const RopeTable t, const RopeArgs a, int tok_per_block, int turn_units, int units) {
  extern __shared__ float2 cs[];  // [token][pair]
  using T2 = typename Two<T>::type;
  const long long tok0 = static_cast<long long>(blockIdx.x) * tok_per_block;
  const int ntok = static_cast<int>(min(static_cast<long long>(tok_per_block), a.tokens - tok0));
  for (int i = threadIdx.x; i < ntok * t.npairs; i += kRopeThreads) {
    const int tok = i / t.npairs;
    const RopePair p = t.pairs[i - tok * t.npairs];
    const double turns = static_cast<double>(a.pos[p.axis * a.tokens + tok0 + tok]) * p.turns;
    float s, c;
    sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();
  const int heads = a.heads[0] + a.heads[1];
  const int per_tok = heads * units;
  for (int i = threadIdx.x; i < ntok * per_tok; i += kRopeThreads) {
    const int tok = i / per_tok;
    const int rem = i - tok * per_tok;
    int h = rem / units;
    const int u = rem - h * units;
    const int w = h >= a.heads[0];
    if (w) h -= a.heads[0];
    const T* in = static_cast<const T*>(a.in[w]) + (tok0 + tok) * a.in_tok[w] + h * a.in_head[w];
    T* out = static_cast<T*>(a.out[w]) + (tok0 + tok) * a.out_tok[w] + h * a.out_head[w];
    const float2* tcs = cs + tok * t.npairs;
    if (u >= turn_units) {  // behind the rotated part
      if constexpr (UNIT == kUnitOne) {
        const int e = t.rot + u - turn_units;
        out[e] = in[e];
      } else {
        const int e = t.rot + (u - turn_units) * 8;
        *reinterpret_cast<uint4*>(out + e) = *reinterpret_cast<const uint4*>(in + e);
      }
      continue;
    }
    if constexpr (UNIT == kUnitPairs) {
      uint4 v = *reinterpret_cast<const uint4*>(in + u * 8);
      T2* p = reinterpret_cast<T2*>(&v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 c = tcs[u * 4 + j], x = unpack(p[j]);
        pack(make_float2(x.x * c.x - x.y * c.y, x.x * c.y + x.y * c.x), p + j);
      }
      *reinterpret_cast<uint4*>(out + u * 8) = v;
    } else if constexpr (UNIT == kUnitHalves) {
      const int e0 = t.pairs[u * 8].e0, e1 = t.pairs[u * 8].e1;
      uint4 va = *reinterpret_cast<const uint4*>(in + e0);
      uint4 vb = *reinterpret_cast<const uint4*>(in + e1);
      T2* pa = reinterpret_cast<T2*>(&va);
      T2* pb = reinterpret_cast<T2*>(&vb);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 c0 = tcs[u * 8 + 2 * j], c1 = tcs[u * 8 + 2 * j + 1];
        const float2 x = unpack(pa[j]), y = unpack(pb[j]);
        pack(make_float2(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y), pa + j);
        pack(make_float2(x.x * c0.y + y.x * c0.x, x.y * c1.y + y.y * c1.x), pb + j);
      }
      *reinterpret_cast<uint4*>(out + e0) = va;
      *reinterpret_cast<uint4*>(out + e1) = vb;
    } else {
      const int e0 = t.pairs[u].e0, e1 = t.pairs[u].e1;
      const float2 c = tcs[u];
      const float x = to_f(in[e0]), y = to_f(in[e1]);
      from_f(x * c.x - y * c.y, out + e0);
      from_f(x * c.y + y * c.x, out + e1);
    }
  }
}

template <typename T, int UNIT>
cudaError_t launch(const RopeTable& t, const RopeArgs& a, int num_sms, cudaStream_t s) {
  const int tail = t.head_dim - t.rot;
  const int turn_units = UNIT == kUnitPairs ? t.rot / 8 : (UNIT == kUnitHalves ? t.npairs / 8 : t.npairs);
  const int units = turn_units + (UNIT == kUnitOne ? tail : tail / 8);
  const int most = std::clamp(kRopeTableBytes / static_cast<int>(t.npairs * sizeof(float2)), 1, 256);
  const long long spread = a.tokens / (num_sms * 4LL);
  const int tpb = static_cast<int>(std::min<long long>(most, std::max<long long>(1, spread)));
  const long long blocks = (a.tokens + tpb - 1) / tpb;
  if (blocks > 0x7fffffffLL) return cudaErrorInvalidValue;
  rope_kernel<T, UNIT><<<static_cast<unsigned>(blocks), kRopeThreads, tpb * t.npairs * sizeof(float2), s>>>(
      t, a, tpb, turn_units, units);
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
