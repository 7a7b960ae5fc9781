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

namespace ah {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeTableBytes = 16384;  // cosines and sines of a block's tokens

// How a head is cut into the units that one thread turns:
//   kUnitPairs   8 elements, four adjacent pairs
//   kUnitHalves  8 pairs: 8 elements and the 8 elements that turn with them
// Elements behind the rotated part are copied, 8 at a time. Heads that cannot be cut so have a
// kernel of their own, below.
enum Unit : int { kUnitPairs = 0, kUnitHalves = 1 };

// Cosine and sine of a pair at a token's position.
__device__ __forceinline__ float2 turn_of(const RopePair& p, const RopeArgs& a, long long tok) {
  const double turns = static_cast<double>(a.pos[p.axis * a.tokens + tok]) * p.turns;
  float s, c;
  sincospif(2.f * static_cast<float>(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

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
  constexpr int kPairs = UNIT == kUnitPairs ? 4 : 8;
  extern __shared__ __align__(16) uint8_t smem[];
  uint4* ring = reinterpret_cast<uint4*>(smem) + threadIdx.x;  // [depth][vector][thread]
  float2* cs = reinterpret_cast<float2*>(smem + kRopeDepth * kVecs * kRopeThreads * 16);
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
        copy_async<16>(ring + (at * kVecs + v) * kRopeThreads, in + (v ? e1 : e0));
      advance(&next_tok, &next_h);
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < kRopeDepth; ++d) issue(d);
  for (int i = threadIdx.x; i < ntok * t.npairs; i += kRopeThreads) {
    const int tok = i / t.npairs;
    cs[i] = turn_of(t.pairs[i - tok * t.npairs], a, tok0 + tok);
  }
  __syncthreads();
  float2 c[kPairs];
  int have = -1;  // the token that c is of
  for (int tok = first, h = h0, at = 0; tok < ntok; advance(&tok, &h), at = (at + 1) % kRopeDepth) {
    copies_wait<kRopeDepth - 1>();
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
        const float2 x = to_f2(pa[j]);
        if constexpr (UNIT == kUnitPairs) {
          from_f2(x.x * c[j].x - x.y * c[j].y, x.x * c[j].y + x.y * c[j].x, pa + j);
        } else {
          const float2 c0 = c[2 * j], c1 = c[2 * j + 1], y = to_f2(pa[4 + j]);
          from_f2(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y, pa + j);
          from_f2(x.x * c0.y + y.x * c0.x, x.y * c1.y + y.y * c1.x, pa + 4 + j);
        }
      }
      if constexpr (UNIT == kUnitHalves) *reinterpret_cast<uint4*>(out + e1) = v[1];
    }
    *reinterpret_cast<uint4*>(out + e0) = v[0];
  }
}

template <typename T, int UNIT>
cudaError_t launch(const RopeTable& t, const RopeArgs& a, int num_sms, cudaStream_t s) {
  const int tail = t.head_dim - t.rot, all = a.heads[0] + a.heads[1];
  RopeGrid g;
  g.turn_units = UNIT == kUnitPairs ? t.rot / 8 : t.npairs / 8;
  g.units = g.turn_units + tail / 8;
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
  constexpr int kRing = kRopeDepth * (UNIT == kUnitHalves ? 2 : 1) * kRopeThreads * 16;
  auto fn = rope_kernel<T, UNIT>;
  static AttrOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(fn), kRing + kRopeTableBytes + 4096);
  if (e != cudaSuccess) return e;
  fn<<<static_cast<unsigned>(blocks), kRopeThreads, kRing + g.tok_per_block * t.npairs * sizeof(float2), s>>>(t, a, g);
  return cudaGetLastError();
}

// Heads of any cut, width, stride and alignment: a warp takes a run of a token's heads into shared
// memory in 16-byte pieces, one run ahead, turns its pairs there and sends them out the same way.
// A lane's pairs are every 32nd of a head, their cosines and sines in registers for all heads of
// the token. Pairs are turned element by element there, so short heads, which leave lanes without a
// pair, cost most: 48 heads of 128 run at 63% of the copy rate (turned in global memory at 31%), 16
// of 64 in sections of 22, 20 and 22 at 47%, 16 of 30 at 23%.
struct RopeRuns {
  int slot = 0;         // bytes of a run in shared memory
  int heads[2] = {};    // of a run of q, of k
  int runs[2] = {};     // of a token
};

template <typename T, int KP>
__global__ void __launch_bounds__(kRopeThreads) rope_staged_kernel(const RopeTable t, const RopeArgs a,
                                                                   const RopeRuns g) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kWarps = kRopeThreads / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint8_t* mine = smem + warp * 3 * g.slot;  // two runs on their way in, one on its way out
  uint8_t* out_at = mine + 2 * g.slot;
  const int per_tok = g.runs[0] + g.runs[1];
  struct Run {
    const T* in;
    T* out;
    long long in_step, out_step;  // between heads
    int heads;
  };
  auto run_of = [&](long long tok, int r) {
    const bool k = r >= g.runs[0];
    const int each = k ? g.heads[1] : g.heads[0], h = (k ? r - g.runs[0] : r) * each;
    Run x;
    x.in_step = k ? a.in_head[1] : a.in_head[0], x.out_step = k ? a.out_head[1] : a.out_head[0];
    x.in = static_cast<const T*>(k ? a.in[1] : a.in[0]) + tok * (k ? a.in_tok[1] : a.in_tok[0]) + h * x.in_step;
    x.out = static_cast<T*>(k ? a.out[1] : a.out[0]) + tok * (k ? a.out_tok[1] : a.out_tok[0]) + h * x.out_step;
    x.heads = min(each, (k ? a.heads[1] : a.heads[0]) - h);
    return x;
  };
  int e0[KP], e1[KP];
#pragma unroll
  for (int k = 0; k < KP; ++k) {
    const int p = min(lane + 32 * k, t.npairs - 1);
    e0[k] = t.pairs[p].e0, e1[k] = t.pairs[p].e1;
  }
  const long long step = static_cast<long long>(gridDim.x) * kWarps;
  long long tok = static_cast<long long>(blockIdx.x) * kWarps + warp, next_tok = tok;
  int next_r = 0;
  auto fetch = [&](int buf) {
    if (next_tok < a.tokens) {
      const Run x = run_of(next_tok, next_r);
      copy_in<T, 32>(mine + buf * g.slot, x.in, x.heads * t.head_dim, lane);
      if (++next_r == per_tok) next_r = 0, next_tok += step;
    }
    copies_commit();
  };
  fetch(0);
  int buf = 0;
  for (; tok < a.tokens; tok += step) {
    float2 c[KP];
#pragma unroll
    for (int k = 0; k < KP; ++k) c[k] = turn_of(t.pairs[min(lane + 32 * k, t.npairs - 1)], a, tok);
    for (int r = 0; r < per_tok; ++r, buf ^= 1) {
      fetch(buf ^ 1);
      copies_wait<1>();
      __syncwarp();
      const Run x = run_of(tok, r);
      const T* from = reinterpret_cast<const T*>(mine + buf * g.slot + reinterpret_cast<uintptr_t>(x.in) % 16);
      T* to = reinterpret_cast<T*>(out_at + reinterpret_cast<uintptr_t>(x.out) % 16);
      for (int h = 0; h < x.heads; ++h, from += t.head_dim, to += t.head_dim) {
#pragma unroll
        for (int k = 0; k < KP; ++k) {
          if (lane + 32 * k >= t.npairs) continue;
          const float u = to_f(from[e0[k]]), v = to_f(from[e1[k]]);
          from_f(u * c[k].x - v * c[k].y, to + e0[k]);
          from_f(u * c[k].y + v * c[k].x, to + e1[k]);
        }
        for (int e = t.rot + lane; e < t.head_dim; e += 32) to[e] = from[e];
      }
      __syncwarp();
      copy_out<T, 32>(x.out, out_at, x.heads * t.head_dim, lane);
      __syncwarp();  // the results have left, and this run's places may be written over
    }
  }
}

template <typename T, int KP>
cudaError_t launch_staged(const RopeTable& t, const RopeArgs& a, int num_sms, cudaStream_t s) {
  RopeRuns g;
  int most = 0;
  for (int w = 0; w < 2; ++w) {
    if (a.heads[w] == 0) continue;
    // Heads one behind the other make one run, up to 4 KB; others go one by one.
    const bool packed = a.heads[w] == 1 || (a.in_head[w] == t.head_dim && a.out_head[w] == t.head_dim);
    g.heads[w] = packed ? std::clamp(2048 / t.head_dim, 1, a.heads[w]) : 1;
    g.runs[w] = (a.heads[w] + g.heads[w] - 1) / g.heads[w];
    most = std::max(most, g.heads[w]);
  }
  g.slot = (most * t.head_dim * 2 + 15) / 16 * 16 + 16;
  constexpr int kWarps = kRopeThreads / 32;
  const int smem = kWarps * 3 * g.slot;
  auto fn = rope_staged_kernel<T, KP>;
  static AttrOnce once;
  const cudaError_t e = once.set(reinterpret_cast<const void*>(fn), kWarps * 3 * (4096 + 32));
  if (e != cudaSuccess) return e;
  const long long places = static_cast<long long>(num_sms) * std::clamp(220 * 1024 / (smem + 1024), 1, 6);
  const long long blocks = std::min<long long>((a.tokens + kWarps - 1) / kWarps, places);
  fn<<<static_cast<unsigned>(blocks), kRopeThreads, smem, s>>>(t, a, g);
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
  if (t.npairs <= 32) return launch_staged<T, 1>(t, a, num_sms, s);
  if (t.npairs <= 64) return launch_staged<T, 2>(t, a, num_sms, s);
  if (t.npairs <= 128) return launch_staged<T, 4>(t, a, num_sms, s);
  return launch_staged<T, 8>(t, a, num_sms, s);
}

}  // namespace

cudaError_t rope_launch(const RopeTable& t, const RopeArgs& a, int dtype, int num_sms, cudaStream_t s) {
  if (a.tokens <= 0 || a.heads[0] + a.heads[1] <= 0) return cudaSuccess;
  return dtype == kTokenBf16 ? by_unit<__nv_bfloat16>(t, a, num_sms, s) : by_unit<__half>(t, a, num_sms, s);
}

}  // namespace ah
