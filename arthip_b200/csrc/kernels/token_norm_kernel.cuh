// The norms around a block, its gate and its residual scale in one pass over the rows:
//
//   b    = post(y) * A[c] (+ B[c])        post: none, RMS or layer norm; A holds the norm's
//                                         weight times layer scale times residual scale
//   out  = x + act(gate) * b
//   norm = pre(out) * w[c] (+ wb[c]),     then * (1 + mscale) + mshift
//
// Everything is fp32 in registers from load to store. Both norms read unrounded values: the
// pre-norm's statistics are those of the fp32 sum, not of the fp16 / bf16 row written out.
// A layer norm takes its variance from the centred values in a second sweep over the
// registers, so that loses nothing to cancellation. Its values are v * mul + add, add being
// -mean * mul, and the mean is an fp32 sum: they are off by a few 2^-24 |mean| / sigma.
//
// Bound: HBM, 8 bytes per element (y, x in; out, norm out), 10 with a per-token gate. Two
// kernels: rows of whole vectors of 16 or 8 bytes (2073600 rows of 64: 178 to 196 us, 93 to 84%
// of the copy rate), and rows of any width, stride or alignment, which pass through shared memory in
// 16-byte pieces all the same (64 Mi elements in rows of 91: loaded element by element 951 us, this
// way 145 us, 57% of the copy rate, bound by the instructions per element; with a gate and a
// modulation per group, which are read element by element, 218 us). Above 512 channels several
// warps share a row there and meet at two barriers a sum: 1026 channels 376 us, 5002 353 us,
// 20 to 31% of the copy rate.
#pragma once

#include "token_common.cuh"
#include "token_norm_shape.h"
#include "tokens.h"

#include <algorithm>
#include <atomic>

namespace ah {
namespace token_norm {

// Vectors of 4 or 8 elements.
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  static_assert(V % 4 == 0, "weights are read four at a time");
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& u, float (&f)[V]) {
  const auto* p = reinterpret_cast<const typename Two<T>::type*>(&u);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 t = to_f2(p[i]);
    f[2 * i] = t.x, f[2 * i + 1] = t.y;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> u;
  auto* q = reinterpret_cast<typename Two<T>::type*>(&u);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) from_f2(f[2 * i], f[2 * i + 1], q + i);
  *reinterpret_cast<Vec<T, V>*>(p) = u;
}

// V floats of a weight array, 16 bytes at a time, or `fill` without one.
template <int V>
__device__ __forceinline__ void load_weight(const float* p, int c, float fill, float (&f)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = fill;
    return;
  }
  p += c;
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
    f[i] = u.x, f[i + 1] = u.y, f[i + 2] = u.z, f[i + 3] = u.w;
  }
}

__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == kGateTanh) return tanhf(g);
  if (act == kGateLinear) return g;
  // __expf is off by up to 2 + 1.16 |g| units in the last place: at the largest |g| that leaves
  // anything, 88, 2^-16 of the result, far below the step of 16-bit tensors. 0 for very negative g.
  const float s = __fdividef(1.f, 1.f + __expf(-g));
  return act == kGateSilu ? (s == 0.f ? s : g * s) : s;
}

// Sum over the L lanes of a warp that hold a row, or (L = 0) over `warps` whole warps that meet
// at the named barrier `bar` and leave their sums in `red`.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red, int warps, int bar) {
#pragma unroll
  for (int o = (L ? L : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (L == 0) {
    const int w = (threadIdx.x >> 5) % warps;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");  // the last sum has been read
    if ((threadIdx.x & 31) == 0) red[w] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
    v = 0.f;
    for (int i = 0; i < warps; ++i) v += red[i];
  }
  return v;
}

// Of a lane's share of a row, E values of which in(e) lie in the row (the others are zeros):
// v -> (v - mean) * rstd as v * mul + add. Four running sums, so that additions overlap.
template <int L, int E, typename In>
__device__ __forceinline__ void statistics(const float (&f)[E], In in, int kind, float eps, float inv_c, float* red,
                                           int warps, int bar, float* mul, float* add) {
  *mul = 1.f, *add = 0.f;
  if (kind == kNormNone) return;
  float mean = 0.f;
  if (kind == kNormLayer) {
    float s[4] = {};
#pragma unroll
    for (int e = 0; e < E; ++e) s[e & 3] += f[e];
    mean = row_sum<L>((s[0] + s[1]) + (s[2] + s[3]), red, warps, bar) * inv_c;
  }
  float s[4] = {};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float d = f[e] - mean;
    if (in(e)) s[e & 3] += d * d;
  }
  *mul = rsqrtf(row_sum<L>((s[0] + s[1]) + (s[2] + s[3]), red, warps, bar) * inv_c + eps);
  *add = -mean * *mul;
}

// ---------------------------------------------------------------------------
// Rows of vectors of 16 or 8 bytes
// ---------------------------------------------------------------------------
template <int V, int E>
__device__ __forceinline__ float (&part(float (&f)[E], int n))[V] {
  return *reinterpret_cast<float(*)[V]>(f + n * V);
}

// A row is held by L lanes of a warp, or (L = 0) by `row_warps` whole warps, N vectors per
// lane: vector n of lane l starts at channel (n * lanes + l) * kV. Each group of lanes walks
// over rows. The next row's loads are issued before this row is worked on, so that memory is not
// idle behind the sums that a row waits for, as asynchronous copies into the lane's own places
// in shared memory: no thread waits for another, and they cost no registers (held in registers
// instead, 1280 channels ran at 60% of the copy rate, this way at 77%).
template <typename T, int kV, int L, int N, int THREADS>
__global__ void __launch_bounds__(THREADS) norm_kernel(const NormArgs a, int row_warps) {
  extern __shared__ __align__(16) uint8_t smem[];  // [2 rows][x, y, per-token gate][N][threads] vectors
  __shared__ float red_all[32];
  const int lanes = L ? L : row_warps * 32;
  const int lane = threadIdx.x % lanes, group = threadIdx.x / lanes;
  float* red = red_all + (L ? 0 : group * row_warps);
  const int bar = 1 + (L ? 0 : group);
  const int groups = blockDim.x / lanes;
  const long long step = static_cast<long long>(gridDim.x) * groups;
  const float inv_c = 1.f / static_cast<float>(a.C);
  const T* x = static_cast<const T*>(a.x);
  const T* y = static_cast<const T*>(a.y);
  const T* gate = static_cast<const T*>(a.gate);

  bool in[N];
#pragma unroll
  for (int n = 0; n < N; ++n) in[n] = (n * lanes + lane) * kV < a.C;
  auto held = [&](int e) { return in[e / kV]; };
  float ka[kV], kw[kV];
  if constexpr (N == 1) {
    load_weight<kV>(a.a, in[0] ? lane * kV : 0, 1.f, ka);
    load_weight<kV>(a.w, in[0] ? lane * kV : 0, 1.f, kw);
  }

  const bool row_gate = gate && a.rows_per_gate == 1;
  const int streams = row_gate ? 3 : 2;
  auto place = [&](int buf, int stream, int n) {
    return reinterpret_cast<Vec<T, kV>*>(smem) + ((buf * streams + stream) * N + n) * THREADS + threadIdx.x;
  };
  auto fetch = [&](long long row, int buf) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * kV;
      if (!in[n]) continue;
      copy_async<kV * 2>(place(buf, 0, n), x + row * a.xs + c);
      if (y) copy_async<kV * 2>(place(buf, 1, n), y + row * a.ys + c);
      if (row_gate) copy_async<kV * 2>(place(buf, 2, n), gate + row * a.gs + c);
    }
  };
  // All lanes of a warp take as many steps as its first group, for the shuffles: a group
  // whose row lies past the end works on an old row (or zeros) and stores nothing.
  long long row = static_cast<long long>(blockIdx.x) * groups + group;
  long long row0 = L ? static_cast<long long>(blockIdx.x) * groups + (threadIdx.x & ~31) / lanes : row;
  if (row < a.rows) fetch(row, 0);
  copies_commit();
  for (int buf = 0; row0 < a.rows; row += step, row0 += step, buf ^= 1) {
    const bool live = row < a.rows;
    if (row + step < a.rows) fetch(row + step, buf ^ 1);
    copies_commit();
    copies_wait<1>();
    float r[N * kV], mul, add;  // y (without one, x), then the sum
#pragma unroll
    for (int n = 0; n < N; ++n) {
      float(&f)[kV] = part<kV>(r, n);
#pragma unroll
      for (int i = 0; i < kV; ++i) f[i] = 0.f;
      if (in[n]) unpack<T, kV>(*place(buf, y ? 1 : 0, n), f);
    }
    if (y) {
      const T* grow = nullptr;
      if (gate && !row_gate && live) grow = gate + row / a.rows_per_gate * a.gs;
      statistics<L, N * kV>(r, held, a.post, a.post_eps, inv_c, red, row_warps, bar, &mul, &add);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + lane) * kV;
        if (!in[n]) continue;
        float(&f)[kV] = part<kV>(r, n);
        float xf[kV];
        unpack<T, kV>(*place(buf, 0, n), xf);
        if constexpr (N > 1) load_weight<kV>(a.a, c, 1.f, ka);
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] = (f[i] * mul + add) * ka[i];
        if (a.b) {
          float kb[kV];
          load_weight<kV>(a.b, c, 0.f, kb);
#pragma unroll
          for (int i = 0; i < kV; ++i) f[i] += kb[i];
        }
        if (grow || row_gate) {
          float g[kV];
          unpack<T, kV>(row_gate ? *place(buf, 2, n) : load<T, kV>(grow + c), g);
          if (a.act != kGateLinear) {
#pragma unroll
            for (int i = 0; i < kV; ++i) g[i] = gate_act(g[i], a.act);
          }
#pragma unroll
          for (int i = 0; i < kV; ++i) f[i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] += xf[i];
      }
    }
    if (a.out && live) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (in[n]) store<T, kV>(static_cast<T*>(a.out) + row * a.os + (n * lanes + lane) * kV, part<kV>(r, n));
    }
    if (!a.norm) continue;
    statistics<L, N * kV>(r, held, a.pre, a.pre_eps, inv_c, red, row_warps, bar, &mul, &add);
    if (!live) continue;
    const long long mrow = (a.mscale || a.mshift) ? row / a.rows_per_mod * a.ms : 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * kV;
      if (!in[n]) continue;
      float(&f)[kV] = part<kV>(r, n);
      if constexpr (N > 1) load_weight<kV>(a.w, c, 1.f, kw);
#pragma unroll
      for (int i = 0; i < kV; ++i) f[i] = (f[i] * mul + add) * kw[i];
      if (a.wb) {
        float kb[kV];
        load_weight<kV>(a.wb, c, 0.f, kb);
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] += kb[i];
      }
      float m[kV];
      if (a.mscale) {
        unpack<T, kV>(load<T, kV>(static_cast<const T*>(a.mscale) + mrow + c), m);
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] += f[i] * m[i];
      }
      if (a.mshift) {
        unpack<T, kV>(load<T, kV>(static_cast<const T*>(a.mshift) + mrow + c), m);
#pragma unroll
        for (int i = 0; i < kV; ++i) f[i] += m[i];
      }
      store<T, kV>(static_cast<T*>(a.norm) + row * a.ns + c, f);
    }
  }
}

// As many blocks as fit at once (the same on every sm_100 GPU), each walking over its work.
template <typename F>
cudaError_t resident_blocks(F fn, int threads, size_t smem, int num_sms, std::atomic<int>* known, long long* blocks) {
  int per_sm = known->load(std::memory_order_relaxed);
  if (per_sm == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, threads, smem);
    if (e != cudaSuccess) return e;
    known->store(per_sm, std::memory_order_relaxed);
  }
  *blocks = static_cast<long long>(num_sms) * per_sm;
  return cudaSuccess;
}

template <typename T, int kV, int L, int N, int THREADS>
cudaError_t launch(const NormArgs& a, int row_warps, int num_sms, cudaStream_t s) {
  auto fn = norm_kernel<T, kV, L, N, THREADS>;
  static std::atomic<int> known[32];  // by row_warps (at most 8), and 16 on with a per-token gate
  const int groups = THREADS / (L ? L : row_warps * 32);
  long long most;
  const bool row_gate = a.gate && a.rows_per_gate == 1;
  constexpr int kStream = 2 * N * THREADS * kV * 2;
  const int smem = (row_gate ? 3 : 2) * kStream;
  static AttrOnce once;
  cudaError_t e = once.set(reinterpret_cast<const void*>(fn), 3 * kStream);
  if (e == cudaSuccess) e = resident_blocks(fn, THREADS, smem, num_sms, known + row_warps + 16 * row_gate, &most);
  if (e != cudaSuccess) return e;
  const long long blocks = std::min<long long>((a.rows + groups - 1) / groups, most);
  fn<<<static_cast<unsigned>(blocks), THREADS, smem, s>>>(a, row_warps);
  return cudaGetLastError();
}

// Two or three vectors a lane where the width allows, so that a row's fixed work is shared by
// few lanes (64 channels on eight lanes of one vector: 80% of the copy rate, on four of two:
// 93%); a warp to a row while that holds it, as sums across warps cost two barriers each.
template <typename T, int V>
cudaError_t by_width(const NormArgs& a, int num_sms, cudaStream_t s) {
  const int n = a.C / V;  // vectors in a row
  if (n <= 4) return launch<T, V, 4, 1, 256>(a, 1, num_sms, s);
  if (n <= 8) return launch<T, V, 4, 2, 256>(a, 1, num_sms, s);
  if (n <= 12) return launch<T, V, 4, 3, 256>(a, 1, num_sms, s);
  if (n <= 16) return launch<T, V, 8, 2, 256>(a, 1, num_sms, s);
  if (n <= 24) return launch<T, V, 8, 3, 256>(a, 1, num_sms, s);
  if (n <= 32) return launch<T, V, 16, 2, 256>(a, 1, num_sms, s);
  if (n <= 48) return launch<T, V, 16, 3, 256>(a, 1, num_sms, s);
  if (n <= 64) return launch<T, V, 32, 2, 256>(a, 1, num_sms, s);
  if (n <= 96) return launch<T, V, 32, 3, 128>(a, 1, num_sms, s);
  if (n <= 128) return launch<T, V, 32, 4, 128>(a, 1, num_sms, s);
  if (n <= 160) return launch<T, V, 32, 5, 128>(a, 1, num_sms, s);
  if (n <= 192) return launch<T, V, 32, 6, 128>(a, 1, num_sms, s);
  if (n <= 256) return launch<T, V, 0, 4, 128>(a, 2, num_sms, s);
  if (n <= 384) return launch<T, V, 0, 6, 128>(a, 2, num_sms, s);
  if (n <= 512) return launch<T, V, 0, 4, 128>(a, 4, num_sms, s);
  if (n <= 768) return launch<T, V, 0, 6, 128>(a, 4, num_sms, s);
  if (n <= 1024) return launch<T, V, 0, 4, 256>(a, 8, num_sms, s);
  // n is at most 8192 / V
  if constexpr (V < 8) return launch<T, V, 0, 8, 256>(a, 8, num_sms, s);
  return cudaErrorInvalidValue;
}

// ---------------------------------------------------------------------------
// Any rows, through shared memory
// ---------------------------------------------------------------------------
// A group of GROUP threads (a warp, or the block for wide rows) takes a tile of some rows: their
// elements come into shared memory by asynchronous 16-byte copies, one tile ahead, the elements
// before the first and behind the last 16-byte boundary one by one; the results leave the same
// way. LANES lanes share a row (a warp has 32 / LANES at once), element e being lane e % LANES'.
// A lane's N channels are the same in every row, and their weights stay in registers. N is even
// and at most one more than a lane needs (staged_shape), so that only its last two elements are
// ever in question (with a test for each, 90 channels took 85 instructions an element).
template <int GROUP>
__device__ __forceinline__ void group_sync() {
  if constexpr (GROUP == 32)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / GROUP), "n"(GROUP) : "memory");
}

struct Tiles {
  int rows = 1;         // of a tile
  int slot = 0;         // bytes of one stream's tile in shared memory
  int streams = 2;      // x, y and a per-token gate
  long long count = 0;
};

template <typename T, int GROUP, int LANES, int N>
__global__ void __launch_bounds__(256, N <= 8 ? 3 : (N <= 16 ? 2 : 1)) norm_staged_kernel(const NormArgs a, const Tiles tiles) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red_all[8];
  constexpr int L = GROUP == 32 ? LANES : 0;  // LANES is GROUP when that is more than a warp
  constexpr int kRows = GROUP / LANES;        // at once
  const int t = threadIdx.x % GROUP, lane = t % LANES, group = threadIdx.x / GROUP;
  float* red = red_all + (L ? 0 : group * (GROUP / 32));
  const int bar = 1 + group;
  const int groups = 256 / GROUP;
  const int slots = 2 * tiles.streams + 2;
  uint8_t* base = smem + static_cast<size_t>(group) * slots * tiles.slot;
  uint8_t* s_out = base + 2 * tiles.streams * tiles.slot;
  uint8_t* s_norm = s_out + tiles.slot;
  const float inv_c = 1.f / static_cast<float>(a.C);
  const T* x = static_cast<const T*>(a.x);
  const T* y = static_cast<const T*>(a.y);
  const T* gate = static_cast<const T*>(a.gate);
  const bool row_gate = gate && a.rows_per_gate == 1;
  const bool in0 = (N - 2) * LANES + lane < a.C, in1 = (N - 1) * LANES + lane < a.C;
  auto in = [&](int k) { return k < N - 2 || (k == N - 2 ? in0 : in1); };
  float ka[N], kw[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    ka[k] = a.a && in(k) ? a.a[lane + k * LANES] : 1.f;
    kw[k] = a.w && in(k) ? a.w[lane + k * LANES] : 1.f;
  }
  auto offset = [](const void* p) { return static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16); };
  auto rows_of = [&](long long tile) {
    return static_cast<int>(min(static_cast<long long>(tiles.rows), a.rows - tile * tiles.rows));
  };
  auto fetch = [&](long long tile, int buf) {
    uint8_t* to = base + buf * tiles.streams * tiles.slot;
    const long long row = tile * tiles.rows;
    const int n = (rows_of(tile) - 1) * a.C + a.C;
    copy_in<T, GROUP>(to, x + row * a.xs, n, t);
    if (y) copy_in<T, GROUP>(to + tiles.slot, y + row * a.ys, n, t);
    if (row_gate) copy_in<T, GROUP>(to + 2 * tiles.slot, gate + row * a.gs, n, t);
  };
  const long long step = static_cast<long long>(gridDim.x) * groups;
  long long tile = static_cast<long long>(blockIdx.x) * groups + group;
  if (tile < tiles.count) fetch(tile, 0);
  copies_commit();
  for (int buf = 0; tile < tiles.count; tile += step, buf ^= 1) {
    if (tile + step < tiles.count) fetch(tile + step, buf ^ 1);
    copies_commit();
    copies_wait<1>();
    group_sync<GROUP>();
    const uint8_t* from = base + buf * tiles.streams * tiles.slot;
    const long long row0 = tile * tiles.rows;
    const int n_rows = rows_of(tile);
    const T* sx = reinterpret_cast<const T*>(from + offset(x + row0 * a.xs));
    const T* sy = reinterpret_cast<const T*>(from + tiles.slot + offset(y + row0 * a.ys));
    const T* sg = reinterpret_cast<const T*>(from + 2 * tiles.slot + offset(gate + row0 * a.gs));
    T* out = static_cast<T*>(a.out) + row0 * a.os;
    T* norm = static_cast<T*>(a.norm) + row0 * a.ns;
    T* so = reinterpret_cast<T*>(s_out + offset(out));
    T* sn = reinterpret_cast<T*>(s_norm + offset(norm));
    for (int i0 = 0; i0 < n_rows; i0 += kRows) {  // past the last row its lanes repeat it
      const int i = min(i0 + t / LANES, n_rows - 1);
      const bool mine = i0 + t / LANES < n_rows;
      const long long row = row0 + i;
      const T* xi = sx + i * a.C + lane;
      float r[N], mul, add;
#pragma unroll
      for (int k = 0; k < N; ++k) r[k] = in(k) ? to_f(xi[k * LANES]) : 0.f;
      if (y) {
        const T* yi = sy + i * a.C + lane;
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = in(k) ? to_f(yi[k * LANES]) : 0.f;
        statistics<L, N>(f, in, a.post, a.post_eps, inv_c, red, GROUP / 32, bar, &mul, &add);
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = (f[k] * mul + add) * ka[k];
        if (a.b) {
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (in(k)) f[k] += __ldg(a.b + lane + k * LANES);
        }
        if (gate) {
          const T* gi = (row_gate ? sg + i * a.C : gate + row / a.rows_per_gate * a.gs) + lane;
          float g[N];
#pragma unroll
          for (int k = 0; k < N; ++k) g[k] = in(k) ? to_f(gi[k * LANES]) : 0.f;
          if (a.act != kGateLinear) {
#pragma unroll
            for (int k = 0; k < N; ++k) g[k] = gate_act(g[k], a.act);
          }
#pragma unroll
          for (int k = 0; k < N; ++k) f[k] *= g[k];
        }
#pragma unroll
        for (int k = 0; k < N; ++k) r[k] = in(k) ? r[k] + f[k] : 0.f;
      }
      if (a.out && mine) {
        T* oi = so + i * a.C + lane;
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (in(k)) from_f(r[k], oi + k * LANES);
      }
      if (!a.norm) continue;
      statistics<L, N>(r, in, a.pre, a.pre_eps, inv_c, red, GROUP / 32, bar, &mul, &add);
#pragma unroll
      for (int k = 0; k < N; ++k) r[k] = (r[k] * mul + add) * kw[k];
      if (a.wb) {
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (in(k)) r[k] += __ldg(a.wb + lane + k * LANES);
      }
      if (a.mscale || a.mshift) {
        const long long mrow = row / a.rows_per_mod * a.ms + lane;
        const T* scale = static_cast<const T*>(a.mscale) + mrow;
        const T* shift = static_cast<const T*>(a.mshift) + mrow;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (!in(k)) continue;
          if (a.mscale) r[k] += r[k] * to_f(scale[k * LANES]);
          if (a.mshift) r[k] += to_f(shift[k * LANES]);
        }
      }
      if (!mine) continue;
      T* ni = sn + i * a.C + lane;
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (in(k)) from_f(r[k], ni + k * LANES);
    }
    group_sync<GROUP>();
    if (a.out) copy_out<T, GROUP>(out, s_out, n_rows * a.C, t);
    if (a.norm) copy_out<T, GROUP>(norm, s_norm, n_rows * a.C, t);
    group_sync<GROUP>();  // the results have left, and the inputs may be written over
  }
}

template <typename T, int GROUP, int LANES, int N>
cudaError_t launch_staged(const NormArgs& a, int num_sms, cudaStream_t s) {
  auto fn = norm_staged_kernel<T, GROUP, LANES, N>;
  Tiles tiles;
  auto packed = [&](const void* p, long long stride) { return !p || stride == a.C; };
  const bool row_gate = a.gate && a.rows_per_gate == 1;
  tiles.streams = row_gate ? 3 : 2;
  if (packed(a.x, a.xs) && packed(a.y, a.ys) && packed(a.out, a.os) && packed(a.norm, a.ns) &&
      (!row_gate || a.gs == a.C)) {
    // About 2 KB of each stream, but enough tiles for every warp: rows of other pitch go one by one.
    constexpr int kRows = GROUP / LANES;
    const long long fair = std::max<long long>(kRows, a.rows / (num_sms * 16LL) / kRows * kRows);
    tiles.rows = static_cast<int>(std::clamp<long long>(1024 / a.C / kRows * kRows, kRows, fair));
  }
  tiles.slot = (tiles.rows * a.C * 2 + 15) / 16 * 16 + 16;
  tiles.count = (a.rows + tiles.rows - 1) / tiles.rows;
  const int groups = 256 / GROUP;
  const size_t smem = static_cast<size_t>(groups) * (2 * tiles.streams + 2) * tiles.slot;
  static AttrOnce once;
  cudaError_t e = once.set(reinterpret_cast<const void*>(fn), 200 * 1024);
  if (e != cudaSuccess) return e;
  const int per_sm = static_cast<int>(std::clamp<size_t>(220 * 1024 / (smem + 1024), 1, 8));
  const long long blocks = std::min<long long>((tiles.count + groups - 1) / groups, static_cast<long long>(num_sms) * per_sm);
  fn<<<static_cast<unsigned>(blocks), 256, smem, s>>>(a, tiles);
  return cudaGetLastError();
}

template <typename T>
struct LaunchStaged {
  const NormArgs& a;
  int num_sms;
  cudaStream_t s;
  template <int GROUP, int LANES, int N>
  cudaError_t operator()() const {
    return launch_staged<T, GROUP, LANES, N>(a, num_sms, s);
  }
};

template <typename T>
cudaError_t by_elements(const NormArgs& a, int num_sms, cudaStream_t s) {
  return staged_shape(a.C, LaunchStaged<T>{a, num_sms, s});
}

// One translation unit each (token_norm_*.cu): rows of vectors (of `vec` elements), any rows.
cudaError_t vectors_f16(const NormArgs& a, int vec, int num_sms, cudaStream_t s);
cudaError_t vectors_bf16(const NormArgs& a, int vec, int num_sms, cudaStream_t s);
cudaError_t elements_f16(const NormArgs& a, int num_sms, cudaStream_t s);
cudaError_t elements_bf16(const NormArgs& a, int num_sms, cudaStream_t s);

}  // namespace token_norm
}  // namespace ah
