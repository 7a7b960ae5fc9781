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
// registers, so a large mean costs no digits.
//
// Bound: HBM, 8 bytes per element (y, x in; out, norm out), 10 with a per-token gate.
#include "tokens.h"

#include <algorithm>
#include <atomic>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ah {

namespace {

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void from_f(float v, __half* o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16* o) { *o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f2(float a, float b, __half2* o) { *o = __floats2half2_rn(a, b); }
__device__ __forceinline__ void from_f2(float a, float b, __nv_bfloat162* o) { *o = __floats2bfloat162_rn(a, b); }

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

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void unpack(const Vec<T, V>& u, float (&f)[V]) {
  if constexpr (V % 2 == 0) {
    const auto* p = reinterpret_cast<const typename Two<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 t = to_f2(p[i]);
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  } else {
    f[0] = to_f(u.e[0]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> u;
  if constexpr (V % 2 == 0) {
    auto* q = reinterpret_cast<typename Two<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) from_f2(f[2 * i], f[2 * i + 1], q + i);
  } else {
    from_f(f[0], &u.e[0]);
  }
  *reinterpret_cast<Vec<T, V>*>(p) = u;
}

// V floats of a weight array, 16 bytes at a time where V allows, or `fill` without one.
template <int V>
__device__ __forceinline__ void load_weight(const float* p, int c, float fill, float (&f)[V]) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = fill;
    return;
  }
  p += c;
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
      f[i] = u.x, f[i + 1] = u.y, f[i + 2] = u.z, f[i + 3] = u.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = __ldg(p + i);
  }
}

__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == kGateTanh) return tanhf(g);
  if (act == kGateLinear) return g;
  const float s = __fdividef(1.f, 1.f + __expf(-g));  // a few fp32 ulp, 0 for very negative g
  return act == kGateSilu ? (s == 0.f ? s : g * s) : s;
}

// Sum over a row's lanes: L of one warp, or for L = 0 `warps` whole warps that meet at the
// named barrier `bar` and leave their sums in `red`.
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

// A row is held by L lanes of a warp, or (L = 0) by `row_warps` whole warps, N vectors of V
// elements per lane: vector n of lane l starts at channel (n * lanes + l) * V. Each group of
// lanes walks over rows, and the next row's loads are issued before this row is worked on, so
// that memory is not idle behind the sums that a row waits for. A lane with one vector keeps
// its two weight vectors in registers throughout.
template <typename T, int V, int L, int N, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) norm_kernel(const NormArgs a, int row_warps) {
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
  for (int n = 0; n < N; ++n) in[n] = (n * lanes + lane) * V < a.C;
  float ka[V], kw[V];
  if constexpr (N == 1) {
    load_weight<V>(a.a, in[0] ? lane * V : 0, 1.f, ka);
    load_weight<V>(a.w, in[0] ? lane * V : 0, 1.f, kw);
  }

  Vec<T, V> xn[N] = {}, yn[N] = {};  // the next row, zeros past its end
  auto fetch = [&](long long row) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * V;
      if (!in[n]) continue;
      xn[n] = load<T, V>(x + row * a.xs + c);
      if (y) yn[n] = load<T, V>(y + row * a.ys + c);
    }
  };
  // Of a row's values: v -> (v - mean) * rstd as v * mul + add.
  auto statistics = [&](const float(&f)[N][V], int kind, float eps, float* mul, float* add) {
    float mean = 0.f;
    *mul = 1.f, *add = 0.f;
    if (kind == kNormNone) return;
    if (kind == kNormLayer) {
      float s = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) s += f[n][i];
      mean = row_sum<L>(s, red, row_warps, bar) * inv_c;
    }
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!in[n]) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) s += (f[n][i] - mean) * (f[n][i] - mean);
    }
    *mul = rsqrtf(row_sum<L>(s, red, row_warps, bar) * inv_c + eps);
    *add = -mean * *mul;
  };
  // All lanes of a warp take as many steps as its first group, for the shuffles: a group
  // whose row lies past the end works on an old row (or zeros) and stores nothing.
  long long row = static_cast<long long>(blockIdx.x) * groups + group;
  long long row0 = L ? static_cast<long long>(blockIdx.x) * groups + (threadIdx.x & ~31) / lanes : row;
  if (row < a.rows) fetch(row);
  for (; row0 < a.rows; row += step, row0 += step) {
    const bool live = row < a.rows;
    float r[N][V], b[N][V], mul, add;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      unpack<T, V>(xn[n], r[n]);
      unpack<T, V>(yn[n], b[n]);
    }
    if (row + step < a.rows) fetch(row + step);
    if (y) {
      const T* grow = nullptr;
      if (gate && live) grow = gate + (a.rows_per_gate == 1 ? row : row / a.rows_per_gate) * a.gs;
      statistics(b, a.post, a.post_eps, &mul, &add);
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + lane) * V;
        if (!in[n]) continue;
        if constexpr (N > 1) load_weight<V>(a.a, c, 1.f, ka);
#pragma unroll
        for (int i = 0; i < V; ++i) b[n][i] = (b[n][i] * mul + add) * ka[i];
        if (a.b) {
          float kb[V];
          load_weight<V>(a.b, c, 0.f, kb);
#pragma unroll
          for (int i = 0; i < V; ++i) b[n][i] += kb[i];
        }
        if (grow) {
          float g[V];
          unpack<T, V>(load<T, V>(grow + c), g);
          if (a.act != kGateLinear) {
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = gate_act(g[i], a.act);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) b[n][i] *= g[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += b[n][i];
      }
    }
    if (a.out && live) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (in[n]) store<T, V>(static_cast<T*>(a.out) + row * a.os + (n * lanes + lane) * V, r[n]);
    }
    if (!a.norm) continue;
    statistics(r, a.pre, a.pre_eps, &mul, &add);
    if (!live) continue;
    const long long mrow = (a.mscale || a.mshift) ? row / a.rows_per_mod * a.ms : 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * V;
      if (!in[n]) continue;
      if constexpr (N > 1) load_weight<V>(a.w, c, 1.f, kw);
#pragma unroll
      for (int i = 0; i < V; ++i) r[n][i] = (r[n][i] * mul + add) * kw[i];
      if (a.wb) {
        float kb[V];
        load_weight<V>(a.wb, c, 0.f, kb);
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += kb[i];
      }
      float m[V];
      if (a.mscale) {
        unpack<T, V>(load<T, V>(static_cast<const T*>(a.mscale) + mrow + c), m);
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += r[n][i] * m[i];
      }
      if (a.mshift) {
        unpack<T, V>(load<T, V>(static_cast<const T*>(a.mshift) + mrow + c), m);
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += m[i];
      }
      store<T, V>(static_cast<T*>(a.norm) + row * a.ns + c, r[n]);
    }
  }
}

template <typename T, int V, int L, int N, int THREADS = 256, int BLOCKS = 1>
cudaError_t launch(const NormArgs& a, int row_warps, int num_sms, cudaStream_t s) {
  auto fn = norm_kernel<T, V, L, N, THREADS, BLOCKS>;
  const int groups = THREADS / (L ? L : row_warps * 32);
  const int threads = groups * (L ? L : row_warps * 32);
  // As many blocks as fit at once (the same on every sm_100 GPU), each walking over its rows.
  static std::atomic<int> fit[33];  // by row_warps
  int per_sm = fit[row_warps].load(std::memory_order_relaxed);
  if (per_sm == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, threads, 0);
    if (e != cudaSuccess) return e;
    fit[row_warps].store(per_sm, std::memory_order_relaxed);
  }
  const long long blocks =
      std::min<long long>((a.rows + groups - 1) / groups, static_cast<long long>(num_sms) * per_sm);
  fn<<<static_cast<unsigned>(blocks), threads, 0, s>>>(a, row_warps);
  return cudaGetLastError();
}

// Few vectors a lane: they and the next row's are held in registers, and it is rows in flight
// that hide the wait for memory and for the sums.
template <typename T, int V>
cudaError_t by_width(const NormArgs& a, int num_sms, cudaStream_t s) {
  const int n = (a.C + V - 1) / V;  // vectors in a row
  if (n <= 8) return launch<T, V, 8, 1, 256, 4>(a, 1, num_sms, s);
  if (n <= 16) return launch<T, V, 16, 1, 256, 4>(a, 1, num_sms, s);
  if (n <= 32) return launch<T, V, 32, 1, 256, 4>(a, 1, num_sms, s);
  if (n <= 48) return launch<T, V, 16, 3>(a, 1, num_sms, s);
  if (n <= 64) return launch<T, V, 32, 2>(a, 1, num_sms, s);
  if (n <= 256) return launch<T, V, 0, 1, 256, 4>(a, (n + 31) / 32, num_sms, s);
  if (n <= 512) return launch<T, V, 0, 2, 256, 2>(a, (n + 63) / 64, num_sms, s);
  if (n <= 1024) return launch<T, V, 0, 4>(a, (n + 127) / 128, num_sms, s);
  // n is at most 8192 / V
  if constexpr (V < 8) {
    if (n <= 4096) return launch<T, V, 0, 4, 1024>(a, 32, num_sms, s);
    return launch<T, V, 0, 8, 1024>(a, 32, num_sms, s);
  }
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t by_vector(const NormArgs& a, int num_sms, cudaStream_t s) {
  // The widest load that divides the row and that every pointer and stride is aligned to.
  uintptr_t bits = static_cast<uintptr_t>(a.C) * 2;
  const void* ptrs[] = {a.x, a.y, a.gate, a.mscale, a.mshift, a.out, a.norm};
  const long long strides[] = {a.xs, a.ys, a.gs, a.ms, a.ms, a.os, a.ns};
  for (int i = 0; i < 7; ++i)
    if (ptrs[i]) bits |= reinterpret_cast<uintptr_t>(ptrs[i]) | static_cast<uintptr_t>(strides[i] * 2);
  if (bits % 16 == 0) return by_width<T, 8>(a, num_sms, s);
  if (bits % 4 == 0) return by_width<T, 2>(a, num_sms, s);
  return by_width<T, 1>(a, num_sms, s);
}

}  // namespace

cudaError_t norm_launch(const NormArgs& a, int dtype, int num_sms, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  return dtype == kTokenBf16 ? by_vector<__nv_bfloat16>(a, num_sms, s) : by_vector<__half>(a, num_sms, s);
}

}  // namespace ah
