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

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ah {

namespace {

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* p, float (&f)[V]) {
  const Vec<T, V> u = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = to_f<T>(u.e[i]);
}

template <typename T, int V>
__device__ __forceinline__ void store(T* p, const float (&f)[V]) {
  Vec<T, V> u;
#pragma unroll
  for (int i = 0; i < V; ++i) u.e[i] = from_f<T>(f[i]);
  *reinterpret_cast<Vec<T, V>*>(p) = u;
}

__device__ __forceinline__ float gate_act(float g, int act) {
  if (act == kGateTanh) return tanhf(g);
  if (act == kGateLinear) return g;
  const float s = __fdividef(1.f, 1.f + __expf(-g));  // a few fp32 ulp, 0 for very negative g
  return act == kGateSilu ? (s == 0.f ? s : g * s) : s;
}

// Sum over the L lanes of a row (L <= 32), or over the block (L = 0, `red` of 32 floats).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = (L ? L : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (L == 0) {
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v += red[i];
  }
  return v;
}

// L lanes per row (0: the whole block), N vectors of V elements per lane. Channel of vector
// n of lane l: (n * lanes + l) * V.
template <typename T, int V, int L, int N>
__global__ void __launch_bounds__(L ? 256 : 1024) norm_kernel(const NormArgs a) {
  __shared__ float red[32];
  const int lanes = L ? L : blockDim.x;
  const int lane = threadIdx.x % lanes;
  const long long per_block = blockDim.x / lanes;
  const float inv_c = 1.f / static_cast<float>(a.C);
  const T* x = static_cast<const T*>(a.x);
  const T* y = static_cast<const T*>(a.y);
  const T* gate = static_cast<const T*>(a.gate);
  const T* mscale = static_cast<const T*>(a.mscale);
  const T* mshift = static_cast<const T*>(a.mshift);
  T* out = static_cast<T*>(a.out);
  T* norm = static_cast<T*>(a.norm);

  for (long long row0 = blockIdx.x * per_block; row0 < a.rows; row0 += gridDim.x * per_block) {
    const long long row = row0 + threadIdx.x / lanes;
    const bool live = row < a.rows;  // the lanes of a row past the end take part in the shuffles only
    float r[N][V];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * V;
      if (live && c < a.C)
        load<T, V>(x + row * a.xs + c, r[n]);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] = 0.f;
    }
    if (y) {
      float b[N][V];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + lane) * V;
        if (live && c < a.C)
          load<T, V>(y + row * a.ys + c, b[n]);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) b[n][i] = 0.f;
      }
      float mean = 0.f, rstd = 1.f;
      if (a.post == kNormLayer) {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int i = 0; i < V; ++i) s += b[n][i];
        mean = row_sum<L>(s, red) * inv_c;
      }
      if (a.post != kNormNone) {
        float s = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
          if ((n * lanes + lane) * V < a.C)
#pragma unroll
            for (int i = 0; i < V; ++i) s += (b[n][i] - mean) * (b[n][i] - mean);
        rstd = rsqrtf(row_sum<L>(s, red) * inv_c + a.post_eps);
      }
      const T* grow = gate && live ? gate + row / a.rows_per_gate * a.gs : nullptr;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + lane) * V;
        if (!live || c >= a.C) continue;
        float g[V];
        if (grow) {
          load<T, V>(grow + c, g);
#pragma unroll
          for (int i = 0; i < V; ++i) g[i] = gate_act(g[i], a.act);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = (b[n][i] - mean) * rstd;
          if (a.a) v *= __ldg(a.a + c + i);
          if (a.b) v += __ldg(a.b + c + i);
          r[n][i] += grow ? g[i] * v : v;
        }
      }
    }
    if (out && live) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + lane) * V;
        if (c < a.C) store<T, V>(out + row * a.os + c, r[n]);
      }
    }
    if (!norm) continue;
    float mean = 0.f, rstd = 1.f;
    if (a.pre == kNormLayer) {
      float s = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) s += r[n][i];
      mean = row_sum<L>(s, red) * inv_c;
    }
    if (a.pre != kNormNone) {
      float s = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if ((n * lanes + lane) * V < a.C)
#pragma unroll
          for (int i = 0; i < V; ++i) s += (r[n][i] - mean) * (r[n][i] - mean);
      rstd = rsqrtf(row_sum<L>(s, red) * inv_c + a.pre_eps);
    }
    const long long mrow = live ? row / a.rows_per_mod * a.ms : 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = (n * lanes + lane) * V;
      if (!live || c >= a.C) continue;
      float m[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = (r[n][i] - mean) * rstd;
        if (a.w) v *= __ldg(a.w + c + i);
        if (a.wb) v += __ldg(a.wb + c + i);
        r[n][i] = v;
      }
      if (mscale) {
        load<T, V>(mscale + mrow + c, m);
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += r[n][i] * m[i];
      }
      if (mshift) {
        load<T, V>(mshift + mrow + c, m);
#pragma unroll
        for (int i = 0; i < V; ++i) r[n][i] += m[i];
      }
      store<T, V>(norm + row * a.ns + c, r[n]);
    }
  }
}

template <typename T, int V, int L, int N>
cudaError_t launch(const NormArgs& a, int threads, int num_sms, cudaStream_t s) {
  const long long per_block = L ? threads / L : 1;
  const long long blocks = std::min<long long>((a.rows + per_block - 1) / per_block, num_sms * (L ? 8LL : 4LL));
  norm_kernel<T, V, L, N><<<static_cast<unsigned>(blocks), threads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t by_width(const NormArgs& a, int num_sms, cudaStream_t s) {
  const int n = (a.C + V - 1) / V;  // vectors in a row
  if (n <= 8) return launch<T, V, 8, 1>(a, 256, num_sms, s);
  if (n <= 16) return launch<T, V, 16, 1>(a, 256, num_sms, s);
  if (n <= 32) return launch<T, V, 32, 1>(a, 256, num_sms, s);
  if (n <= 64) return launch<T, V, 32, 2>(a, 256, num_sms, s);
  if (n <= 128) return launch<T, V, 32, 4>(a, 256, num_sms, s);
  if (n <= 1024) return launch<T, V, 0, 1>(a, (n + 31) / 32 * 32, num_sms, s);
  if constexpr (V < 8) {  // n is at most 8192 / V
    if (n <= 2048) return launch<T, V, 0, 2>(a, 1024, num_sms, s);
    return launch<T, V, 0, 8>(a, 1024, num_sms, s);
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
