// extern "C" boundary of the token operators (declarations and contracts in
// include/arthip_b200.h): argument checks, the uploaded parameters of each handle, launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <exception>
#include <initializer_list>
#include <limits>
#include <memory>
#include <string>
#include <vector>

#include "../../include/arthip_b200.h"
#include "kernels/tokens.h"

namespace {

int Fail(const std::string& s, char* dst, int len, int rc = 1) {
  if (dst && len > 0) {
    const size_t n = std::min(s.size(), static_cast<size_t>(len) - 1);
    std::memcpy(dst, s.data(), n);
    dst[n] = '\0';
  }
  return rc;
}

int CudaFail(const char* what, cudaError_t e, char* dst, int len, int rc) {
  (void)cudaGetLastError();
  return Fail(std::string(what) + ": " + cudaGetErrorString(e), dst, len, rc);
}

// Makes `device` current for a call and gives the caller's device back afterwards.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    error_ = cudaGetDevice(&prev_);
    if (error_ == cudaSuccess && prev_ != device) {
      error_ = cudaSetDevice(device);
      changed_ = true;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(prev_);
  }
  cudaError_t error() const { return error_; }

 private:
  int prev_ = 0;
  bool changed_ = false;
  cudaError_t error_ = cudaSuccess;
};

// A handle's device memory.
class DeviceBuffer {
 public:
  DeviceBuffer() = default;
  DeviceBuffer(const DeviceBuffer&) = delete;
  DeviceBuffer& operator=(const DeviceBuffer&) = delete;
  ~DeviceBuffer() {
    if (p_) cudaFree(p_);
  }
  cudaError_t Upload(const void* src, size_t bytes) {
    if (bytes == 0) return cudaSuccess;
    const cudaError_t e = cudaMalloc(&p_, bytes);
    return e == cudaSuccess ? cudaMemcpy(p_, src, bytes, cudaMemcpyHostToDevice) : e;
  }
  template <typename T>
  T* as() const {
    return static_cast<T*>(p_);
  }

 private:
  void* p_ = nullptr;
};

// Waits for the uploads of a handle's buffers. A copy from pageable memory may return before it
// has arrived, ordered with the legacy stream only, while the handle's first run may come at once
// on a stream that does not wait for that one. A copy back is behind them, and done on return.
cudaError_t AwaitUploads(std::initializer_list<const DeviceBuffer*> buffers) {
  for (const DeviceBuffer* b : buffers) {
    char byte;
    if (b->as<char>()) return cudaMemcpy(&byte, b->as<char>(), 1, cudaMemcpyDeviceToHost);
  }
  return cudaSuccess;
}

int CheckDevice(const DeviceScope& scope, int device, int* num_sms, char* err, int errlen) {
  if (scope.error() != cudaSuccess) {
    const std::string what = "cudaSetDevice(" + std::to_string(device) + ") failed";
    return CudaFail(what.c_str(), scope.error(), err, errlen, 1);
  }
  int major = 0;
  cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(num_sms, cudaDevAttrMultiProcessorCount, device);
  if (e != cudaSuccess) return CudaFail("device query failed", e, err, errlen, 1);
  if (major != 10) return Fail("the kernels are built for sm_100a only", err, errlen);
  return 0;
}

// The null stream is the current device's own, and a stream that is being captured cannot be
// asked for its device: there the launch itself fails on a mismatch.
int CheckStream(cudaStream_t s, int device, char* err, int errlen) {
  if (!s) return 0;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(s, &capture);
  if (e == cudaSuccess && capture != cudaStreamCaptureStatusNone) return 0;
  int sdev = device;
  if (e == cudaSuccess) e = cudaStreamGetDevice(s, &sdev);
  if (e != cudaSuccess) return CudaFail("invalid stream", e, err, errlen, 1);
  if (sdev != device)
    return Fail("the stream belongs to device " + std::to_string(sdev) + ", not device " + std::to_string(device), err,
                errlen);
  return 0;
}

constexpr int64_t kMaxElements = int64_t(1) << 46;  // of a tensor's span: byte offsets stay far below 2^63

bool FitsSpan(int64_t n, int64_t stride) { return n <= 1 || stride <= kMaxElements / n; }

// A 2-byte tensor [tokens][heads][dim] by its strides, in elements.
struct View {
  const void* p = nullptr;
  int64_t tokens = 0, tok = 0, heads = 1, head = 0, dim = 0;
  bool empty() const { return !p || tokens <= 0 || heads <= 0 || dim <= 0; }
  int64_t span() const { return (tokens - 1) * tok + (heads - 1) * head + dim; }
  bool sane() const { return tok >= 0 && head >= 0 && FitsSpan(tokens, tok) && FitsSpan(heads, head); }
  // No two elements share an address: tokens of whole heads, or heads of whole tokens.
  bool distinct() const {
    const bool h_ok = heads <= 1 || head >= dim, t_ok = tokens <= 1 || tok >= dim;
    return h_ok && t_ok &&
           (tokens <= 1 || heads <= 1 || tok >= (heads - 1) * head + dim || head >= (tokens - 1) * tok + dim);
  }
  bool same(const View& o) const {
    return p == o.p && tokens == o.tokens && heads == o.heads && dim == o.dim && (tokens <= 1 || tok == o.tok) &&
           (heads <= 1 || head == o.head);
  }
};

// Whether two views may share an element: exact for slices of rows of one pitch, else by the
// whole ranges that they span.
bool Overlap(const View& a, const View& b) {
  if (a.empty() || b.empty()) return false;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  if (pa + a.span() * 2 <= pb || pb + b.span() * 2 <= pa) return false;
  auto rows = [](const View& v, int64_t* pitch, int64_t* width) {  // the outer of the two dimensions
    const bool tok_outer = v.heads <= 1 || (v.tokens > 1 && v.tok >= v.head);
    *pitch = tok_outer ? v.tok : v.head;
    *width = tok_outer ? (v.heads - 1) * v.head + v.dim : (v.tokens - 1) * v.tok + v.dim;
  };
  int64_t sa, wa, sb, wb;
  rows(a, &sa, &wa);
  rows(b, &sb, &wb);
  if (sa != sb || sa <= 0 || wa > sa || wb > sa) return true;
  const int64_t pitch = sa * 2;
  const int64_t d = static_cast<int64_t>(((static_cast<int64_t>(pb) - static_cast<int64_t>(pa)) % pitch + pitch) % pitch);
  return !(d >= wa * 2 && d + wb * 2 <= pitch);
}

bool Aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int64_t CeilDiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which documents the tcgen05 kernel takes and which the mma.sync kernel: the one that is
// expected to be done sooner. A CTA's time on an SM, in us, is about
//   tcgen05   start + tile * (tiles of 128 keys), for 256 rows
//   mma.sync  start + tile * (tiles of 64 keys), for 64 rows, with the SM full of CTAs
// with the constants below, by width of the head, from equal documents of 65 to 512 tokens
// (131072 in all, 4 heads). They meet at about 400 tokens of 32 elements (384: 236 us here, 220
// us there; 512: 253 and 284), 150 of 64 (128: 160 and 135; 160: 199 and 211) and 70 of 128
// (65: 610 and 588; 96: 269 and 439). Where the tcgen05 kernel's few large CTAs leave SMs empty,
// its time does not fall, while the mma.sync kernel cuts its keys up further, at about 1.7 times
// the work and 8 us for the joining: 1024 queries on 8192 keys, 4 heads of 64, 111 us and 59;
// 1024 on 1024, 12 heads of 64, 23 and 33.
// What it does not know: a causal mask, which halves the keys of both kernels, and how far a cache
// is filled. Over documents of 96 to 768 tokens (131072 in all, 4 heads) its choice costs at most
// 27% with a causal mask (256 of 32: 108 us, the other kernel 85) and 19% without (192 of 64: 173
// and 145), and nothing at 38 of 42 sizes; but 64 causal queries on each of 16 caches of 4096 keys
// filled to a quarter, heads of 128, take 61 us where the tcgen05 kernel would take 21, and on each
// of 128 caches of 512, heads of 64, 23 us where the mma.sync kernel would take 13. A caller that
// knows names the kernel (algo).
class KernelChoice {
 public:
  KernelChoice(const std::vector<ah::AttnDoc>& docs, int algo, int q_heads, int kv_heads, int head_dim, int num_sms)
      : algo_(algo), group_(q_heads / kv_heads), q_heads_(q_heads), kv_heads_(kv_heads), num_sms_(num_sms) {
    static constexpr Cost kCosts[3] = {{4.7, 3.0, 0.65, 0.56}, {3.4, 2.3, 1.2, 0.62}, {4.1, 3.4, 3.1, 1.41}};
    cost_ = kCosts[head_dim <= 32 ? 0 : (head_dim <= 64 ? 1 : 2)];
    for (const ah::AttnDoc& d : docs) {
      if (!Candidate(d)) continue;
      tc_ctas_ += TcCtas(d);
      mma_blocks_ += MmaBlocks(d);
      ++candidates_;
    }
  }
  bool TensorMemory(const ah::AttnDoc& d) const {
    if (algo_ != 0) return algo_ == 2 && d.nq > 0 && d.nk > 0;
    if (!Candidate(d)) return false;
    const double tc = TcCtas(d) * (cost_.tc_start + cost_.tc_tile * CeilDiv(d.nk, ah::kTcKeys));
    double mma = MmaBlocks(d) * (cost_.mma_start + cost_.mma_tile * CeilDiv(d.nk, ah::kMmaKeys)) / num_sms_;
    if (mma_blocks_ < 8 * num_sms_) mma = 1.7 * mma + 8.0 / candidates_;
    return tc / std::min<int64_t>(num_sms_, tc_ctas_) < mma;
  }

 private:
  struct Cost {
    double tc_start, tc_tile, mma_start, mma_tile;
  };
  bool Candidate(const ah::AttnDoc& d) const { return d.nk > 0 && int64_t{d.nq} * group_ > ah::kMmaRowsFew; }
  int64_t TcCtas(const ah::AttnDoc& d) const {
    return CeilDiv(d.nq, ah::attn_tc_item_tokens(group_)) * (ah::attn_tc_head_pairs(group_) ? q_heads_ / 2 : q_heads_);
  }
  int64_t MmaBlocks(const ah::AttnDoc& d) const {
    return CeilDiv(int64_t{d.nq} * group_, ah::kMmaRowsWide) * kv_heads_;
  }
  int algo_, group_, q_heads_, kv_heads_, num_sms_;
  Cost cost_;
  int64_t tc_ctas_ = 0, mma_blocks_ = 0, candidates_ = 0;
};

View Floats(const float* p, int64_t n) { return View{p, 1, 0, 1, 0, 2 * n}; }

}  // namespace

struct ah_norm {
  int device = 0, num_sms = 0, dtype = 0;
  bool has_post = false;
  ah::NormArgs args;
  DeviceBuffer a, b, w, wb;
};

struct ah_rope {
  int device = 0, num_sms = 0, dtype = 0;
  ah::RopeTable table;
  DeviceBuffer pairs;
};

struct ah_attn {
  int device = 0, num_sms = 0, dtype = 0;
  ah::AttnArgs args;
  int64_t q_total = 0, k_total = 0, docs_n = 0;
  DeviceBuffer docs, few, wide, tc, slopes, status;
  int n_few = 0, n_wide = 0, n_tc = 0, few_cluster = 1, wide_cluster = 1, few_tiles = 0, wide_tiles = 0;
};

extern "C" {

// ---------------------------------------------------------------------------
// Norms around a block
// ---------------------------------------------------------------------------
int ah_norm_create(int device, const ah_norm_desc* d, const float* post_weight, const float* post_bias,
                   const float* pre_weight, const float* pre_bias, const float* layer_scale, ah_norm** out, char* err,
                   int errlen) try {
  if (!d || !out) return Fail("invalid norm arguments", err, errlen);
  if (d->dtype != ah::kTokenF16 && d->dtype != ah::kTokenBf16) return Fail("norm: unknown element type", err, errlen);
  if (d->channels < 1 || d->channels > ah::kNormMaxChannels)
    return Fail("norm: channels must be 1.." + std::to_string(ah::kNormMaxChannels) + " (got " +
                    std::to_string(d->channels) + ")",
                err, errlen);
  if (d->post_norm < 0 || d->post_norm > 2 || d->pre_norm < 0 || d->pre_norm > 2)
    return Fail("norm: unknown norm kind", err, errlen);
  if (d->gate_act < 0 || d->gate_act > 3) return Fail("norm: unknown gate activation", err, errlen);
  if (!(d->post_eps >= 0.f) || !(d->pre_eps >= 0.f) || !std::isfinite(d->post_eps) || !std::isfinite(d->pre_eps))
    return Fail("norm: eps must be finite and not negative", err, errlen);
  if (!std::isfinite(d->residual_scale)) return Fail("norm: residual_scale must be finite", err, errlen);
  if (d->post_norm == 0 && (post_weight || post_bias))
    return Fail("norm: post_weight / post_bias without a post norm", err, errlen);
  if (d->pre_norm == 0 && (pre_weight || pre_bias))
    return Fail("norm: pre_weight / pre_bias without a pre norm", err, errlen);
  DeviceScope scope(device);
  auto h = std::make_unique<ah_norm>();
  if (const int rc = CheckDevice(scope, device, &h->num_sms, err, errlen)) return rc;
  h->device = device;
  h->dtype = d->dtype;
  h->args.C = d->channels;
  h->args.post = d->post_norm;
  h->args.pre = d->pre_norm;
  h->args.act = d->gate_act;
  h->args.post_eps = d->post_eps;
  h->args.pre_eps = d->pre_eps;
  const size_t n = d->channels, bytes = n * sizeof(float);
  cudaError_t e = cudaSuccess;
  if (post_weight || layer_scale || d->residual_scale != 1.f || post_bias) {
    std::vector<float> a(n), b(n);
    for (size_t c = 0; c < n; ++c) {
      const double s = static_cast<double>(d->residual_scale) * (layer_scale ? layer_scale[c] : 1.f);
      a[c] = static_cast<float>(s * (post_weight ? post_weight[c] : 1.f));
      if (post_bias) b[c] = static_cast<float>(s * post_bias[c]);
    }
    e = h->a.Upload(a.data(), bytes);
    if (e == cudaSuccess && post_bias) e = h->b.Upload(b.data(), bytes);
  }
  if (e == cudaSuccess && pre_weight) e = h->w.Upload(pre_weight, bytes);
  if (e == cudaSuccess && pre_bias) e = h->wb.Upload(pre_bias, bytes);
  if (e == cudaSuccess) e = AwaitUploads({&h->a, &h->b, &h->w, &h->wb});
  if (e != cudaSuccess) return CudaFail("norm weight upload failed", e, err, errlen, 1);
  h->args.a = h->a.as<float>();
  h->args.b = h->b.as<float>();
  h->args.w = h->w.as<float>();
  h->args.wb = h->wb.as<float>();
  *out = h.release();
  return 0;
} catch (const std::exception& e) {
  return Fail(std::string("norm: ") + e.what(), err, errlen);
}

int ah_norm_run(ah_norm* h, const ah_norm_io* io, void* stream, char* err, int errlen) try {
  if (!h || !io) return Fail("invalid norm run arguments", err, errlen);
  if (io->rows < 0 || io->rows_per_gate < 1 || io->rows_per_mod < 1)
    return Fail("norm: rows must not be negative, rows_per_gate and rows_per_mod at least 1", err, errlen);
  // Tensors of no rows may be null.
  if (io->rows > 0 && (!io->x || (!io->out && !io->norm)))
    return Fail("norm: x and one of out and norm are needed", err, errlen);
  if (io->rows > 0 && (io->gate || io->out) && !io->y)
    return Fail("norm: out and gate need the block output y", err, errlen);
  const int64_t C = h->args.C, rows = io->rows;
  auto pitch = [&](int64_t s) { return s ? s : C; };
  const int64_t grows = rows ? (rows - 1) / io->rows_per_gate + 1 : 0;
  const int64_t mrows = rows ? (rows - 1) / io->rows_per_mod + 1 : 0;
  const View x{io->x, rows, pitch(io->x_stride), 1, 0, C}, y{io->y, rows, pitch(io->y_stride), 1, 0, C};
  const View gate{io->gate, grows, pitch(io->gate_stride), 1, 0, C};
  const View ms{io->mod_scale, mrows, pitch(io->mod_stride), 1, 0, C};
  const View mb{io->mod_shift, mrows, pitch(io->mod_stride), 1, 0, C};
  const View out{io->out, rows, pitch(io->out_stride), 1, 0, C}, norm{io->norm, rows, pitch(io->norm_stride), 1, 0, C};
  for (const View* v : {&x, &y, &gate, &ms, &mb, &out, &norm}) {
    if (!v->sane() || !Aligned(v->p, 2)) return Fail("norm: bad row stride or a pointer off 2 bytes", err, errlen);
  }
  if (!out.distinct() || !norm.distinct()) return Fail("norm: output rows overlap one another", err, errlen);
  if (Overlap(out, norm)) return Fail("norm: out and norm overlap", err, errlen);
  for (const View* o : {&out, &norm}) {
    for (const View* v : {&x, &y})
      if (!o->same(*v) && Overlap(*o, *v))
        return Fail("norm: an output may be x or y itself but not overlap it otherwise", err, errlen);
    for (const View* v : {&gate, &ms, &mb})
      if (Overlap(*o, *v)) return Fail("norm: an output overlaps the gate or the modulation", err, errlen);
  }
  DeviceScope scope(h->device);
  if (scope.error() != cudaSuccess) return CudaFail("norm: cudaSetDevice failed", scope.error(), err, errlen, 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = CheckStream(s, h->device, err, errlen)) return rc;
  ah::NormArgs a = h->args;
  a.x = io->x, a.y = io->y, a.gate = io->gate, a.mscale = io->mod_scale, a.mshift = io->mod_shift;
  a.out = io->out, a.norm = io->norm;
  a.xs = x.tok, a.ys = y.tok, a.gs = gate.tok, a.ms = ms.tok, a.os = out.tok, a.ns = norm.tok;
  a.rows = rows, a.rows_per_gate = io->rows_per_gate, a.rows_per_mod = io->rows_per_mod;
  const cudaError_t e = ah::norm_launch(a, h->dtype, h->num_sms, s);
  return e == cudaSuccess ? 0 : CudaFail("norm launch failed", e, err, errlen, 2);
} catch (const std::exception& e) {
  return Fail(std::string("norm: ") + e.what(), err, errlen, 2);
}

void ah_norm_destroy(ah_norm* h) {
  if (!h) return;
  DeviceScope scope(h->device);
  delete h;
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------
int ah_rope_create(int device, const ah_rope_desc* d, ah_rope** out, char* err, int errlen) try {
  if (!d || !out) return Fail("invalid rope arguments", err, errlen);
  if (d->dtype != ah::kTokenF16 && d->dtype != ah::kTokenBf16) return Fail("rope: unknown element type", err, errlen);
  if (d->head_dim < 2 || d->head_dim > 512) return Fail("rope: head_dim must be 2..512", err, errlen);
  if (d->axes < 1 || d->axes > 3) return Fail("rope: 1 to 3 axes", err, errlen);
  if (d->layout < 0 || d->layout > 2) return Fail("rope: unknown layout", err, errlen);
  int rot = 0;
  for (int i = 0; i < d->axes; ++i) {
    if (d->axis_dims[i] < 0 || d->axis_dims[i] % 2 || d->axis_dims[i] > d->head_dim)
      return Fail("rope: the axes' dims must be even and within the head", err, errlen);
    if (!(d->theta[i] > 0.0) || !std::isfinite(d->theta[i]))
      return Fail("rope: theta must be positive and finite", err, errlen);
    rot += d->axis_dims[i];
  }
  if (rot < 2 || rot > d->head_dim) return Fail("rope: the axes' dims must sum to 2..head_dim", err, errlen);
  for (int i = 1; i < d->axes; ++i)
    if (d->layout == ah::kRopeShared && d->theta[i] != d->theta[0])
      return Fail("rope: the shared layout has one theta", err, errlen);
  DeviceScope scope(device);
  auto h = std::make_unique<ah_rope>();
  if (const int rc = CheckDevice(scope, device, &h->num_sms, err, errlen)) return rc;
  h->device = device;
  h->dtype = d->dtype;
  const double kTwoPi = 6.283185307179586476925;
  std::vector<ah::RopePair> pairs;
  bool halves8 = d->layout != ah::kRopePairs && rot % 16 == 0;
  for (int ax = 0, base = 0; ax < d->axes; base += d->axis_dims[ax++]) {
    const int n = d->axis_dims[ax];
    if (d->layout == ah::kRopeHalves && n % 16) halves8 = false;
    for (int j = 0; j < n / 2; ++j) {
      ah::RopePair p{};
      const int g = static_cast<int>(pairs.size());
      const double power = d->layout == ah::kRopeShared ? 2.0 * g / rot : 2.0 * j / n;
      p.turns = std::pow(d->theta[ax], -power) / kTwoPi * (d->inverse ? -1.0 : 1.0);
      p.axis = ax;
      p.e0 = d->layout == ah::kRopePairs ? base + 2 * j : (d->layout == ah::kRopeHalves ? base + j : g);
      p.e1 = d->layout == ah::kRopePairs ? p.e0 + 1 : (d->layout == ah::kRopeHalves ? p.e0 + n / 2 : g + rot / 2);
      pairs.push_back(p);
    }
  }
  cudaError_t e = h->pairs.Upload(pairs.data(), pairs.size() * sizeof(ah::RopePair));
  if (e == cudaSuccess) e = AwaitUploads({&h->pairs});
  if (e != cudaSuccess) return CudaFail("rope table upload failed", e, err, errlen, 1);
  ah::RopeTable& t = h->table;
  t.pairs = h->pairs.as<ah::RopePair>();
  t.npairs = static_cast<int>(pairs.size());
  t.rot = rot;
  t.head_dim = d->head_dim;
  t.axes = d->axes;
  t.layout = d->layout;
  t.halves8 = halves8;
  *out = h.release();
  return 0;
} catch (const std::exception& e) {
  return Fail(std::string("rope: ") + e.what(), err, errlen);
}

int ah_rope_run(ah_rope* h, int64_t tokens, const float* positions, const ah_rope_io* q, const ah_rope_io* k,
                void* stream, char* err, int errlen) try {
  if (!h || (tokens > 0 && (!positions || (!q && !k))))  // tensors of no tokens may be null
    return Fail("invalid rope run arguments", err, errlen);
  if (tokens < 0 || tokens > (int64_t(1) << 31) - 1) return Fail("rope: tokens must be 0..2^31-1", err, errlen);
  if (!Aligned(positions, 4)) return Fail("rope: positions must be 4-byte aligned", err, errlen);
  const int D = h->table.head_dim;
  ah::RopeArgs a;
  a.pos = positions;
  a.tokens = tokens;
  View in[2], out[2];
  for (int w = 0; w < 2; ++w) {
    const ah_rope_io* io = w ? k : q;
    if (!io) continue;
    if (io->heads < 1 || io->heads > 1024) return Fail("rope: heads must be 1..1024", err, errlen);
    if (tokens > 0 && (!io->in || !io->out)) return Fail("rope: null tensor", err, errlen);
    const int64_t packed = static_cast<int64_t>(io->heads) * D;
    in[w] = View{io->in, tokens, io->in_token_stride ? io->in_token_stride : packed, io->heads,
                 io->in_head_stride ? io->in_head_stride : D, D};
    out[w] = View{io->out, tokens, io->out_token_stride ? io->out_token_stride : packed, io->heads,
                  io->out_head_stride ? io->out_head_stride : D, D};
    for (const View* v : {&in[w], &out[w]})
      if (!v->sane() || !Aligned(v->p, 2)) return Fail("rope: bad stride or a pointer off 2 bytes", err, errlen);
    if (!out[w].distinct()) return Fail("rope: output heads or tokens overlap one another", err, errlen);
    a.in[w] = io->in, a.out[w] = io->out, a.heads[w] = io->heads;
    a.in_tok[w] = in[w].tok, a.in_head[w] = in[w].head, a.out_tok[w] = out[w].tok, a.out_head[w] = out[w].head;
  }
  const View pos = Floats(positions, tokens * h->table.axes);
  for (int w = 0; w < 2; ++w) {
    if (!out[w].same(in[w]) && Overlap(out[w], in[w]))
      return Fail("rope: the output may be the input itself but not overlap it otherwise", err, errlen);
    if (Overlap(out[w], in[1 - w]) || Overlap(out[w], pos))
      return Fail("rope: an output overlaps another input", err, errlen);
  }
  if (Overlap(out[0], out[1])) return Fail("rope: the outputs overlap", err, errlen);
  DeviceScope scope(h->device);
  if (scope.error() != cudaSuccess) return CudaFail("rope: cudaSetDevice failed", scope.error(), err, errlen, 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = CheckStream(s, h->device, err, errlen)) return rc;
  const cudaError_t e = ah::rope_launch(h->table, a, h->dtype, h->num_sms, s);
  return e == cudaSuccess ? 0 : CudaFail("rope launch failed", e, err, errlen, 2);
} catch (const std::exception& e) {
  return Fail(std::string("rope: ") + e.what(), err, errlen, 2);
}

void ah_rope_destroy(ah_rope* h) {
  if (!h) return;
  DeviceScope scope(h->device);
  delete h;
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
int ah_attn_create(int device, const ah_attn_desc* d, int docs, const int64_t* q_offsets, const int64_t* k_offsets,
                   const int64_t* prefix, const float* slopes, ah_attn** out, char* err, int errlen) try {
  if (!d || !out || docs < 0 || !q_offsets || !k_offsets) return Fail("invalid attention arguments", err, errlen);
  if (d->dtype != ah::kTokenF16 && d->dtype != ah::kTokenBf16)
    return Fail("attention: unknown element type", err, errlen);
  if (d->head_dim < 8 || d->head_dim > ah::kAttnMaxHeadDim || d->head_dim % 8)
    return Fail("attention: head_dim must be a multiple of 8 up to 128 (got " + std::to_string(d->head_dim) + ")", err,
                errlen);
  if (d->kv_heads < 1 || d->kv_heads > 1024 || d->q_heads < 1 || d->q_heads > 1024 || d->q_heads % d->kv_heads)
    return Fail("attention: q_heads must be a multiple of kv_heads, both 1..1024", err, errlen);
  if (!(d->scale > 0.f) || !std::isfinite(2.f * d->scale))
    return Fail("attention: scale must be positive and finite", err, errlen);
  if (!(d->cap >= 0.f) || !std::isfinite(d->cap))
    return Fail("attention: cap must be finite, 0 for none", err, errlen);
  if (d->cap > 0.f && !(std::isfinite(2.f * d->cap * 1.44269504f) && std::isfinite(3.f * d->scale / d->cap)))
    return Fail("attention: scale / cap or cap is out of fp32 range", err, errlen);
  if (d->mask < 0 || d->mask > 1) return Fail("attention: unknown mask", err, errlen);
  if (prefix && d->mask != 1) return Fail("attention: a prefix needs the causal mask", err, errlen);
  if (d->algo < 0 || d->algo > 2) return Fail("attention: unknown algo", err, errlen);
  if (d->axes < 0 || d->axes > ah::kAttnMaxAxes) return Fail("attention: 0 to 3 bias axes", err, errlen);
  if ((d->axes > 0) != (slopes != nullptr)) return Fail("attention: slopes go with bias axes", err, errlen);
  const int group = d->q_heads / d->kv_heads;
  const int64_t most = std::numeric_limits<int32_t>::max() - 1024;
  if (q_offsets[0] != 0 || k_offsets[0] != 0) return Fail("attention: offsets begin with 0", err, errlen);
  for (int i = 0; i < docs; ++i)
    if (q_offsets[i + 1] < q_offsets[i] || k_offsets[i + 1] < k_offsets[i] || q_offsets[i + 1] > most / group ||
        k_offsets[i + 1] > most)
      return Fail("attention: offsets must not fall, and stay below 2^31 - 1024 (queries times group too)", err,
                  errlen);
  std::vector<ah::AttnDoc> table(docs);
  for (int i = 0; i < docs; ++i) {
    const int64_t nk = k_offsets[i + 1] - k_offsets[i];
    if (prefix && (prefix[i] < 0 || prefix[i] > nk))
      return Fail("attention: prefix of document " + std::to_string(i) + " is outside its keys", err, errlen);
    table[i] = {static_cast<int>(q_offsets[i]), static_cast<int>(q_offsets[i + 1] - q_offsets[i]),
                static_cast<int>(k_offsets[i]), static_cast<int>(nk), prefix ? static_cast<int>(prefix[i]) : 0};
  }
  const double kLog2e = 1.44269504088896340736;
  std::vector<float> bias(slopes ? static_cast<size_t>(d->q_heads) * d->axes : 0);
  // In the units of the kernels' scores: powers of two behind a cap, else as the product q.k.
  for (size_t i = 0; i < bias.size(); ++i) {
    bias[i] = static_cast<float>(d->cap > 0.f ? slopes[i] * kLog2e : static_cast<double>(slopes[i]) / d->scale);
    if (!std::isfinite(slopes[i]) || !std::isfinite(bias[i]))
      return Fail("attention: slopes, and slopes / scale, must be finite", err, errlen);
  }
  DeviceScope scope(device);
  auto h = std::make_unique<ah_attn>();
  if (const int rc = CheckDevice(scope, device, &h->num_sms, err, errlen)) return rc;
  h->device = device;
  h->dtype = d->dtype;
  h->q_total = q_offsets[docs];
  h->k_total = k_offsets[docs];
  h->docs_n = docs;
  ah::AttnArgs& a = h->args;
  a.q_heads = d->q_heads, a.kv_heads = d->kv_heads, a.group = group, a.head_dim = d->head_dim;
  a.axes = d->axes, a.causal = d->mask;
  a.q_total = h->q_total, a.k_total = h->k_total, a.num_sms = h->num_sms;
  if (d->cap > 0.f) {
    a.cap_log2 = static_cast<float>(d->cap * kLog2e);
    a.cap_arg = static_cast<float>(static_cast<double>(d->scale) / d->cap);
    a.cap_exp = static_cast<float>(2 * kLog2e * d->scale / d->cap);
  } else {
    a.score_mul = static_cast<float>(d->scale * kLog2e);
  }
  // Blocks of rows, those with the most keys first, so that the last ones to start are short.
  const KernelChoice choice(table, d->algo, d->q_heads, d->kv_heads, d->head_dim, h->num_sms);
  std::vector<ah::AttnItem> few, wide, tc;
  int few_tiles = 0, wide_tiles = 0;
  std::vector<int> order(docs);
  for (int i = 0; i < docs; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int i, int j) { return table[i].nk > table[j].nk; });
  for (int i : order) {
    const ah::AttnDoc& doc = table[i];
    if (choice.TensorMemory(doc)) {
      const int step = ah::attn_tc_item_tokens(group);
      for (int r = (doc.nq - 1) / step * step; r >= 0; r -= step) tc.push_back({i, r});  // causal: longest first
      continue;
    }
    const int rows = doc.nq * group, tiles = (doc.nk + ah::kMmaKeys - 1) / ah::kMmaKeys;
    const bool is_few = rows <= ah::kMmaRowsFew;
    const int step = is_few ? ah::kMmaRowsFew : ah::kMmaRowsWide;
    for (int r = 0; r < rows; r += step) (is_few ? few : wide).push_back({i, r});
    int& t = is_few ? few_tiles : wide_tiles;
    if (rows) t = std::max(t, tiles);
  }
  if (few.size() + wide.size() + tc.size() > (1u << 26))
    return Fail("attention: more than 2^26 blocks of rows", err, errlen);
  // A cluster of CTAs shares one block's keys until there are as many CTAs as places (two to an
  // SM), while each keeps at least four tiles. One token in each of 8 documents of half-filled
  // 65536-key caches, 8 key heads: 344 us in clusters of 4, 313 us of 8, 332 us of 16.
  auto cluster = [&](size_t items, int tiles) {
    int c = 1;
    while (c < 16 && items * d->kv_heads * c < 2u * h->num_sms && tiles >= c * 8) c *= 2;
    return c;
  };
  h->n_few = static_cast<int>(few.size());
  h->n_wide = static_cast<int>(wide.size());
  h->n_tc = static_cast<int>(tc.size());
  h->few_tiles = few_tiles;
  h->wide_tiles = wide_tiles;
  h->few_cluster = cluster(few.size(), few_tiles);
  h->wide_cluster = cluster(wide.size(), wide_tiles);
  cudaError_t e = h->docs.Upload(table.data(), table.size() * sizeof(ah::AttnDoc));
  if (e == cudaSuccess) e = h->few.Upload(few.data(), few.size() * sizeof(ah::AttnItem));
  if (e == cudaSuccess) e = h->wide.Upload(wide.data(), wide.size() * sizeof(ah::AttnItem));
  if (e == cudaSuccess) e = h->tc.Upload(tc.data(), tc.size() * sizeof(ah::AttnItem));
  if (e == cudaSuccess) e = h->slopes.Upload(bias.data(), bias.size() * sizeof(float));
  const uint32_t zero = 0;
  if (e == cudaSuccess) e = h->status.Upload(&zero, sizeof zero);
  if (e == cudaSuccess) e = AwaitUploads({&h->status});
  if (e != cudaSuccess) return CudaFail("attention plan upload failed", e, err, errlen, 1);
  a.docs = h->docs.as<ah::AttnDoc>();
  a.slopes = h->slopes.as<float>();
  a.status = h->status.as<uint32_t>();
  *out = h.release();
  return 0;
} catch (const std::exception& e) {
  return Fail(std::string("attention: ") + e.what(), err, errlen);
}

int ah_attn_run(ah_attn* h, const ah_attn_io* io, void* stream, char* err, int errlen) try {
  if (!h || !io) return Fail("invalid attention run arguments", err, errlen);
  const int64_t D = h->args.head_dim, hq = h->args.q_heads, hk = h->args.kv_heads;
  auto view = [&](const void* p, int64_t tokens, int64_t tok, int64_t heads, int64_t head) {
    return View{p, tokens, tok ? tok : heads * D, heads, head ? head : D, D};
  };
  const View q = view(io->q, h->q_total, io->q_token_stride, hq, io->q_head_stride);
  const View k = view(io->k, h->k_total, io->k_token_stride, hk, io->k_head_stride);
  const View v = view(io->v, h->k_total, io->v_token_stride, hk, io->v_head_stride);
  const View o = view(io->out, h->q_total, io->out_token_stride, hq, io->out_head_stride);
  if (h->q_total > 0 && (!io->q || !io->out)) return Fail("attention: null tensor", err, errlen);
  if (h->k_total > 0 && (!io->k || !io->v)) return Fail("attention: null tensor", err, errlen);
  if (h->args.axes > 0 && ((h->q_total > 0 && !io->q_positions) || (h->k_total > 0 && !io->k_positions)))
    return Fail("attention: the distance bias needs q_positions and k_positions", err, errlen);
  for (const View* t : {&q, &k, &v, &o}) {
    if (!t->sane()) return Fail("attention: bad stride", err, errlen);
    if (!Aligned(t->p, 16) || t->tok % 8 || t->head % 8)
      return Fail("attention: tensors must be 16-byte aligned, with strides that are multiples of 8 elements", err,
                  errlen);
  }
  if (!Aligned(io->q_positions, 4) || !Aligned(io->k_positions, 4) || !Aligned(io->k_lens, 4))
    return Fail("attention: positions and k_lens must be 4-byte aligned", err, errlen);
  if (!o.distinct()) return Fail("attention: output heads or tokens overlap one another", err, errlen);
  const View qp = Floats(io->q_positions, h->q_total * h->args.axes);
  const View kp = Floats(io->k_positions, h->k_total * h->args.axes);
  const View lens{io->k_lens, 1, 0, 1, 0, 2 * h->docs_n};
  for (const View* t : {&q, &k, &v, &qp, &kp, &lens})
    if (Overlap(o, *t)) return Fail("attention: the output overlaps an input", err, errlen);
  DeviceScope scope(h->device);
  if (scope.error() != cudaSuccess) return CudaFail("attention: cudaSetDevice failed", scope.error(), err, errlen, 2);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = CheckStream(s, h->device, err, errlen)) return rc;
  ah::AttnArgs a = h->args;
  a.q = io->q, a.k = io->k, a.v = io->v, a.out = io->out;
  a.q_tok = q.tok, a.q_head = q.head, a.k_tok = k.tok, a.k_head = k.head;
  a.v_tok = v.tok, a.v_head = v.head, a.o_tok = o.tok, a.o_head = o.head;
  a.q_pos = io->q_positions, a.k_pos = io->k_positions, a.k_lens = io->k_lens;
  cudaError_t e = cudaSuccess;
  std::string what = "attention launch failed";
  if (h->n_tc) {
    a.items = h->tc.as<ah::AttnItem>();
    a.num_items = h->n_tc;
    e = ah::attn_tc_launch(a, h->dtype, s, &what);
  }
  if (e == cudaSuccess && h->n_wide) {
    a.items = h->wide.as<ah::AttnItem>();
    a.num_items = h->n_wide;
    e = ah::attn_mma_launch(a, h->dtype, false, h->wide_cluster, h->wide_tiles, s);
  }
  if (e == cudaSuccess && h->n_few) {
    a.items = h->few.as<ah::AttnItem>();
    a.num_items = h->n_few;
    e = ah::attn_mma_launch(a, h->dtype, true, h->few_cluster, h->few_tiles, s);
  }
  return e == cudaSuccess ? 0 : CudaFail(what.c_str(), e, err, errlen, 2);
} catch (const std::exception& e) {
  return Fail(std::string("attention: ") + e.what(), err, errlen, 2);
}

int ah_attn_status(ah_attn* h, uint32_t* status) {
  if (!h || !status) return 1;
  DeviceScope scope(h->device);
  if (scope.error() != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess) return 2;
  if (cudaMemcpy(status, h->args.status, sizeof(uint32_t), cudaMemcpyDeviceToHost) != cudaSuccess) return 2;
  if (*status == 0) return 0;
  // The fill is waited for, so that it cannot wipe out what a later run reports.
  if (cudaMemset(h->args.status, 0, sizeof(uint32_t)) != cudaSuccess) return 2;
  return cudaDeviceSynchronize() == cudaSuccess ? 0 : 2;
}

void ah_attn_destroy(ah_attn* h) {
  if (!h) return;
  DeviceScope scope(h->device);
  delete h;
}

}  // extern "C"
