"""When a token operator's handle is there, its parameters are on the device: the C boundary
(tokens_capi.cc) compiled against a stand-in for the CUDA runtime whose copies from the host and
fills arrive only when something waits for them, as those from pageable memory may."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import numpy as np
import pytest

from arthip_b200 import build, native, token_ops
from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm

STAND_IN = r"""
#include <cuda_runtime.h>
#include <cstdlib>
#include <cstring>
#include <vector>
#include "kernels/tokens.h"
struct Pending { void* dst; std::vector<char> data; };
static std::vector<Pending> g_pending;
static uint32_t* g_status = nullptr;
static int g_late = 0;  // launches that come before the uploads have arrived
static void arrive() {
  for (const Pending& p : g_pending) std::memcpy(p.dst, p.data.data(), p.data.size());
  g_pending.clear();
}
extern "C" {
int fake_pending() { return static_cast<int>(g_pending.size()); }
int fake_late() { return g_late; }
void fake_timeout() { *g_status = 1; }
cudaError_t cudaGetDevice(int* d) { *d = 0; return cudaSuccess; }
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
  *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : 148;
  return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::calloc(n, 1); return cudaSuccess; }
cudaError_t cudaFree(void* p) { arrive(); std::free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind kind) {
  const char* from = static_cast<const char*>(s);
  if (kind == cudaMemcpyHostToDevice) {
    g_pending.push_back({d, std::vector<char>(from, from + n)});
  } else {  // to the host: behind all that went before, and done on return
    arrive();
    std::memcpy(d, s, n);
  }
  return cudaSuccess;
}
cudaError_t cudaMemset(void* d, int v, size_t n) {
  g_pending.push_back({d, std::vector<char>(n, static_cast<char>(v))});
  return cudaSuccess;
}
cudaError_t cudaDeviceSynchronize() { arrive(); return cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t) { arrive(); return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "stand-in error"; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) {
  *c = cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
cudaError_t cudaStreamGetDevice(cudaStream_t, int* d) { *d = 0; return cudaSuccess; }
}
namespace ah {
static cudaError_t launched() { g_late += !g_pending.empty(); return cudaSuccess; }
cudaError_t norm_launch(const NormArgs&, int, int, cudaStream_t) { return launched(); }
cudaError_t rope_launch(const RopeTable&, const RopeArgs&, int, int, cudaStream_t) { return launched(); }
cudaError_t attn_tc_launch(const AttnArgs& a, int, cudaStream_t, std::string*) { g_status = a.status; return launched(); }
cudaError_t attn_mma_launch(const AttnArgs& a, int, bool, int, int, cudaStream_t) { g_status = a.status; return launched(); }
}
"""

BASE = 0x10000000  # a 16-byte aligned address; nothing reads it
MB = 1 << 20


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    td = tmp_path_factory.mktemp("uploads")
    (td / "stand_in.cc").write_text(STAND_IN)
    so = td / "libuploads_host.so"
    cuda = Path(build.nvcc()).resolve().parents[1]
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", str(build.CSRC), "-I",
                        str(cuda / "include"), str(build.CSRC / "tokens_capi.cc"), str(td / "stand_in.cc"), "-o",
                        str(so)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    l = ctypes.CDLL(str(so))
    for name, (res, args) in native.SIGNATURES.items():
        if name.startswith(("ah_norm_", "ah_rope_", "ah_attn_")):
            fn = getattr(l, name)
            fn.restype, fn.argtypes = res, args
    return l


@pytest.fixture
def fake(fake_lib, monkeypatch):
    monkeypatch.setattr(token_ops, "lib", lambda: fake_lib)
    fake_lib.cudaDeviceSynchronize()
    return fake_lib


def test_uploads_have_arrived_when_a_handle_is_there(fake):
    """The first run may follow at once on a stream that nothing orders behind the uploads."""
    w = np.ones(8)
    for make in (lambda: TokenNorm(8), lambda: TokenNorm(8, pre_weight=w), lambda: TokenNorm(8, layer_scale=w),
                 lambda: TokenNorm(8, post_norm="rms", post_bias=w), lambda: TokenNorm(8, pre_norm="layer", pre_bias=w)):
        op = make()
        assert fake.fake_pending() == 0
        op.run(4, BASE, norm_ptr=BASE + MB)
    rope = AxisRotary(8, [8])
    assert fake.fake_pending() == 0
    rope.run(4, BASE, BASE + MB, 1)
    for docs in ([0], [0, 1, 300]):
        attn = TokenAttention(docs, docs, 1, 1, 64, slopes=[[1.0]])
        assert fake.fake_pending() == 0
        attn.run(*(BASE + i * MB for i in range(4)), BASE + 4 * MB, BASE + 4 * MB)
    assert fake.fake_late() == 0


def test_status_is_cleared_when_its_read_returns(fake):
    """A later run's error word must not be wiped by a fill that is still on its way."""
    attn = TokenAttention([0, 9], [0, 9], 1, 1, 64)
    attn.run(*(BASE + i * MB for i in range(4)))
    fake.fake_timeout()
    assert attn.status() == 1
    assert fake.fake_pending() == 0
    fake.fake_timeout()
    assert attn.status() == 1
    assert attn.status() == 0
