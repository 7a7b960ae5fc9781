"""Argument checks and plans of the token operators on a CPU-only host: the C boundary
(tokens_capi.cc) compiled against a stand-in for the CUDA runtime whose devices are two
sm_100 ones, whose memory is the host's and whose launches are only counted."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

from arthip_b200 import build, native, token_ops
from arthip_b200.engine import EngineHarnessError
from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm

STAND_IN = r"""
#include <cuda_runtime.h>
#include <cstdlib>
#include <cstring>
#include "kernels/tokens.h"
static int g_device = 0, g_sets = 0, g_launches = 0, g_live = 0, g_fail_malloc = 0;
extern "C" {
int fake_device() { return g_device; }
int fake_launches() { return g_launches; }
int fake_live() { return g_live; }
void fake_fail_malloc(int n) { g_fail_malloc = n; }
cudaError_t cudaGetDevice(int* d) { *d = g_device; return cudaSuccess; }
cudaError_t cudaSetDevice(int d) {
  if (d < 0 || d > 1) return cudaErrorInvalidDevice;
  g_device = d;
  return cudaSuccess;
}
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr a, int) {
  *v = a == cudaDevAttrComputeCapabilityMajor ? 10 : 148;
  return cudaSuccess;
}
cudaError_t cudaMalloc(void** p, size_t n) {
  if (g_fail_malloc > 0 && --g_fail_malloc == 0) return cudaErrorMemoryAllocation;
  *p = std::malloc(n);
  ++g_live;
  return cudaSuccess;
}
cudaError_t cudaFree(void* p) { std::free(p); --g_live; return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind) { std::memcpy(d, s, n); return cudaSuccess; }
cudaError_t cudaMemset(void* d, int v, size_t n) { std::memset(d, v, n); return cudaSuccess; }
cudaError_t cudaDeviceSynchronize() { return cudaSuccess; }
const char* cudaGetErrorString(cudaError_t) { return "stand-in error"; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t, cudaStreamCaptureStatus* c) {
  *c = cudaStreamCaptureStatusNone;
  return cudaSuccess;
}
// the stream 0x1000 belongs to device 1, all others to device 0 (and the null one to any)
cudaError_t cudaStreamGetDevice(cudaStream_t s, int* d) {
  *d = s == nullptr ? g_device : (reinterpret_cast<size_t>(s) == 0x1000 ? 1 : 0);
  return cudaSuccess;
}
}
namespace ah {
cudaError_t norm_launch(const NormArgs&, int, int, cudaStream_t) { ++g_launches; return cudaSuccess; }
cudaError_t rope_launch(const RopeTable&, const RopeArgs&, int, int, cudaStream_t) { ++g_launches; return cudaSuccess; }
cudaError_t attn_tc_launch(const AttnArgs&, int, cudaStream_t, std::string*) { ++g_launches; return cudaSuccess; }
cudaError_t attn_mma_launch(const AttnArgs&, int, bool, int, int, cudaStream_t) { ++g_launches; return cudaSuccess; }
}
"""


@pytest.fixture(scope="module")
def fake_lib(tmp_path_factory):
    td = tmp_path_factory.mktemp("tokens_capi")
    (td / "stand_in.cc").write_text(STAND_IN)
    so = td / "libtokens_host.so"
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
    return fake_lib


def refused(match, fn, *args, **kw):
    with pytest.raises(EngineHarnessError, match=match):
        fn(*args, **kw)


BASE = 0x10000000  # a 16-byte aligned address; nothing reads it
MB = 1 << 20


def test_norm_create_refusals(fake):
    for c in (0, -1, 8193):
        refused("channels", TokenNorm, c)
    refused("dtype", TokenNorm, 8, dtype="fp32")
    refused("norm", TokenNorm, 8, post_norm="batch")
    refused("gate", TokenNorm, 8, gate_act="relu")
    refused("eps", TokenNorm, 8, pre_eps=-1e-6)
    refused("eps", TokenNorm, 8, post_eps=math.nan)
    refused("residual_scale", TokenNorm, 8, residual_scale=math.inf)
    refused("shape", TokenNorm, 8, pre_weight=np.ones(7))
    refused("without a post norm", TokenNorm, 8, post_weight=np.ones(8))
    refused("without a pre norm", TokenNorm, 8, pre_norm="none", pre_bias=np.ones(8))
    refused("cudaSetDevice", TokenNorm, 8, device=5)
    assert fake.fake_live() == 0


def test_failed_uploads_free_what_was_taken(fake):
    for n in (1, 2, 3, 4):
        fake.fake_fail_malloc(n)
        refused("upload", TokenNorm, 8, post_norm="rms", post_weight=np.ones(8), post_bias=np.ones(8),
                pre_weight=np.ones(8), pre_bias=np.ones(8))
        assert fake.fake_live() == 0
    for n in (1, 2, 3):
        fake.fake_fail_malloc(n)
        refused("upload", TokenAttention, [0, 1, 300], [0, 300, 700], 1, 1, 64, slopes=[[1.0]])
        assert fake.fake_live() == 0
    fake.fake_fail_malloc(0)


def test_norm_run_refusals(fake):
    op = TokenNorm(64)
    x, y, o, n, g = (BASE + i * MB for i in range(5))
    before = fake.fake_launches()
    ok = dict(rows=100, x_ptr=x, out_ptr=o, norm_ptr=n, y_ptr=y)
    for match, bad in [("rows", dict(rows=-1)), ("rows", dict(rows_per_gate=0)), ("rows", dict(rows_per_mod=-2)),
                       ("needed", dict(x_ptr=0)), ("needed", dict(out_ptr=0, norm_ptr=0)),
                       ("block output", dict(y_ptr=0)), ("block output", dict(y_ptr=0, out_ptr=0, gate_ptr=g)),
                       ("stride", dict(x_stride=-64)), ("stride", dict(x_ptr=x + 1)),
                       ("stride", dict(y_stride=1 << 62)), ("overlap", dict(out_stride=63)),
                       ("out and norm", dict(norm_ptr=o)), ("out and norm", dict(norm_ptr=o + 64)),
                       ("x or y itself", dict(out_ptr=x + 2)), ("x or y itself", dict(norm_ptr=y + 128)),
                       ("x or y itself", dict(out_ptr=x, out_stride=128)),
                       ("gate", dict(gate_ptr=o)), ("gate", dict(mod_shift_ptr=n + 2, rows_per_mod=100)),
                       ("device 1", dict(stream=0x1000))]:
        refused(match, op.run, **(ok | bad))
    assert fake.fake_launches() == before
    # the second slice of each row of one buffer is no overlap; in place is allowed
    op.run(100, x, x + 128, n, y, x_stride=128, out_stride=128)
    op.run(100, x, x, y, y)
    op.run(0, x, o, n, y)
    op.run(100, x, norm_ptr=n)
    assert fake.fake_launches() == before + 4


def test_rope_refusals(fake):
    refused("head_dim", AxisRotary, 1, [2])
    refused("head_dim", AxisRotary, 514, [2])
    refused("axes", AxisRotary, 64, [])
    refused("axes", AxisRotary, 64, [2, 2, 2, 2])
    refused("even", AxisRotary, 64, [3])
    refused("even", AxisRotary, 64, [-2, 4])
    refused("sum", AxisRotary, 64, [32, 34])
    refused("sum", AxisRotary, 64, [0, 0])
    refused("theta", AxisRotary, 64, [32], theta=0.0)
    refused("theta", AxisRotary, 64, [32], theta=math.inf)
    refused("one theta", AxisRotary, 64, [32, 32], theta=(1e4, 1e2), layout="shared")
    refused("layout", AxisRotary, 64, [32], layout="spiral")
    op = AxisRotary(64, [32, 32])
    pos, q, k, o = (BASE + i * MB for i in range(4))
    before = fake.fake_launches()
    for match, args, kw in [
            ("invalid", (10, 0, q, 2), {}), ("invalid", (10, pos, 0, 2), {}), ("tokens", (-1, pos, q, 2), {}),
            ("tokens", (1 << 31, pos, q, 2), {}), ("heads", (10, pos, q, 0), {}), ("heads", (10, pos, q, 2000), {}),
            ("4-byte", (10, pos + 2, q, 2), {}), ("stride", (10, pos, q + 1, 2), {}),
            ("stride", (10, pos, q, 2), dict(q_strides=(-128, 64))),
            ("overlap one another", (10, pos, q, 2), dict(q_strides=(100, 64))),
            ("input itself", (10, pos, q, 2, q + 128), {}), ("another input", (10, pos, q, 2, o, k, 2, q), {}),
            ("another input", (10, pos, q, 2, pos), {}), ("outputs overlap", (10, pos, q, 2, o, k, 2, o + 16), {}),
            ("device 1", (10, pos, q, 2), dict(stream=0x1000))]:
        refused(match, op.run, *args, **kw)
    assert fake.fake_launches() == before
    # q and k side by side in one row, in place
    op.run(10, pos, q, 2, k_ptr=q + 256, k_heads=2, q_strides=(256, 64), k_strides=(256, 64))
    op.run(10, pos, q, 2, k_ptr=q + 64 * 10 * 2 * 2, k_heads=1, q_strides=(64, 640), k_strides=(64, 640))
    assert fake.fake_launches() == before + 2


def test_attention_create_refusals(fake):
    good = dict(q_offsets=[0, 4], k_offsets=[0, 4], q_heads=4, kv_heads=2, head_dim=64)
    for match, bad in [("head_dim", dict(head_dim=0)), ("head_dim", dict(head_dim=12)),
                       ("head_dim", dict(head_dim=136)), ("q_heads", dict(q_heads=3)), ("q_heads", dict(kv_heads=0)),
                       ("q_heads", dict(q_heads=2048)), ("scale", dict(scale=0.0)), ("scale", dict(scale=-1.0)),
                       ("scale", dict(scale=math.nan)), ("cap", dict(cap=-1.0)), ("cap", dict(cap=math.inf)),
                       ("cap", dict(cap=3e38)), ("mask", dict(mask="window")), ("prefix", dict(prefix=[1])),
                       ("prefix", dict(mask="causal", prefix=[5])), ("prefix", dict(mask="causal", prefix=[-1])),
                       ("prefix", dict(mask="causal", prefix=[1, 1])), ("begin", dict(q_offsets=[1, 4])),
                       ("fall", dict(k_offsets=[0, -1])), ("fall", dict(q_offsets=[0, 1 << 31])),
                       ("fall", dict(q_offsets=[0, 1 << 30])), ("offsets", dict(q_offsets=[0])),
                       ("offsets", dict(q_offsets=[], k_offsets=[])), ("whole", dict(q_offsets=[0.0, 4.0])),
                       ("slopes", dict(slopes=[1.0] * 4)), ("slopes", dict(slopes=[[1.0]] * 3)),
                       ("axes", dict(slopes=[[1.0] * 4] * 4)), ("finite", dict(slopes=[[math.inf]] * 4)),
                       ("dtype", dict(dtype="fp8")), ("algo", dict(algo="simt")), ("cudaSetDevice", dict(device=-1))]:
        refused(match, TokenAttention, **(good | bad))
    assert fake.fake_live() == 0


def test_attention_run_refusals(fake):
    op = TokenAttention([0, 100], [0, 100], 2, 1, 64, slopes=[[0.5], [0.25]])
    q, k, v, o, p = (BASE + i * MB for i in range(5))
    ok = dict(q_ptr=q, k_ptr=k, v_ptr=v, out_ptr=o, q_pos_ptr=p, k_pos_ptr=p)
    before = fake.fake_launches()
    for match, bad in [("null", dict(q_ptr=0)), ("null", dict(v_ptr=0)), ("null", dict(out_ptr=0)),
                       ("positions", dict(q_pos_ptr=0)), ("positions", dict(k_pos_ptr=0)),
                       ("4-byte", dict(k_lens_ptr=p + 2)), ("16-byte", dict(q_ptr=q + 8)),
                       ("16-byte", dict(k_strides=(68, 64))), ("16-byte", dict(q_strides=(128, 60))),
                       ("stride", dict(v_strides=(-64, 64))), ("overlap one another", dict(out_strides=(64, 64))),
                       ("overlaps an input", dict(out_ptr=q)), ("overlaps an input", dict(out_ptr=k + 128)),
                       ("overlaps an input", dict(out_ptr=p)),
                       ("overlaps an input", dict(k_lens_ptr=o + 256)), ("device 1", dict(stream=0x1000))]:
        refused(match, op.run, **(ok | bad))
    assert fake.fake_launches() == before
    op.run(**ok)
    # q, k, v and out as slices of one row of 5 * 64
    op.run(q, q + 256, q + 384, q + 512, p, p, q_strides=(384, 64), k_strides=(384, 64), v_strides=(384, 64),
           out_strides=(384, 64))
    assert fake.fake_launches() == before + 2


def test_empty_plans_launch_nothing(fake):
    before = fake.fake_launches()
    TokenAttention([0], [0], 1, 1, 8).run(0, 0, 0, 0)
    TokenAttention([0, 0], [0, 4], 1, 1, 8).run(0, BASE, BASE, 0)
    assert fake.fake_launches() == before


def test_the_callers_device_is_kept(fake):
    fake.cudaSetDevice(1)
    op = TokenNorm(64, device=0)
    assert fake.fake_device() == 1
    op.run(4, BASE, norm_ptr=BASE + MB)
    assert fake.fake_device() == 1
    op.close()
    assert fake.fake_device() == 1
    fake.cudaSetDevice(0)


def test_handles_free_their_memory(fake):
    before = fake.fake_live()
    ops = [TokenNorm(8, pre_weight=np.ones(8)), AxisRotary(8, [8]), TokenAttention([0, 9], [0, 9], 1, 1, 8)]
    assert fake.fake_live() > before
    for op in ops:
        op.close()
        op.close()
    assert fake.fake_live() == before
