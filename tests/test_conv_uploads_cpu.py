"""When a conv layer's handle is there, its weights are on the device: the C boundary (capi.cc)
linked with a stand-in for the CUDA runtime whose copies from the host and fills arrive only when
something waits for them. Nothing else of the library is linked, as creation calls nothing else."""

from __future__ import annotations

import subprocess
from pathlib import Path

import pytest

from arthip_b200 import build

HOST = r"""
#include <cuda_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>
#include "arthip_b200.h"
#include "kernels/kernels.h"
struct Pending { void* dst; std::vector<char> data; };
static std::vector<Pending> g_pending;
static void arrive() {
  for (const Pending& p : g_pending) std::memcpy(p.dst, p.data.data(), p.data.size());
  g_pending.clear();
}
extern "C" {
cudaError_t cudaSetDevice(int) { return cudaSuccess; }
cudaError_t cudaGetLastError() { return cudaSuccess; }
cudaError_t cudaDeviceGetAttribute(int* v, cudaDeviceAttr, int) { *v = 148; return cudaSuccess; }
cudaError_t cudaMalloc(void** p, size_t n) { *p = std::calloc(n, 1); return cudaSuccess; }
cudaError_t cudaFree(void* p) { arrive(); std::free(p); return cudaSuccess; }
cudaError_t cudaMemcpy(void* d, const void* s, size_t n, cudaMemcpyKind kind) {
  const char* from = static_cast<const char*>(s);
  if (kind == cudaMemcpyHostToDevice) {
    g_pending.push_back({d, std::vector<char>(from, from + n)});
  } else {
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
}
static char g_weights[64];
static uint32_t* g_status = nullptr;
static cudaError_t upload() { return cudaMemcpy(g_weights, "weights", 8, cudaMemcpyHostToDevice); }
namespace ah {
bool conv_tc_supported(int C, int, std::string*) { return C >= 16; }
bool wino_supported(int, int) { return true; }
bool pair_supported(int, int) { return true; }
cudaError_t conv_tc_upload(const uint16_t*, const float*, int, int, ConvTcWeights*) { return upload(); }
cudaError_t simt_conv_upload(const uint16_t*, const float*, int, int, SimtConvWeights*) { return upload(); }
cudaError_t wino_upload(const uint16_t*, const float*, int, int, WinoWeights*) { return upload(); }
cudaError_t pair_upload(const uint16_t*, const float*, int, int, PairWeights*) { return upload(); }
void conv_tc_free(ConvTcWeights*) {}
void simt_conv_free(SimtConvWeights*) {}
void wino_free(WinoWeights*) {}
void pair_free(PairWeights*) {}
cudaError_t simt_conv_launch(const SimtConvWeights&, const __half*, int, int, const __half*, const __half*, int,
                             const SimtOut&, cudaStream_t) { return cudaSuccess; }
bool wino_plan(const WinoWeights*, const __half*, int, int, __half*, int, WinoPlan*, std::string*) { return true; }
cudaError_t wino_launch(const WinoPlan&, const __half*, const __half*, int, uint32_t* status, cudaStream_t) {
  g_status = status;
  return cudaSuccess;
}
}
int main() {
  std::vector<uint16_t> w(64 * 64 * 9);
  const int forms[][2] = {{64, 0}, {1, 0}, {64, 1}, {64, 2}};  // channels, algo
  for (const auto& f : forms) {
    ah_conv* c = nullptr;
    if (ah_conv3x3_create_algo(0, f[0], 64, w.data(), nullptr, 0, f[1], &c, nullptr, 0)) return 2;
    std::printf("created %zu\n", g_pending.size());
    arrive();
    if (f[1] == 1) {
      if (ah_conv3x3_run(c, w.data(), 8, 8, nullptr, nullptr, w.data(), nullptr, nullptr, 0)) return 3;
      *g_status = 1;
      uint32_t got = 0;
      if (ah_conv3x3_status(c, &got) || got != 1) return 4;
      std::printf("cleared %zu\n", g_pending.size());
      arrive();
      if (ah_conv3x3_status(c, &got) || got != 0) return 5;
    }
    ah_conv3x3_destroy(c);
  }
}
"""


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    td = tmp_path_factory.mktemp("conv_uploads")
    (td / "host.cc").write_text(HOST)
    cuda = Path(build.nvcc()).resolve().parents[1]
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(build.CSRC), "-I", str(build.ROOT / "include"), "-I",
                        str(cuda / "include"), "-Wl,--unresolved-symbols=ignore-all", str(build.CSRC / "capi.cc"),
                        str(td / "host.cc"), "-o", str(td / "host")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(td / "host")], capture_output=True, text=True)
    assert r.returncode == 0, r.returncode
    return r.stdout.splitlines()


def test_uploads_have_arrived_when_a_handle_is_there(lines):
    """Tensor-core, plain, Winograd and two-SM form: the first run may follow at once on a stream
    that nothing orders behind the uploads."""
    assert [l for l in lines if l.startswith("created")] == ["created 0"] * 4


def test_status_is_cleared_when_its_read_returns(lines):
    assert [l for l in lines if l.startswith("cleared")] == ["cleared 0"]
