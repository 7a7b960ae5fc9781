"""Token operators at the edges of what they accept, on the GPU against the float64 definitions."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from arthip_b200.native import lib  # noqa: E402
from arthip_b200.token_ops import TokenAttention  # noqa: E402
from test_token_ops_gpu import gen, ptr, randn, run_attn, run_norm, stream  # noqa: E402
from token_ref import attn_ref, check  # noqa: E402


# 4097 to 4607: more elements than 16 a lane of the widest group, fewer than 18
@pytest.mark.parametrize("c", [1025, 1026, 2049, 4095, 4097, 4098, 4303, 4351, 4606, 4607, 4609, 5121, 8191])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_norm_wide_odd_rows(c, dtype):
    run_norm(19, c, dtype, post="layer", pre="rms", seed=c)


@pytest.mark.parametrize("c", [4100, 4352, 4600, 4608])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_wide_rows_of_odd_pitch(c, in_place):
    run_norm(21, c, "bf16", "rms", "layer", gate=True, strides=1, in_place=in_place, seed=c)


def test_norm_wide_odd_rows_modulated():
    run_norm(20, 4303, "fp16", "layer", "layer", gate=True, gate_act="sigmoid", rows_per_gate=7, mod=True,
             rows_per_mod=7, seed=1)


@pytest.mark.parametrize("d", [40, 64, 72, 128])
@pytest.mark.parametrize("n", [97, 130, 161, 255, 289])
def test_attention_ragged_last_tiles_of_wide_heads(n, d):
    """Lanes behind the last query take part in every load of a head of several loads."""
    run_attn([n], [200], 2, 1, d, "bf16", seed=n)
    run_attn([n, 31], [n, 140], 2, 2, d, "fp16", causal=True, seed=d)


@pytest.mark.parametrize("stall", [0, 1, 2, 5, 8])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bias", [False, True])
def test_attention_wait_that_runs_out_is_reported_and_recovers(stall, d, bias):
    """Failure detection without a GPU fault: every block arms the slot of one load of keys or
    values without loading it, so the waits on it (shortened to 50 ms) run out. The kernel must
    drain, free its tensor memory and say so in the error word, and the same handle must then run
    correctly."""
    g = gen(stall)
    q, k, v = randn(g, (300, 2, d), "fp16"), randn(g, (700, 2, d), "fp16"), randn(g, (700, 2, d), "fp16")
    q_pos, k_pos = (torch.rand(1, n, generator=g, device="cuda") for n in (300, 700))
    slopes = np.full((2, 1), 0.5, dtype=np.float32) if bias else None
    out = torch.empty_like(q)
    op = TokenAttention([0, 300], [0, 700], 2, 2, d, slopes=slopes, algo="tc")

    def run():
        op.run(ptr(q), ptr(k), ptr(v), ptr(out), ptr(q_pos) if bias else 0, ptr(k_pos) if bias else 0, stream=stream())

    lib().ah_test_set_attn_fault_hook(50, stall)
    try:
        run()
        assert op.status() != 0, "a wait that cannot complete must be reported"
    finally:
        lib().ah_test_set_attn_fault_hook(0, -1)
    out.fill_(7.0)
    run()
    assert op.status() == 0
    ref, bound = attn_ref(q, k, v, [0, 300], [0, 700], d ** -0.5, slopes=slopes, q_pos=q_pos, k_pos=k_pos)
    check(out, ref, bound, "fp16", "after recovery")
