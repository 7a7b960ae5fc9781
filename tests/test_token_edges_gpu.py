"""Token operators at the edges of what they accept, on the GPU against the float64 definitions."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_token_ops_gpu import run_attn, run_norm  # noqa: E402


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
