"""Token operators at the edges of what they accept, on the GPU against the float64 definitions."""

from __future__ import annotations

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from arthip_b200.native import lib  # noqa: E402
from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm  # noqa: E402
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


def infinite_key(nq, nk, d, dtype, seed):
    """q, k, v of one head, key 77 with an infinity in element 5 where every query is 1 to 2 or -1
    to -2, and which queries see it as +inf."""
    g = gen(seed)
    q, k, v = (randn(g, (n, 1, d), dtype) for n in (nq, nk, nk))
    sign = torch.where(torch.rand(nq, generator=g, device="cuda") < 0.5, -1.0, 1.0)
    sign[0], sign[-1] = 1.0, -1.0
    q[:, 0, 5] = (sign * (1 + torch.rand(nq, generator=g, device="cuda"))).to(q.dtype)
    k[77, 0, 5] = math.inf
    return q, k, v, sign > 0


# Queries, keys: the tcgen05 form, 64 rows a block with and without a cluster, 16 rows likewise
INFINITE = [(200, 300, "tc"), (200, 300, "mma"), (64, 4000, "mma"), (3, 300, "mma"), (3, 9000, "mma")]


@pytest.mark.parametrize("nq,nk,algo", INFINITE)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_infinite_key(nq, nk, algo, d, dtype):
    """A score of +inf makes its row NaN, as inf - inf in its softmax does; one of -inf is a key of no
    weight."""
    q, k, v, plus = infinite_key(nq, nk, d, dtype, nq + nk)
    out = torch.zeros_like(q)
    op = TokenAttention([0, nq], [0, nk], 1, 1, d, dtype=dtype, algo=algo)
    op.run(ptr(q), ptr(k), ptr(v), ptr(out), stream=stream())
    assert torch.isnan(out[plus]).all()
    rest = [torch.cat([t[:77], t[78:]]) for t in (k, v)]
    ref, bound = attn_ref(q[~plus], *rest, [0, int((~plus).sum())], [0, nk - 1], d ** -0.5, dtype=dtype)
    check(out[~plus], ref, bound, dtype, "rows of a score of -inf")


@pytest.mark.parametrize("nq,nk,algo", INFINITE)
@pytest.mark.parametrize("cap", [5.0, 1000.0])
def test_attention_infinite_key_under_a_cap(nq, nk, algo, cap):
    """A cap makes an infinite score the cap, or minus the cap."""
    q, k, v, plus = infinite_key(nq, nk, 64, "fp16", nq + nk)
    out = torch.zeros_like(q)
    op = TokenAttention([0, nq], [0, nk], 1, 1, 64, cap=cap, algo=algo)
    op.run(ptr(q), ptr(k), ptr(v), ptr(out), stream=stream())
    if cap == 1000.0:  # exp(-990) of anything else is left: the row is that key's value, or without it
        assert torch.equal(out[plus], v[77:78].expand(int(plus.sum()), 1, 64))
        rest = [torch.cat([t[:77], t[78:]]) for t in (k, v)]
        ref, bound = attn_ref(q[~plus], *rest, [0, int((~plus).sum())], [0, nk - 1], 0.125, cap)
        check(out[~plus], ref, bound, "fp16", "rows of a score of -cap")
    else:
        # 2^9 gives scores of some 64 or more, 12 caps: 1 - tanh 12 = 8e-11. (The infinite score is the
        # cap exactly; the bound's term for a product sum, 68 E 2^9 2 / 8 = 5e-4, is to spare.)
        k[77, 0, 5] = 2.0 ** 9
        ref, bound = attn_ref(q, k, v, [0, nq], [0, nk], 0.125, cap)
        check(out, ref, bound, "fp16", "rows of a score of the cap")


def test_runs_of_no_tokens_do_nothing():
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    pos = torch.empty(1, 0, device="cuda")
    assert x.data_ptr() == 0
    TokenNorm(64).run(0, ptr(x), ptr(x), ptr(x), ptr(x), stream=stream())
    AxisRotary(64, [64]).run(0, ptr(pos), ptr(x), 1, stream=stream())
    TokenAttention([0, 0], [0, 0], 1, 1, 64).run(ptr(x), ptr(x), ptr(x), ptr(x), stream=stream())
    torch.cuda.synchronize()


@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("nq", [3, 70])
def test_attention_widest_clusters(nq, d):
    """Few blocks on long caches: the keys are shared out over clusters of sixteen."""
    run_attn([nq], [20000], 1, 1, d, "bf16", causal=True, lens=[19001], seed=d)


@pytest.mark.parametrize("hq,hk", [(1024, 1), (1024, 1024), (1023, 341)])
@pytest.mark.parametrize("nq", [1, 130])
def test_attention_most_heads(hq, hk, nq):
    run_attn([nq], [140], hq, hk, 8, causal=True, seed=hq + nq)
