"""The token operators on the GPU against their float64 definitions, with bounds derived from
their roundings (token_ref.py)."""

from __future__ import annotations

import math
import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from arthip_b200.engine import Conv3x3, EngineHarnessError  # noqa: E402
from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm  # noqa: E402
from token_ref import TORCH, attn_ref, check, norm_ref, rope_ref  # noqa: E402


def stream():
    return torch.cuda.current_stream().cuda_stream


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(TORCH[dtype])


def ptr(t):
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------
# Norms
# ---------------------------------------------------------------------------
def run_norm(rows, c, dtype="fp16", post="none", pre="rms", gate=None, gate_act="none", rows_per_gate=1, mod=False,
             rows_per_mod=1, weights=True, with_y=True, seed=0, mean=0.0, strides=None, in_place=False):
    g = gen(seed)
    pad = strides or 0

    def tensor(n):
        t = torch.full((n, c + pad), math.nan, dtype=TORCH[dtype], device="cuda")
        t[:, :c] = randn(g, (n, c), dtype, 1.5) + mean
        return t

    x, y = tensor(rows), tensor(rows) if with_y else None
    gt = tensor((rows - 1) // rows_per_gate + 1) if gate else None
    mrows = (rows - 1) // rows_per_mod + 1
    mods = [randn(g, (mrows, c), dtype, 0.3) for _ in range(2)] if mod else [None, None]
    rng = np.random.default_rng(seed)
    w = {}
    if weights:
        if post != "none":
            w["post_weight"], w["post_bias"] = rng.normal(1, 0.3, c), rng.normal(0, 0.2, c)
        if pre != "none":
            w["pre_weight"], w["pre_bias"] = rng.normal(1, 0.3, c), rng.normal(0, 0.2, c)
        if with_y:
            w["layer_scale"] = rng.normal(0.5, 0.2, c)
    w = {n: v.astype(np.float32) for n, v in w.items()}
    rs = 0.625 if weights and with_y else 1.0
    x0, y0 = x[:, :c].clone(), None if y is None else y[:, :c].clone()
    out = (x if in_place else torch.full_like(x, 7.0)) if with_y else None
    norm = y if in_place and with_y else torch.full_like(x, 7.0)
    op = TokenNorm(c, dtype, post, pre, gate_act=gate_act, residual_scale=rs, **w)
    op.run(rows, ptr(x), ptr(out), ptr(norm), ptr(y), ptr(gt), rows_per_gate, ptr(mods[0]), ptr(mods[1]), rows_per_mod,
           x_stride=c + pad, y_stride=c + pad, gate_stride=c + pad, out_stride=c + pad, norm_stride=c + pad,
           stream=stream())
    torch.cuda.synchronize()
    ro, do, rn, dn = norm_ref(x0, y0, post, pre, gate=None if gt is None else gt[:, :c], gate_act=gate_act,
                              rows_per_gate=rows_per_gate, mod_scale=mods[0], mod_shift=mods[1],
                              rows_per_mod=rows_per_mod, residual_scale=rs, **w)
    if with_y:
        check(out[:, :c], ro, do, dtype, "out")
    check(norm[:, :c], rn, dn, dtype, "norm")
    if pad and not in_place:
        assert (norm[:, c:] == 7).all() and (out is None or (out[:, c:] == 7).all())
    op.close()


@pytest.mark.parametrize("c", [1, 3, 8, 30, 64, 75, 90, 128, 180, 256, 300, 512, 1000, 1152, 2047, 2050, 4096, 5001,
                               8192])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_norm_widths(c, dtype):
    run_norm(37, c, dtype, post="rms", pre="layer", seed=c)


@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("weights", [False, True])
def test_norm_kinds(post, pre, weights):
    run_norm(129, 96, "fp16", post, pre, weights=weights, seed=3)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 257, 40001])
def test_norm_rows(rows):
    run_norm(rows, 64, "fp16", "layer", "rms", seed=rows)


@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh", "silu"])
@pytest.mark.parametrize("rows_per_gate", [1, 7, 50])
def test_norm_gates(act, rows_per_gate):
    run_norm(50, 136, "bf16", "rms", "rms", gate=True, gate_act=act, rows_per_gate=rows_per_gate, seed=5)


@pytest.mark.parametrize("rows_per_mod", [1, 9, 1000])
def test_norm_modulation(rows_per_mod):
    run_norm(45, 640, "bf16", "none", "layer", gate=True, rows_per_gate=rows_per_mod, mod=True,
             rows_per_mod=rows_per_mod, seed=6)


@pytest.mark.parametrize("pad", [1, 2, 8])
@pytest.mark.parametrize("in_place", [False, True])
def test_norm_strides_and_in_place(pad, in_place):
    run_norm(65, 88, "fp16", "rms", "layer", gate=True, strides=pad, in_place=in_place, seed=7)


def test_norm_without_a_block():
    run_norm(77, 192, "fp16", pre="layer", with_y=False, seed=8)


def test_norm_large_mean_keeps_its_digits():
    run_norm(64, 512, "fp16", "layer", "layer", mean=200.0, seed=9)


def test_norm_constant_rows_and_zero_rows():
    op = TokenNorm(64, "fp16", "none", "layer")
    x = torch.ones(5, 64, dtype=torch.float16, device="cuda") * 3
    n = torch.full_like(x, 7)
    op.run(0, ptr(x), 0, ptr(n), stream=stream())
    assert (n == 7).all()
    op.run(5, ptr(x), 0, ptr(n), stream=stream())
    assert (n == 0).all()  # 0 / sqrt(eps)


# ---------------------------------------------------------------------------
# Rotary positions
# ---------------------------------------------------------------------------
def run_rope(tokens, d, dims, layout="halves", dtype="fp16", hq=3, hk=2, theta=10000.0, inverse=False, extra=0,
             in_place=False, head_major=False, offset=0.0, fractional=False, seed=0):
    g = gen(seed)
    row = (hq + hk) * d + extra
    if head_major:
        buf = randn(g, (hq + hk, tokens, d), dtype)
        x = buf.permute(1, 0, 2)
        st, qk_off = (d, tokens * d), hq * tokens * d
    else:
        buf = randn(g, (tokens, row), dtype)
        x = buf[:, :(hq + hk) * d].view(tokens, hq + hk, d) if not extra else \
            buf.as_strided((tokens, hq + hk, d), (row, d, 1))
        st, qk_off = (row, d), hq * d
    pos = torch.randint(0, 3000, (len(dims), tokens), generator=g, device="cuda").float() + offset
    if fractional:
        pos += 0.3125
    before = buf.clone()
    x0 = x.clone()
    op = AxisRotary(d, dims, theta, layout, dtype, inverse)
    q_out = k_out = None
    if not in_place:
        q_out = torch.full((tokens, hq, d), 7.0, dtype=TORCH[dtype], device="cuda")
        k_out = torch.full((tokens, hk, d), 7.0, dtype=TORCH[dtype], device="cuda")
    op.run(tokens, ptr(pos), ptr(buf), hq, ptr(q_out), buf.data_ptr() + 2 * qk_off, hk, ptr(k_out), st, st,
           stream=stream())
    torch.cuda.synchronize()
    ref, bound = rope_ref(x0, pos, dims, theta, layout, inverse)
    got = x if in_place else torch.cat([q_out, k_out], 1)
    check(got, ref, bound, dtype, "rope")
    rest = sum(dims)
    assert torch.equal(got[..., rest:], x0[..., rest:])  # copied as it is
    if not in_place:
        assert torch.equal(buf, before)
    elif extra:
        assert torch.equal(buf[:, -extra:], before[:, -extra:])
    op.close()


@pytest.mark.parametrize("layout", ["halves", "pairs", "shared"])
@pytest.mark.parametrize("d,dims", [(32, [16, 16]), (64, [16, 16, 32]), (128, [44, 42, 42]), (72, [24, 24, 16]),
                                    (80, [16, 32]), (30, [10, 8, 12]), (2, [2]), (128, [128]), (33, [6, 0, 4]),
                                    (512, [256, 128, 128])])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rope_layouts(layout, d, dims, dtype):
    run_rope(41, d, dims, layout, dtype, seed=d)


@pytest.mark.parametrize("tokens", [1, 2, 15, 600, 5000])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rope_tokens(tokens, layout):
    run_rope(tokens, 64, [32, 16, 16], layout, hq=8, hk=2, seed=tokens)


@pytest.mark.parametrize("layout", ["halves", "pairs", "shared"])
@pytest.mark.parametrize("extra", [0, 1, 24])
def test_rope_in_place_and_slices(layout, extra):
    run_rope(70, 48, [16, 32], layout, extra=extra, in_place=True, seed=1)
    run_rope(70, 48, [16, 32], layout, extra=extra, seed=2)


@pytest.mark.parametrize("in_place", [False, True])
def test_rope_head_major(in_place):
    run_rope(33, 64, [32, 32], head_major=True, in_place=in_place, seed=3)


def test_rope_far_and_fractional_positions_and_own_bases():
    # 2^23 - 3000: the last binade in which a half is still a position of its own
    run_rope(50, 64, [32, 32], offset=float(2 ** 23 - 4096), seed=4)
    run_rope(50, 64, [32, 32], fractional=True, theta=(100.0, 1e6), seed=5)


def test_rope_inverse_undoes():
    run_rope(50, 64, [32, 32], inverse=True, seed=6)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def run_attn(qs, ks, hq=4, hk=2, d=64, dtype="fp16", causal=False, prefix=None, cap=0.0, axes=0, lens=None,
             std=1.0, head_major=False, seed=0, garbage=True, scale=None):
    g = gen(seed)
    nq, nk = sum(qs), sum(ks)
    tail = 3  # tokens behind the last document

    def tensor(n, h, s):
        if head_major:
            return randn(g, (h, n + tail, d + 8), dtype, s)[..., :d].permute(1, 0, 2)
        return randn(g, (n + tail, h, d), dtype, s)

    q, k, v = tensor(nq, hq, std), tensor(nk, hk, 1.0), tensor(nk, hk, 1.0)
    out = torch.full((nq + tail, hq, d), 7.0, dtype=TORCH[dtype], device="cuda")
    qo, ko = np.cumsum([0] + qs), np.cumsum([0] + ks)
    q_pos = k_pos = slopes = None
    if axes:
        k_pos = torch.randint(0, 60, (axes, nk), generator=g, device="cuda").float()
        q_pos = torch.randint(0, 60, (axes, nq), generator=g, device="cuda").float()
        slopes = np.random.default_rng(seed).uniform(0.0, 0.2, (hq, axes)).astype(np.float32)
    dl = None
    if lens is not None:
        dl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if garbage:
            for n, u in enumerate(lens):
                a, b = int(ko[n]) + max(0, min(u, ks[n])), int(ko[n + 1])
                k[a:b], v[a:b] = math.nan, math.inf
    if garbage:
        k[nk:], v[nk:] = math.nan, math.nan
    scale = d ** -0.5 if scale is None else scale
    ref, bound = attn_ref(q[:nq], k[:nk], v[:nk], qo, ko, scale, cap, causal, prefix, slopes, q_pos, k_pos, lens,
                          dtype)
    for algo in ("auto", "mma", "tc"):  # the choice by expected time, and each kernel on everything
        op = TokenAttention(qo, ko, hq, hk, d, scale=scale, cap=cap, mask="causal" if causal else "full",
                            prefix=prefix, slopes=slopes, dtype=dtype, algo=algo)
        out.fill_(7.0)
        op.run(ptr(q), ptr(k), ptr(v), ptr(out), ptr(q_pos), ptr(k_pos), ptr(dl), q.stride()[:2], k.stride()[:2],
               v.stride()[:2], stream=stream())
        torch.cuda.synchronize()
        check(out[:nq], ref, bound, dtype, f"attention ({algo})")
        assert (out[nq:] == 7).all()
        assert op.status() == 0
        op.close()


@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_head_dims(d, dtype):
    run_attn([100], [150], d=d, dtype=dtype, seed=d)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 300, 513])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_lengths(n, causal):
    run_attn([n], [n], causal=causal, seed=n)


@pytest.mark.parametrize("nq,nk", [(1, 1), (1, 1000), (3, 129), (5, 64), (200, 7), (130, 1), (64, 4000), (257, 640),
                                   (700, 300)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_unequal_lengths(nq, nk, causal):
    """With more queries than keys a causal mask leaves the first rows nothing: zeros."""
    run_attn([nq], [nk], causal=causal, seed=nq + nk)


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 3), (8, 2), (6, 1), (32, 8), (40, 2)])
@pytest.mark.parametrize("nq", [1, 2, 150])
def test_attention_shared_heads(hq, hk, nq):
    run_attn([nq, nq], [300, 77], hq, hk, 32, causal=True, seed=hq)


RAGGED = [0, 1, 77, 300, 0, 129, 2, 513, 64]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_ragged_documents(dtype, causal):
    run_attn(RAGGED, RAGGED, 6, 2, 64, dtype, causal, seed=1)


def test_attention_documents_without_queries_or_keys():
    run_attn([5, 0, 200, 3, 0], [0, 9, 100, 40, 0], seed=2)
    run_attn([], [], seed=2)
    run_attn([0], [0], seed=2)
    run_attn([4, 170], [0, 0], seed=2)


def test_attention_prefix():
    run_attn(RAGGED, RAGGED, 4, 4, 64, causal=True, prefix=[0, 1, 70, 129, 0, 0, 1, 513, 10], seed=3)
    run_attn([40, 2, 300], [10, 300, 290], 4, 2, 128, causal=True, prefix=[10, 150, 7], seed=4)


@pytest.mark.parametrize("cap", [0.5, 5.0, 50.0, 1000.0, 1e5])
@pytest.mark.parametrize("std", [0.1, 8.0])
def test_attention_cap(cap, std):
    run_attn([150, 1], [170, 90], 4, 2, 64, cap=cap, std=std, seed=5)
    run_attn([200], [300], 4, 2, 64, cap=cap, std=std, causal=True, seed=5)


@pytest.mark.parametrize("axes", [1, 2, 3])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_attention_distance_bias(axes, cap):
    run_attn([150, 1, 300], [170, 90, 300], 4, 2, 64, axes=axes, cap=cap, causal=axes != 1, seed=6)


def test_attention_bias_that_outweighs_the_scores():
    run_attn([300], [900], 2, 2, 32, axes=1, std=30.0, seed=7)


@pytest.mark.parametrize("nq", [1, 3, 140])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_keys_in_use(nq, causal, dtype):
    """Behind the keys in use the cache holds NaN and infinities; lengths outside the
    capacity are clamped."""
    run_attn([nq] * 6, [400, 400, 64, 400, 100, 0], 8, 2, 128, dtype, causal, lens=[0, 1, 63, 257, 5000, -3], seed=8)


def test_attention_prefix_beyond_the_keys_in_use():
    run_attn([2, 150], [400, 400], 2, 2, 64, causal=True, prefix=[300, 390], lens=[100, 200], seed=9)


@pytest.mark.parametrize("nq", [2, 200])
def test_attention_head_major(nq):
    run_attn([nq, 50], [333, 50], 4, 2, 40, head_major=True, causal=True, seed=10)


def test_attention_windows():
    run_attn([64] * 150, [64] * 150, 6, 6, 32, axes=2, seed=11)
    run_attn([49] * 40, [49] * 40, 3, 3, 24, axes=2, seed=12)
    run_attn([256] * 9, [256] * 9, 2, 2, 64, axes=2, seed=13)


def test_attention_long():
    run_attn([2100], [2100], 2, 1, 128, "bf16", causal=True, cap=30.0, axes=3, seed=14)
    run_attn([1, 2], [20000, 9000], 8, 2, 128, "bf16", causal=True, seed=15)
    run_attn([70], [20000], 2, 2, 64, seed=16)
    run_attn([1500], [3000], 3, 3, 80, seed=17)


def test_attention_far_offsets():
    """A cache whose later tokens lie beyond 2^31 elements (and 2^32 bytes)."""
    d, n, pitch = 64, 40000, 65536
    g = gen(18)
    cache = torch.empty(n * pitch, dtype=torch.float16, device="cuda")
    k = cache.as_strided((n, 1, d), (pitch, d, 1))
    v = cache.as_strided((n, 1, d), (pitch, d, 1), d)
    k.copy_(randn(g, (n, 1, d), "fp16"))
    v.copy_(randn(g, (n, 1, d), "fp16"))
    for nq, algo in ((1, "mma"), (150, "mma"), (150, "tc")):
        q = randn(g, (nq, 1, d), "fp16", 3.0)
        out = torch.empty_like(q)
        op = TokenAttention([0, nq], [0, n], 1, 1, d, algo=algo)
        op.run(ptr(q), ptr(k), ptr(v), ptr(out), k_strides=(pitch, d), v_strides=(pitch, d), stream=stream())
        ref, bound = attn_ref(q, k, v, [0, nq], [0, n], d ** -0.5)
        check(out, ref, bound, "fp16", "far offsets")


@pytest.mark.parametrize("algo", ["mma", "tc"])
def test_attention_nan_stays_in_its_document(algo):
    qs = [64, 70, 300, 1]
    off = np.cumsum([0] + qs)
    g = gen(19)
    q, k, v = (randn(g, (int(off[-1]), 2, 32), "fp16") for _ in range(3))
    op = TokenAttention(off, off, 2, 2, 32, algo=algo)
    a, b = torch.empty_like(q), torch.empty_like(q)
    op.run(ptr(q), ptr(k), ptr(v), ptr(a), stream=stream())
    k[off[1]:off[2]] = math.nan
    v[off[1]:off[2]] = math.inf
    op.run(ptr(q), ptr(k), ptr(v), ptr(b), stream=stream())
    for n in (0, 2, 3):
        assert torch.equal(a[off[n]:off[n + 1]], b[off[n]:off[n + 1]])
    assert torch.isnan(b[off[1]:off[2]]).all()


def test_attention_repeats_bit_for_bit():
    g = gen(20)
    for nq, nk, algo in ((1, 9000, "auto"), (500, 500, "tc"), (500, 500, "mma"), (64, 3000, "mma")):
        q, k, v = randn(g, (nq, 8, 64), "bf16"), randn(g, (nk, 2, 64), "bf16"), randn(g, (nk, 2, 64), "bf16")
        op = TokenAttention([0, nq], [0, nk], 8, 2, 64, dtype="bf16", algo=algo)
        outs = []
        for _ in range(4):
            out = torch.empty_like(q)
            op.run(ptr(q), ptr(k), ptr(v), ptr(out), stream=stream())
            outs.append(out)
        assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("algo", ["mma", "tc"])
@pytest.mark.parametrize("where", ["q", "k", "v"])
def test_attention_infinities_and_nan_in_use_show(algo, where):
    """A NaN or infinity that a row sees makes that row NaN or infinite, and no other row's query
    is touched by one in q."""
    for value in (math.nan, math.inf):
        g = gen(24)
        t = {n: randn(g, (200, 1, 64), "fp16") for n in ("q", "k", "v")}
        t[where][77] = value
        out = torch.zeros(200, 1, 64, dtype=torch.float16, device="cuda")
        op = TokenAttention([0, 200], [0, 200], 1, 1, 64, algo=algo)
        op.run(ptr(t["q"]), ptr(t["k"]), ptr(t["v"]), ptr(out), stream=stream())
        bad = ~torch.isfinite(out).all(-1)[:, 0]
        if where == "q":
            assert bad.nonzero().flatten().tolist() == [77]
        elif where == "v" or value != value:
            assert bad.all()


# ---------------------------------------------------------------------------
# Graphs, streams, threads
# ---------------------------------------------------------------------------
FIRST_CALL_CAPTURED = """
import sys, torch
sys.path.insert(0, {root!r})
from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm
x = torch.randn(200, 2, 64, device="cuda").half()
outs = [torch.zeros_like(x) for _ in range(4)]
pos = torch.zeros(1, 200, device="cuda")
off = [0, 200]
ops = [TokenNorm(128), AxisRotary(64, [64]), TokenAttention(off, off, 2, 2, 64, algo="mma"),
       TokenAttention(off, off, 2, 2, 64, algo="tc")]
p, o = x.data_ptr(), [t.data_ptr() for t in outs]
def run(s):
    ops[0].run(200, p, 0, o[0], stream=s)
    ops[1].run(200, pos.data_ptr(), p, 2, o[1], stream=s)
    ops[2].run(p, p, p, o[2], stream=s)
    ops[3].run(p, p, p, o[3], stream=s)
side = torch.cuda.Stream()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=side):
    run(side.cuda_stream)
assert all((t == 0).all() for t in outs)
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in outs]
run(torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert all(torch.equal(a, b) and (a != 0).any() for a, b in zip(got, outs))
print("captured first calls ok")
"""


def test_first_calls_of_a_process_may_be_captured():
    """Kernels load, and their attributes are set, on a first call: also under capture."""
    import subprocess
    import sys
    from pathlib import Path
    root = str(Path(__file__).resolve().parents[1])
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED.format(root=root)], capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "captured first calls ok" in r.stdout, r.stderr[-2000:]


def test_captured_run_follows_the_cache():
    """One graph, replayed while k_lens grows and after the inputs change."""
    d, cap_len = 64, 700
    g = gen(21)
    q, out = randn(g, (2, 4, d), "fp16"), torch.empty(2, 4, d, dtype=torch.float16, device="cuda")
    k, v = randn(g, (2 * cap_len, 2, d), "fp16"), randn(g, (2 * cap_len, 2, d), "fp16")
    lens = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    op = TokenAttention([0, 1, 2], [0, cap_len, 2 * cap_len], 4, 2, d, mask="causal")
    rope = AxisRotary(d, [32, 32])
    pos = torch.zeros(2, 2, device="cuda")
    turned = torch.empty_like(q)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        rope.run(2, ptr(pos), ptr(q), 4, ptr(turned), stream=side.cuda_stream)
        op.run(ptr(turned), ptr(k), ptr(v), ptr(out), k_lens_ptr=ptr(lens), stream=side.cuda_stream)
    for step in (1, 64, 65, 699):
        lens.copy_(torch.tensor([step, cap_len - step], dtype=torch.int32))
        pos.fill_(float(step))
        q.copy_(randn(g, (2, 4, d), "fp16"))
        graph.replay()
        torch.cuda.synchronize()
        ref, bound = rope_ref(q, pos, [32, 32])
        check(turned, ref, bound, "fp16", "captured rope")
        ref, bound = attn_ref(turned, k, v, [0, 1, 2], [0, cap_len, 2 * cap_len], d ** -0.5, causal=True,
                              k_lens=[step, cap_len - step])
        check(out, ref, bound, "fp16", "captured attention")


def test_one_handle_on_two_streams_and_threads():
    g = gen(22)
    qo, ko = [0, 1, 301], [0, 5000, 5300]
    op = TokenAttention(qo, ko, 4, 2, 64)
    sets = [[randn(g, (301, 4, 64), "fp16"), randn(g, (5300, 2, 64), "fp16"), randn(g, (5300, 2, 64), "fp16")]
            for _ in range(2)]
    wants = []
    for q, k, v in sets:
        out = torch.empty_like(q)
        op.run(ptr(q), ptr(k), ptr(v), ptr(out), stream=stream())
        wants.append(out)
    torch.cuda.synchronize()
    outs = [torch.zeros_like(w) for w in wants]
    streams = [torch.cuda.Stream() for _ in range(2)]
    errors = []

    def work(i):
        try:
            q, k, v = sets[i]
            for _ in range(20):
                op.run(ptr(q), ptr(k), ptr(v), ptr(outs[i]), stream=streams[i].cuda_stream)
        except Exception as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not errors and all(torch.equal(a, b) for a, b in zip(outs, wants))


def test_two_graphs_of_one_handle_run_side_by_side():
    """Split keys are joined without a workspace, so graphs of one handle share nothing."""
    g = gen(25)
    op = TokenAttention([0, 1], [0, 30000], 4, 2, 64)
    sets = [[randn(g, (1, 4, 64), "fp16"), randn(g, (30000, 2, 64), "fp16"), randn(g, (30000, 2, 64), "fp16")]
            for _ in range(2)]
    outs, wants, graphs, streams = [], [], [], []
    for q, k, v in sets:
        want, out = torch.empty_like(q), torch.zeros_like(q)
        op.run(ptr(q), ptr(k), ptr(v), ptr(want), stream=stream())
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(20):
                op.run(ptr(q), ptr(k), ptr(v), ptr(out), stream=side.cuda_stream)
        outs.append(out), wants.append(want), graphs.append(graph), streams.append(side)
    for _ in range(5):
        for graph, side in zip(graphs, streams):
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, wants))


def test_run_refusals_launch_nothing():
    q = torch.zeros(64, 2, 32, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, 7.0)
    op = TokenAttention([0, 64], [0, 64], 2, 2, 32)
    for bad in (dict(k_ptr=0), dict(out_ptr=ptr(q)), dict(q_ptr=ptr(q) + 2), dict(q_strides=(65, 32)),
                dict(q_strides=(-64, 32)), dict(out_strides=(32, 32))):
        args = dict(q_ptr=ptr(q), k_ptr=ptr(q), v_ptr=ptr(q), out_ptr=ptr(out), stream=stream()) | bad
        with pytest.raises(EngineHarnessError):
            op.run(**args)
    norm = TokenNorm(64)
    with pytest.raises(EngineHarnessError):
        norm.run(64, ptr(q), 0, ptr(q) + 128, stream=stream())
    rope = AxisRotary(32, [32])
    with pytest.raises(EngineHarnessError):
        rope.run(64, ptr(out), ptr(q), 2, ptr(q) + 64, stream=stream())
    torch.cuda.synchronize()
    assert (out == 7).all() and (q == 0).all()


@pytest.mark.parametrize("args", [["--op", "norm"], ["--op", "rope"], ["--op", "attention"],
                                  ["--op", "attention", "--window", "0"]])
def test_layerbench_times_the_operators(args, capsys):
    import json
    from arthip_b200 import layerbench
    assert layerbench.main(args + ["--C", "96", "--H", "40", "--W", "64", "--iters", "2"]) == 0
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert line["us_per_launch"] > 0 and line["algorithmic_bytes"] > 0 and line["status"] == 0


# ---------------------------------------------------------------------------
# A token block between conv layers
# ---------------------------------------------------------------------------
def test_conv_rope_attention_norm_together():
    """A 24x40 frame: Conv3x3 makes q, k and v (64 -> 192 channels), q and k turn in place by
    row and column, 8x8 windows attend with a distance bias, Conv3x3 projects, and the norm
    adds the block to the frame under its gate. Each stage is checked on the stage before
    it as the library left it."""
    H, W, C, heads = 24, 40, 64, 2
    d = C // heads
    n = H * W
    rng = np.random.default_rng(23)
    wq = (rng.standard_normal((3 * C, C, 3, 3)) * 0.06).astype(np.float16)
    wo = (rng.standard_normal((C, C, 3, 3)) * 0.06).astype(np.float16)
    g = gen(23)
    frame = randn(g, (n, C), "fp16")
    gate = randn(g, (1, C), "fp16")
    # window order: tokens of one 8x8 window follow one another
    at = torch.arange(n, device="cuda").view(H // 8, 8, W // 8, 8).permute(0, 2, 1, 3).reshape(-1)
    pos = torch.stack([at // W, at % W]).float().contiguous()
    pre = TokenNorm(C, pre_norm="layer")
    qkv_conv, out_conv = Conv3x3(wq, None), Conv3x3(wo, None)
    rope = AxisRotary(d, [16, 16])
    off = np.arange(0, n + 1, 64)
    slopes = np.array([[0.1, 0.1], [0.02, 0.05]], dtype=np.float32)
    attn = TokenAttention(off, off, heads, heads, d, slopes=slopes)
    post = TokenNorm(C, post_norm="rms", pre_norm="layer", gate_act="tanh", residual_scale=0.5)
    s = stream()
    normed, qkv, mixed, block, out, nxt = (torch.empty(n, c, dtype=torch.float16, device="cuda")
                                           for c in (C, 3 * C, C, C, C, C))
    pre.run(n, ptr(frame), 0, ptr(normed), stream=s)
    qkv_conv.run(ptr(normed), H, W, ptr(qkv), stream=s)
    win = qkv[at].contiguous()
    before = win.clone()
    st = (3 * C, d)
    rope.run(n, ptr(pos), ptr(win), heads, k_ptr=ptr(win) + 2 * C, k_heads=heads, q_strides=st, k_strides=st, stream=s)
    attn.run(ptr(win), ptr(win) + 2 * C, ptr(win) + 4 * C, ptr(mixed), ptr(pos), ptr(pos), q_strides=st, k_strides=st,
             v_strides=st, stream=s)
    back = torch.empty_like(mixed)
    back[at] = mixed
    out_conv.run(ptr(back), H, W, ptr(block), stream=s)
    post.run(n, ptr(frame), ptr(out), ptr(nxt), ptr(block), ptr(gate), rows_per_gate=n, stream=s)
    torch.cuda.synchronize()
    assert qkv_conv.status() == 0 and out_conv.status() == 0
    ref, bound = norm_ref(frame, pre="layer")[2:]
    check(normed, ref, bound, "fp16", "pre-norm")
    qk = before[:, :2 * C].view(n, 2 * heads, d)
    ref, bound = rope_ref(qk, pos, [16, 16])
    check(win[:, :2 * C].view(n, 2 * heads, d), ref, bound, "fp16", "rope")
    assert torch.equal(win[:, 2 * C:], before[:, 2 * C:])
    parts = [win[:, i * C:(i + 1) * C].reshape(n, heads, d) for i in range(3)]
    ref, bound = attn_ref(*parts, off, off, d ** -0.5, slopes=slopes, q_pos=pos, k_pos=pos)
    check(mixed.view(n, heads, d), ref, bound, "fp16", "attention")
    ro, do, rn, dn = norm_ref(frame, block, "rms", "layer", gate=gate, gate_act="tanh", rows_per_gate=n,
                              residual_scale=0.5)
    check(out, ro, do, "fp16", "block out")
    check(nxt, rn, dn, "fp16", "next norm")
