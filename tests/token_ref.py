"""The token operators' definitions in float64, with the error bounds that their arithmetic
allows, for the tests of ``arthip_b200.token_ops``.

A value written as fp16 or bf16 is off by at most U[dtype] of itself (half a step) or, for
fp16, half of the smallest subnormal. In between, everything is fp32: E = 2^-24 a rounding."""

from __future__ import annotations

import math

import numpy as np
import torch

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134}
E = 2.0 ** -24


def norm_ref(x, y=None, post="none", pre="rms", post_weight=None, post_bias=None, pre_weight=None, pre_bias=None,
             layer_scale=None, residual_scale=1.0, gate=None, gate_act="none", rows_per_gate=1, mod_scale=None,
             mod_shift=None, rows_per_mod=1, post_eps=1e-6, pre_eps=1e-6):
    """(out, its fp32 error bound, norm, its bound), all float64 [rows][channels].

    Bounds. A row's sums run over at most 64 values a lane and 10 steps across lanes, so a
    mean or mean square is off by under 74 E of the mean magnitude, its root by half of that;
    with the elementwise roundings each normed value is off by at most 96 E of
    (|value| + root mean square before centring) / sigma, plus what its input was off by
    (which reaches a row's value directly and through the mean and sigma: at most three times
    the row's largest). sigmoid and tanh are good to 8 E."""
    k = 96 * E

    def stat(v, dv, kind, w, b, eps):
        w = 1.0 if w is None else torch.as_tensor(w, device=v.device).double()
        b = torch.zeros(1, dtype=torch.float64, device=v.device) if b is None else torch.as_tensor(b, device=v.device).double()
        if kind == "none":
            n, dn = v, dv
        else:
            raw = v.square().mean(1, keepdim=True).sqrt()
            c = v - v.mean(1, keepdim=True) if kind == "layer" else v
            sigma = (c.square().mean(1, keepdim=True) + eps).sqrt()
            n = c / sigma
            rel = dv.amax(1, keepdim=True) / sigma
            dn = k * (n.abs() + raw / sigma) + 2 * rel + rel * n.abs()
            # a centred row much smaller than its mean: its sigma is off too
            dn = dn + n.abs() * k * raw / sigma
        out = n * w + b
        return out, dn * (abs(w) if isinstance(w, float) else w.abs()) + 4 * E * (out.abs() + b.abs())

    x = x.double()
    rows = torch.arange(x.shape[0], device=x.device)
    out, dout = x, torch.zeros_like(x)
    if y is not None:
        b, db = stat(y.double(), torch.zeros_like(x), post, post_weight, post_bias, post_eps)
        s = residual_scale * (1.0 if layer_scale is None else torch.as_tensor(layer_scale, device=x.device).double())
        b, db = b * s, db * abs(s) + 4 * E * (b * s).abs()
        if gate is not None:
            g = gate.double()[rows // rows_per_gate]
            g = {"none": g, "sigmoid": torch.sigmoid(g), "tanh": torch.tanh(g), "silu": g * torch.sigmoid(g)}[gate_act]
            b, db = b * g, db * g.abs() + 16 * E * (b * g).abs()
        out = x + b
        dout = db + 2 * E * (x.abs() + b.abs())
    n, dn = stat(out, dout, pre, pre_weight, pre_bias, pre_eps)
    if mod_scale is not None:
        m = 1 + mod_scale.double()[rows // rows_per_mod]
        n, dn = n * m, dn * m.abs() + 4 * E * n.abs() * (1 + m.abs())
    if mod_shift is not None:
        m = mod_shift.double()[rows // rows_per_mod]
        n, dn = n + m, dn + 2 * E * (n.abs() + m.abs())
    return out, dout, n, dn


def rope_ref(x, pos, dims, theta=10000.0, layout="halves", inverse=False):
    """x [tokens][heads][dim], pos [axes][tokens]; (out, bound): the cosine and sine come from
    turns rounded to fp32 (at most half a turn, so 2 pi E off) and are good to 4 E more."""
    x = x.double()
    out, bound = x.clone(), torch.zeros_like(x)
    thetas = [theta] * len(dims) if np.isscalar(theta) else theta
    total, base = sum(dims), 0
    for a, n in enumerate(dims):
        for j in range(n // 2):
            if layout == "pairs":
                e0, e1, f = base + 2 * j, base + 2 * j + 1, thetas[a] ** (-2.0 * j / n)
            elif layout == "halves":
                e0, e1, f = base + j, base + j + n // 2, thetas[a] ** (-2.0 * j / n)
            else:
                p = base // 2 + j
                e0, e1, f = p, p + total // 2, thetas[a] ** (-2.0 * p / total)
            ang = pos[a].double() * (-f if inverse else f)
            c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
            u, v = x[..., e0], x[..., e1]
            out[..., e0], out[..., e1] = u * c - v * s, u * s + v * c
            bound[..., e0] = bound[..., e1] = 14 * E * (u.abs() + v.abs())
        base += n
    return out, bound


def attn_ref(q, k, v, q_off, k_off, scale, cap=0.0, causal=False, prefix=None, slopes=None, q_pos=None, k_pos=None,
             k_lens=None, dtype="fp16"):
    """(out, bound) as float64 [queries][heads][dim]; tokens outside every document are NaN in
    both.

    Bound. A score's fp32 product sum is off by at most (dim + 4) E of the sum of its terms'
    magnitudes, the cap by 8 E cap and 2 E of the score, the bias by 4 E of its terms; the
    running maximum enters as a difference (2 E of both). So a weight is off by that (d) as a
    relative error, and by U when it is rounded for the second product, or TINY where it
    falls below the type's normal range. With A = sum p |v| / sum p, the result is off by
    (U + 2 d + 64 E) A + TINY sum |v| and its own rounding."""
    hq, group = q.shape[1], q.shape[1] // k.shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    bound = out.clone()
    for n in range(len(q_off) - 1):
        q0, q1, k0, k1 = int(q_off[n]), int(q_off[n + 1]), int(k_off[n]), int(k_off[n + 1])
        nk = k1 - k0 if k_lens is None else max(0, min(int(k_lens[n]), k1 - k0))
        nq = q1 - q0
        if nq == 0:
            continue
        i = torch.arange(nq, device=q.device)[:, None]
        j = torch.arange(nk, device=q.device)[None]
        seen = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            seen = (j <= i + nk - nq) | (j < (0 if prefix is None else int(prefix[n])))
        for h in range(hq):
            kk, vv = k[k0:k0 + nk, h // group].double(), v[k0:k0 + nk, h // group].double()
            qq = q[q0:q1, h].double()
            s = qq @ kk.T * scale
            d = (q.shape[2] + 4) * E * scale * (qq.abs() @ kk.abs().T)
            if cap:
                s = cap * torch.tanh(s / cap)
                d = d + 8 * E * cap + 2 * E * s.abs()
            for a in range(0 if slopes is None else len(slopes[h])):
                b = float(slopes[h][a]) * (q_pos[a, q0:q1, None].double() - k_pos[a, None, k0:k0 + nk].double()).abs()
                s = s - b
                d = d + 4 * E * b.abs() + 2 * E * s.abs()
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True) if nk else s.new_zeros(nq, 1)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            inv = torch.where(total > 0, 1 / total, torch.zeros_like(total))
            o = p @ vv * inv
            worst = (torch.where(seen & (p > 1e-9), d + 4 * E * (s.abs() + top.abs()), 0.0).amax(1, keepdim=True)
                     if nk else s.new_zeros(nq, 1))
            mag = p @ vv.abs() * inv
            err = (U[dtype] + 2 * worst + 64 * E) * mag + (seen.double() @ vv.abs()) * (TINY[dtype] + 1e-9 * worst)
            out[q0:q1, h], bound[q0:q1, h] = o, err
    return out, bound


def check(got, ref, bound, dtype: str, what: str):
    """`got` against `ref`: within `bound` plus the rounding to its type, everywhere."""
    g = got.double()
    assert g.shape == ref.shape, f"{what}: shape {tuple(g.shape)} vs {tuple(ref.shape)}"
    assert torch.isfinite(g).all(), f"{what}: non-finite output"
    lim = bound + U[dtype] * (ref.abs() + bound) + TINY[dtype]
    d = (g - ref).abs()
    bad = d > lim
    if bad.any():
        at = int((d / lim).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bound; at flat index {at}: "
                             f"got {g.flatten()[at].item():.6g}, is {ref.flatten()[at].item():.6g}, "
                             f"allowed {lim.flatten()[at].item():.3g}")
