"""Timed cases of the token operators: the norms around a block with its gate and residual
scale (``TokenNorm``), rotary positions over time, height and width (``AxisRotary``) and
attention with a score cap, distance biases, documents and prefixes (``TokenAttention``).

Tokens are the pixels or patches of a frame in row-major order, several frames or windows
packed one after another as documents; activations are ``[tokens][channels]``, which is the
NHWC layout of the conv layers. ``run`` computes a case with elementary torch operations in
32 bits, or, where ``own`` is true, with the library's kernels. ``exact`` is the definition
in 64 bits.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One 16x16 tile between two conv layers: launch latency is what counts.
        norm_case("norm tile", 256, 64, "fp16", post="none", pre="rms"),
        # Every pixel of a 1080p frame at the width of the 64-channel chains: memory bound.
        norm_case("norm 1080p", 1080 * 1920, 64, "fp16", post="rms", pre="rms"),
        # A batch of four 90x90-patch images whose gate, scale and shift come per image.
        norm_case("norm modulated", 4 * 8100, 1280, "bf16", post="none", pre="layer", gate="group", mod=True, groups=4),
        # A width that no vector load divides, gated per pixel by a side branch.
        norm_case("norm odd width", 270 * 480, 90, "fp16", post="layer", pre="layer", gate="sigmoid"),
        # One new token of a streaming clip.
        rope_case("rope one token", 1, 8, 2, 64, "16,24,24", "halves", "bf16"),
        # Nine frames of 45x80 patches, adjacent pairs, sections that are no multiple of 8.
        rope_case("rope clip", 9 * 45 * 80, 24, 24, 128, "44,42,42", "pairs", "bf16"),
        # The q and k slices of a fused projection of a 270x480 frame, height and width only.
        rope_case("rope frame slices", 270 * 480, 4, 4, 32, "16,16", "halves", "fp16", strided=True),
        # The smallest attention: a 4x4 patch.
        attn_case("attention patch", "1*16", "1*16", 2, 2, 32, "fp16"),
        # The 8x8 windows of a 272x480 frame with a height and width distance bias.
        attn_case("attention windows", "2040*64", "2040*64", 6, 6, 32, "fp16", axes=2),
        # Every pixel of a 135x240 frame against every other.
        attn_case("attention frame", "1*32400", "1*32400", 8, 8, 64, "fp16"),
        # Clips of unlike lengths: causal after a conditioning prefix, capped scores, biases
        # over three axes, four query heads to a key head.
        attn_case("attention clips", "3001,1,777,4099,256,1538", "3001,1,777,4099,256,1538", 16, 4, 128, "bf16",
                  mask="causal", prefix="257,0,64,1000,256,31", cap=30.0, axes=3),
        # One new token in each of eight streams against long caches of unlike fill.
        attn_case("attention one token", "8*1", "8*65536", 32, 8, 128, "bf16", mask="causal", lens=True),
    ]


def norm_case(name, rows, channels, dtype, post, pre, gate="none", mod=False, groups=1):
    """gate: none, group (one row per image), or the activation of a per-token gate."""
    return {"name": name, "op": "norm", "rows": rows, "channels": channels, "dtype": dtype, "post": post, "pre": pre,
            "gate": gate, "mod": mod, "groups": groups}


def rope_case(name, tokens, q_heads, k_heads, head_dim, axes, layout, dtype, strided=False):
    return {"name": name, "op": "rope", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "head_dim": head_dim,
            "axes": axes, "layout": layout, "dtype": dtype, "strided": strided}


def attn_case(name, q, k, q_heads, kv_heads, head_dim, dtype, mask="full", prefix="", cap=0.0, axes=0, lens=False):
    """q, k: the documents' lengths ("2040*64" is 2040 documents of 64); lens: the keys in use
    are a device array below the given capacities."""
    return {"name": name, "op": "attention", "q": q, "k": k, "q_heads": q_heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "mask": mask, "prefix": prefix, "cap": cap, "axes": axes,
            "lens": lens}


def log_int(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "norm", "rope", "attention", "attention"))
    dtype = rng.choice(("fp16", "bf16"))
    if kind == "norm":
        channels = log_int(rng, 8, 4096)
        rows = log_int(rng, 1, 1080 * 1920 * 64 // channels)
        gate = rng.choice(("none", "group", "sigmoid", "tanh", "silu"))
        groups = rng.choice((1, 2, 3, 5)) if rows % 30 == 0 else 1
        c = norm_case("", rows, channels, dtype, rng.choice(("none", "rms", "layer")), rng.choice(("rms", "layer")),
                      gate, rng.random() < 0.5, groups)
    elif kind == "rope":
        layout = rng.choice(("halves", "pairs", "shared"))
        dims = [2 * rng.randint(2, 21) for _ in range(rng.randint(1, 3))]
        head_dim = sum(dims) + 2 * rng.choice((0, 0, 1, 8))
        q_heads = rng.randint(1, 32)
        k_heads = rng.choice((q_heads, max(1, q_heads // 4)))
        tokens = log_int(rng, 1, 9 * 45 * 80 * 24 * 128 // (max(q_heads, 4) * max(head_dim, 32)))
        c = rope_case("", tokens, q_heads, k_heads, head_dim, ",".join(map(str, dims)), layout, dtype,
                      rng.random() < 0.3)
    else:
        head_dim = 8 * rng.randint(2, 16)
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        q_heads = kv_heads * rng.choice((1, 1, 2, 4))
        mask = rng.choice(("full", "causal", "causal"))
        few = rng.random() < 0.35  # a few new tokens against caches
        docs = log_int(rng, 1, 16 if few else 40)
        longest = log_int(rng, 4, 30000 if few else 12000 // docs + 4)
        k = [log_int(rng, 1, longest) for _ in range(docs)]
        q = [rng.randint(1, min(8, n)) for n in k] if few else k
        prefix = [rng.randint(0, n) for n in k] if mask == "causal" and rng.random() < 0.5 else []
        c = attn_case("", ",".join(map(str, q)), ",".join(map(str, k)), q_heads, kv_heads, head_dim, dtype, mask,
                      ",".join(map(str, prefix)), rng.choice((0.0, 0.0, 20.0, 50.0)), rng.choice((0, 0, 1, 2, 3)),
                      few and rng.random() < 0.5)
    del c["name"]
    return c


def lengths(text):
    got = []
    for part in filter(None, text.split(",")):
        n, _, v = part.rpartition("*")
        got += [int(v)] * (int(n) if n else 1)
    return got


def pairs_seen(case, ks):
    """How many (query, key) pairs the mask leaves, with ks keys in use in each document."""
    qs = lengths(case["q"])
    if case["mask"] == "full":
        return sum(a * b for a, b in zip(qs, ks))
    pre = lengths(case["prefix"]) or [0] * len(qs)
    total = 0
    for nq, nk, p in zip(qs, ks, pre):
        hi = np.arange(nq, dtype=np.int64) + (nk - nq + 1)
        total += int(np.clip(np.maximum(hi, min(p, nk)), 0, nk).sum())
    return total


def work(case):
    size = 2
    if case["op"] == "norm":
        n = case["rows"] * case["channels"]
        per_token = case["gate"] not in ("none", "group")
        small = case["channels"] * size * case["groups"] * ((case["gate"] == "group") + 2 * case["mod"])
        return {"bytes": n * size * (4 + per_token) + small + 5 * 4 * case["channels"], "flops": 12 * n}
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * size + case["tokens"] * 4 * len(lengths(case["axes"])), "flops": 3 * n}
    ks = lengths(case["k"])
    tq, d = sum(lengths(case["q"])), case["head_dim"]
    if case["lens"]:  # prepare() fills the caches between a half and the whole
        ks = [(3 * n) // 4 for n in ks]
    nbytes = size * d * (2 * tq * case["q_heads"] + 2 * sum(ks) * case["kv_heads"]) + 4 * case["axes"] * (tq + sum(ks))
    return {"bytes": nbytes, "flops": 4 * pairs_seen(case, ks) * d * case["q_heads"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
class Maker:
    """Seeded tensors made on the GPU."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype, std=1.0, mean=0.0):
        return torch.randn(shape, generator=self.g, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)

    def large_normal(self, shape, dtype, std=1.0):
        """As normal(), drawn in the type itself: half the memory."""
        return torch.randn(shape, generator=self.g, device="cuda", dtype=dtype).mul_(std)

    def whole(self, lo, hi, shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)


def grid_positions(counts):
    """fp32 [3][tokens] (time, height, width) of each document as frames of about square
    shape, row-major."""
    t, y, x = [], [], []
    for n in counts:
        w = max(1, int(math.sqrt(n)))
        h = min(w, 64)
        i = np.arange(n)
        t.append(i // (w * h))
        y.append(i // w % h)
        x.append(i % w)
    return np.stack([np.concatenate(v) for v in (t, y, x)]).astype(np.float32)


def prepare(case, seed):
    make = Maker(seed)
    s = {"case": dict(case)}
    return {"norm": prepare_norm, "rope": prepare_rope, "attention": prepare_attention}[case["op"]](case, make, s)


def prepare_norm(case, make, s):
    rows, c, dt = case["rows"], case["channels"], DTYPES[case["dtype"]]
    s["x"] = make.large_normal((rows, c), dt, 2.0)
    s["y"] = make.large_normal((rows, c), dt).add_(0.25)
    for name in ("post_weight", "pre_weight"):
        s[name] = make.normal((c,), torch.float32, 0.2, 1.0)
    for name, kind in (("post_bias", case["post"]), ("pre_bias", case["pre"])):
        s[name] = make.normal((c,), torch.float32, 0.1) if kind == "layer" else None
    s["layer_scale"] = make.normal((c,), torch.float32, 0.1, 0.5)
    s["residual_scale"] = 0.75
    per_group = (case["groups"], c)
    s["gate"] = None
    if case["gate"] == "group":
        s["gate"] = make.normal(per_group, dt, 0.5)
    elif case["gate"] != "none":
        s["gate"] = make.large_normal((rows, c), dt)
    s["mod_scale"] = make.normal(per_group, dt, 0.2) if case["mod"] else None
    s["mod_shift"] = make.normal(per_group, dt, 0.2) if case["mod"] else None
    s["out"], s["norm"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    if own:
        from arthip_b200.token_ops import TokenNorm
        host = {k: None if s[k] is None else s[k].cpu().numpy()
                for k in ("post_weight", "post_bias", "pre_weight", "pre_bias", "layer_scale")}
        if case["post"] == "none":
            host["post_weight"] = None
        s["op"] = TokenNorm(c, dtype=case["dtype"], post_norm=case["post"], pre_norm=case["pre"],
                            gate_act=case["gate"] if case["gate"] in ("sigmoid", "tanh", "silu") else "none",
                            residual_scale=s["residual_scale"], post_eps=EPS, pre_eps=EPS, **host)
    return s


def prepare_rope(case, make, s):
    n, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["head_dim"]
    dt, dims = DTYPES[case["dtype"]], lengths(case["axes"])
    extra = d * 3 if case["strided"] else 0  # q, k and something else side by side in a token's row
    s["qk"] = make.large_normal((n, (hq + hk) * d + extra), dt)
    first = int(make.whole(0, 5000, (1,)).item())  # the clip is a part of a longer stream
    pos = grid_positions([n])[3 - len(dims):]
    pos[0] += first
    s["pos"] = torch.from_numpy(np.ascontiguousarray(pos)).cuda()
    s["theta"] = 10000.0
    s["q_out"] = torch.empty((n, hq, d), dtype=dt, device="cuda")
    s["k_out"] = torch.empty((n, hk, d), dtype=dt, device="cuda")
    if own:
        from arthip_b200.token_ops import AxisRotary
        s["op"] = AxisRotary(d, dims, theta=s["theta"], layout=case["layout"], dtype=case["dtype"])
    return s


def prepare_attention(case, make, s):
    qs, ks = lengths(case["q"]), lengths(case["k"])
    hq, hk, d, dt = case["q_heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    # Scores of a standard deviation of 1.5, and of several times that where a cap bounds them.
    s["q"] = make.large_normal((sum(qs), hq, d), dt, 8.0 if case["cap"] else 1.5)
    s["k"] = make.large_normal((sum(ks), hk, d), dt)
    s["v"] = make.large_normal((sum(ks), hk, d), dt)
    s["q_offsets"], s["k_offsets"] = np.cumsum([0] + qs), np.cumsum([0] + ks)
    s["prefix"] = lengths(case["prefix"]) or None
    s["q_pos"] = s["k_pos"] = s["slopes"] = s["k_lens"] = None
    lens = ks
    if case["lens"]:
        share = np.random.RandomState(make.whole(0, 1 << 30, (1,)).item()).uniform(0.5, 1.0, len(ks))
        lens = [max(b, int(round(n * f))) for b, n, f in zip(qs, ks, share)]
        s["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if case["axes"]:
        kp = grid_positions(ks)[3 - case["axes"]:]
        at = np.concatenate([o + np.arange(b) + (n - b) for o, b, n in zip(s["k_offsets"], qs, lens)])
        s["k_pos"] = torch.from_numpy(np.ascontiguousarray(kp)).cuda()
        s["q_pos"] = torch.from_numpy(np.ascontiguousarray(kp[:, at])).cuda()
        s["slopes"] = (2.0 ** -(1.0 + 7.0 * np.arange(hq * case["axes"]) / (hq * case["axes"]))).reshape(hq, -1)
        s["slopes"] = s["slopes"].astype(np.float32)
        s["slopes_gpu"] = torch.from_numpy(s["slopes"]).cuda()
    s["scale"] = 1.0 / math.sqrt(d)
    s["out"] = torch.empty_like(s["q"])
    s["spans"] = [torch.tensor(v, dtype=torch.int64, device="cuda") for v in (s["q_offsets"], s["k_offsets"])]
    s["prefix_gpu"] = torch.tensor(s["prefix"] or [0] * len(qs), dtype=torch.int64, device="cuda")
    if own:
        from arthip_b200.token_ops import TokenAttention
        s["op"] = TokenAttention(s["q_offsets"], s["k_offsets"], hq, hk, d, scale=s["scale"], cap=case["cap"],
                                 mask=case["mask"], prefix=s["prefix"], slopes=s["slopes"], dtype=case["dtype"])
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(s):
    kind = s["case"]["op"]
    if own:
        return {"norm": own_norm, "rope": own_rope, "attention": own_attention}[kind](s)
    return {"norm": plain_norm, "rope": plain_rope, "attention": plain_attention}[kind](s)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def own_norm(s):
    rows = s["case"]["rows"]
    per = rows // s["case"]["groups"]
    s["op"].run(rows, s["x"].data_ptr(), s["out"].data_ptr(), s["norm"].data_ptr(), y_ptr=s["y"].data_ptr(),
                gate_ptr=ptr(s["gate"]), rows_per_gate=per if s["case"]["gate"] == "group" else 1,
                mod_scale_ptr=ptr(s["mod_scale"]), mod_shift_ptr=ptr(s["mod_shift"]), rows_per_mod=per,
                stream=torch.cuda.current_stream().cuda_stream)
    return s["out"], s["norm"]


def own_rope(s):
    c = s["case"]
    hq, d, row = c["q_heads"], c["head_dim"], s["qk"].shape[1]
    s["op"].run(c["tokens"], s["pos"].data_ptr(), s["qk"].data_ptr(), hq, s["q_out"].data_ptr(),
                k_ptr=s["qk"].data_ptr() + hq * d * 2, k_heads=c["k_heads"], k_out_ptr=s["k_out"].data_ptr(),
                q_strides=(row, d), k_strides=(row, d), stream=torch.cuda.current_stream().cuda_stream)
    return s["q_out"], s["k_out"]


def own_attention(s):
    s["op"].run(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), q_pos_ptr=ptr(s["q_pos"]),
                k_pos_ptr=ptr(s["k_pos"]), k_lens_ptr=ptr(s["k_lens"]),
                stream=torch.cuda.current_stream().cuda_stream)
    return s["out"]


def normed(v, kind, weight, bias):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * weight
    return v if bias is None else v + bias


def plain_norm(s):
    c = s["case"]
    rows = c["rows"]
    b = s["y"].float()
    if c["post"] != "none":
        b = normed(b, c["post"], s["post_weight"], s["post_bias"])
    b = b * (s["layer_scale"] * s["residual_scale"])
    if s["gate"] is not None:
        g = s["gate"].float()
        if c["gate"] == "tanh":
            g = 1 - 2 / (torch.exp(2 * g) + 1)
        elif c["gate"] in ("sigmoid", "silu"):
            g = (g if c["gate"] == "silu" else 1) / (1 + torch.exp(-g))
        b = (b.view(g.shape[0], -1, c["channels"]) * g[:, None]).view(rows, -1)
    out = s["x"].float() + b
    n = normed(out, c["pre"], s["pre_weight"], s["pre_bias"])
    if c["mod"]:
        n = n.view(c["groups"], -1, c["channels"])
        n = (n * (1 + s["mod_scale"].float()[:, None]) + s["mod_shift"].float()[:, None]).view(rows, -1)
    return out.to(s["x"].dtype), n.to(s["x"].dtype)


def rotary_pairs(layout, dims, theta):
    """Of each rotated pair: its two elements, its axis and its frequency."""
    a = np.repeat(np.arange(len(dims)), [n // 2 for n in dims])
    j = np.concatenate([np.arange(n // 2) for n in dims])
    n = np.asarray(dims)[a]
    p = np.arange(len(a))
    if layout == "pairs":
        return 2 * p, 2 * p + 1, a, theta ** (-2.0 * j / n)
    if layout == "halves":
        base = (np.cumsum(dims) - dims)[a]
        return base + j, base + j + n // 2, a, theta ** (-2.0 * j / n)
    return p, p + len(a), a, theta ** (-1.0 * p / len(a))


def plain_rope(s):
    c = s["case"]
    i0, i1, axis, freq = rotary_pairs(c["layout"], lengths(c["axes"]), s["theta"])
    i0, i1, axis = (torch.from_numpy(v).cuda() for v in (i0, i1, axis))
    angle = s["pos"].double()[axis].T * torch.from_numpy(freq).cuda()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = s["qk"][:, :(c["q_heads"] + c["k_heads"]) * c["head_dim"]].float()
    x = x.view(c["tokens"], -1, c["head_dim"])
    a, b = x[..., i0], x[..., i1]
    out = x.clone()
    out[..., i0] = a * cos - b * sin
    out[..., i1] = a * sin + b * cos
    out = out.to(s["qk"].dtype)
    return out[:, :c["q_heads"]].contiguous(), out[:, c["q_heads"]:].contiguous()


def plain_attention(s):
    """The documents padded to one length, one key head at a time."""
    c = s["case"]
    qo, ko = s["spans"]
    nq, nk = qo[1:] - qo[:-1], ko[1:] - ko[:-1]
    group = c["q_heads"] // c["kv_heads"]
    iq = torch.arange(max(lengths(c["q"])), device="cuda")
    ik = torch.arange(max(lengths(c["k"])), device="cuda")
    at_q = (qo[:-1, None] + iq).clamp(max=s["q"].shape[0] - 1)
    at_k = (ko[:-1, None] + ik).clamp(max=s["k"].shape[0] - 1)
    used = nk if s["k_lens"] is None else s["k_lens"].long()
    seen = (ik < used[:, None])[:, None]
    if c["mask"] == "causal":
        last = iq + (used - nq)[:, None]
        seen = seen & ((ik <= last[..., None]) | (ik < s["prefix_gpu"][:, None])[:, None])
    out = torch.zeros_like(s["q"])
    mine = iq < nq[:, None]
    for h in range(c["kv_heads"]):
        k, v = s["k"][:, h][at_k].float(), s["v"][:, h][at_k].float()
        for j in range(h * group, (h + 1) * group):
            x = (s["q"][:, j][at_q].float() * s["scale"]) @ k.transpose(1, 2)
            if c["cap"]:
                x = c["cap"] * torch.tanh(x / c["cap"])
            for a in range(c["axes"]):
                far = (s["q_pos"][a][at_q][:, :, None] - s["k_pos"][a][at_k][:, None]).abs_()
                x = x - s["slopes_gpu"][j, a] * far
            x = x.masked_fill_(~seen, -math.inf)
            top = x.amax(2, keepdim=True).clamp_(min=-1e30)
            x = torch.exp(x - top)
            o = (x @ v) / x.sum(2, keepdim=True).clamp_(min=1e-30)
            out[:, j][at_q[mine]] = o[mine].to(out.dtype)
    return out


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": exact_norm, "rope": exact_rope, "attention": exact_attention}[case["op"]](case, s)


def exact_norm(case, s):
    group = torch.arange(case["rows"], device="cuda") // (case["rows"] // case["groups"])
    outs, norms = [], []

    def statistics(v, kind, w, b):
        w, b = w.double(), 0.0 if b is None else b.double()
        mean = v.mean(dim=-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
        var = ((v - mean) ** 2).sum(dim=-1, keepdim=True) / case["channels"]
        return (v - mean) / torch.sqrt(var + EPS) * w + b

    step = max(1, (1 << 26) // case["channels"])
    for r in range(0, case["rows"], step):
        part = slice(r, min(r + step, case["rows"]))
        b = s["y"][part].double()
        if case["post"] != "none":
            b = statistics(b, case["post"], s["post_weight"], s["post_bias"])
        gate = 1.0
        if case["gate"] == "group":
            gate = s["gate"].double()[group[part]]
        elif case["gate"] != "none":
            g = s["gate"][part].double()
            gate = {"sigmoid": torch.sigmoid(g), "tanh": torch.tanh(g), "silu": g * torch.sigmoid(g)}[case["gate"]]
        out = s["x"][part].double() + s["residual_scale"] * s["layer_scale"].double() * gate * b
        n = statistics(out, case["pre"], s["pre_weight"], s["pre_bias"])
        if case["mod"]:
            n = n * (1.0 + s["mod_scale"].double()[group[part]]) + s["mod_shift"].double()[group[part]]
        outs.append(out)
        norms.append(n)
    return torch.cat(outs), torch.cat(norms)


def exact_rope(case, s):
    """Each rotated pair as a complex number times exp(i angle)."""
    dims, d, n = lengths(case["axes"]), case["head_dim"], case["tokens"]
    heads = case["q_heads"] + case["k_heads"]
    x = s["qk"][:, :heads * d].reshape(n, heads, d).double()
    out = x.clone()
    total, base = sum(dims), 0
    for a, size in enumerate(dims):
        for j in range(size // 2):
            if case["layout"] == "pairs":
                e0, e1, f = base + 2 * j, base + 2 * j + 1, s["theta"] ** (-2 * j / size)
            elif case["layout"] == "halves":
                e0, e1, f = base + j, base + size // 2 + j, s["theta"] ** (-2 * j / size)
            else:
                p = base // 2 + j
                e0, e1, f = p, total // 2 + p, s["theta"] ** (-2 * p / total)
            turn = torch.polar(torch.ones(n, dtype=torch.float64, device="cuda"), s["pos"][a].double() * f)
            z = torch.complex(x[:, :, e0], x[:, :, e1]) * turn[:, None]
            out[:, :, e0], out[:, :, e1] = z.real, z.imag
        base += size
    return out[:, :case["q_heads"]].contiguous(), out[:, case["q_heads"]:].contiguous()


def exact_attention(case, s):
    """Document by document, some rows of all heads at a time."""
    hq, group = case["q_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens = np.diff(s["k_offsets"]) if s["k_lens"] is None else s["k_lens"].cpu().numpy()
    for n in range(len(lens)):
        q0, q1, k0, nk = int(s["q_offsets"][n]), int(s["q_offsets"][n + 1]), int(s["k_offsets"][n]), int(lens[n])
        j = torch.arange(nk, device="cuda")
        k = s["k"][k0:k0 + nk].double().permute(1, 2, 0).repeat_interleave(group, 0)
        v = s["v"][k0:k0 + nk].double().transpose(0, 1).repeat_interleave(group, 0)
        step = max(1, int(5e8 / (hq * max(nk, 1))))
        for r in range(q0, q1, step):
            e = min(r + step, q1)
            i = torch.arange(r - q0, e - q0, device="cuda")[:, None]
            x = torch.bmm(s["q"][r:e].double().transpose(0, 1), k) * s["scale"]
            if case["cap"]:
                x = torch.tanh(x / case["cap"]) * case["cap"]
            for a in range(case["axes"]):
                dist = (s["q_pos"][a, r:e].double()[:, None] - s["k_pos"][a, k0:k0 + nk].double()[None]).abs()
                x -= s["slopes_gpu"].double()[:, a][:, None, None] * dist
            if case["mask"] == "causal":
                hidden = j > i + (nk - (q1 - q0))
                if s["prefix"]:
                    hidden &= j >= s["prefix"][n]
                x = x.masked_fill_(hidden, -math.inf)
            if nk:
                w = torch.softmax(x, dim=-1).nan_to_num_(0.0)
                out[r:e] = torch.bmm(w, v).transpose(0, 1)
    return out
