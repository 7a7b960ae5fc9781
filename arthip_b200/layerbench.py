"""Single conv layer benchmark (the 64->64 + bias + ReLU microbench on a 1080x1920 NHWC frame
by default), through the ``ah_conv3x3_*`` C ABI, or single token operator over the same frame
(``--op norm | rope | attention``, ``ah_norm_*`` / ``ah_rope_*`` / ``ah_attn_*``).

    python -m arthip_b200.layerbench [--C 64 --M 64 --H 1080 --W 1920 --act 1 --adds 0]
                                     [--warmup 3 --iters 20] [--algo direct|winograd]
    python -m arthip_b200.layerbench --op attention [--C 64 --H 1080 --W 1920 --head-dim 32 --window 8]

Of the token operators, ``norm`` is the RMS norms before and after a block with its layer scale
over H x W pixels of C channels; ``rope`` turns q and k of C / head-dim heads by row and column;
``attention`` is that many heads over windows of window x window pixels with a distance bias by
row and column (``--window 0``: the whole frame as one document).

Prints one JSON line: mean launch time from CUDA events around `iters` back-to-back
launches on the current stream, the algorithmic direct-conv FLOPs (2*9*C*M*H*W) and bytes
(input + residual inputs + weights read once, output written once) per launch, and their
rates against the measured B200 peaks (MEASURED_PEAKS.json beside the repository root when
present, else the pool's earlier figures). At the default size every tensor (265 MB) is
larger than the 126 MB L2, so consecutive launches do not hit in L2.
"""

from __future__ import annotations

import argparse
import json
from pathlib import Path

import numpy as np

_FALLBACK = {"hbm_gbs": 6650.0, "bf16_tflops": 1590.0}


def _peaks():
    p = Path(__file__).resolve().parent.parent / "MEASURED_PEAKS.json"
    if p.exists():
        try:
            d = json.loads(p.read_text())
            return {"hbm_gbs": float(d["hbm_gbs"]), "bf16_tflops": float(d["bf16_tflops"])}, "measured"
        except Exception:
            pass
    return dict(_FALLBACK), "fallback"


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--C", type=int, default=64)
    ap.add_argument("--M", type=int, default=64)
    ap.add_argument("--H", type=int, default=1080)
    ap.add_argument("--W", type=int, default=1920)
    ap.add_argument("--act", type=int, default=1, help="0 none, 1 ReLU, 2 SiLU")
    ap.add_argument("--adds", type=int, default=0, choices=[0, 1, 2])
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--iters", type=int, default=20)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--in-place", action="store_true",
                    help="write over the last residual operand (reduce-add stores); the "
                         "operand then accumulates across launches, which does not change the timing")
    ap.add_argument("--algo", default="direct", choices=["direct", "winograd", "pair"],
                    help="conv kernel: the direct implicit GEMM, Winograd F(2x2,3x3), or the direct conv on "
                         "two SMs per MMA (the last two 64 -> 64 only)")
    ap.add_argument("--model", choices=["C4F32", "R8F64", "R16F96"],
                    help="time whole frames of this BASELINE chain (luma, 2x) at --H x --W through the "
                         "engine's CUDA graph instead of one layer (a small-frame case for profilers)")
    ap.add_argument("--op", choices=["conv", "norm", "rope", "attention"], default="conv",
                    help="the conv layer, or a token operator over the frame")
    ap.add_argument("--head-dim", type=int, default=32, help="elements per attention head (--op rope, attention)")
    ap.add_argument("--window", type=int, default=8, help="side of the attention windows; 0: the whole frame")
    args = ap.parse_args(argv)
    if args.model:
        return _model_frames(args)
    if args.op != "conv":
        return _token_operator(args, ap)

    import torch

    from arthip_b200.engine import Conv3x3

    dev = torch.device("cuda:0")
    C, M, H, W = args.C, args.M, args.H, args.W
    g = torch.Generator(device="cpu").manual_seed(args.seed)
    x = torch.rand(1, H, W, C, generator=g).half().to(dev)
    adds = [torch.rand(1, H, W, M, generator=g).half().to(dev) for _ in range(args.adds)]
    out = torch.empty(1, H, W, M, dtype=torch.float16, device=dev)
    rng = np.random.default_rng(args.seed)
    w = (rng.standard_normal((M, C, 3, 3)) * (2.0 / (9 * C)) ** 0.5).astype(np.float16)
    b = (rng.standard_normal(M) * 0.01).astype(np.float16).astype(np.float32)
    conv = Conv3x3(w, b, act=args.act, algo=args.algo)
    s = torch.cuda.current_stream().cuda_stream
    ptrs = [a.data_ptr() for a in adds]
    if args.in_place:
        if not adds:
            ap.error("--in-place needs --adds 1 or 2")
        out = adds[-1]

    def launch():
        conv.run(x.data_ptr(), H, W, out.data_ptr(), *ptrs, stream=s)

    for _ in range(max(1, args.warmup)):
        launch()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(args.iters):
        launch()
    e1.record()
    torch.cuda.synchronize()
    status = conv.status()
    ms = e0.elapsed_time(e1) / args.iters
    flops = 2.0 * 9 * C * M * H * W
    nbytes = 2.0 * H * W * (C + M * (1 + args.adds)) + 2.0 * 9 * C * M + 4.0 * M
    peaks, src = _peaks()
    tflops = flops / (ms * 1e-3) / 1e12
    gbs = nbytes / (ms * 1e-3) / 1e9
    roof_ms = max(flops / (peaks["bf16_tflops"] * 1e12), nbytes / (peaks["hbm_gbs"] * 1e9)) * 1e3
    print(json.dumps({
        "layer": f"conv3x3 {C}->{M} act{args.act} adds{args.adds}{' in place' if args.in_place else ''} {H}x{W}", "kernel": conv.kind,
        "us_per_launch": ms * 1e3, "tflops": tflops, "gbs": gbs, "algorithmic_flops": flops,
        "algorithmic_bytes": nbytes, "roofline_us": roof_ms * 1e3, "roofline_frac": roof_ms / ms,
        "tflops_frac": tflops / peaks["bf16_tflops"], "peaks": src, "iters": args.iters, "status": status,
    }))
    conv.close()
    return 0 if status == 0 else 1


def _token_operator(args, ap) -> int:
    import torch

    from arthip_b200.token_ops import AxisRotary, TokenAttention, TokenNorm

    C, H, W, d = args.C, args.H, args.W, args.head_dim
    n = H * W
    g = torch.Generator(device="cuda").manual_seed(args.seed)

    def tensor(channels):
        return torch.randn(n, channels, generator=g, device="cuda", dtype=torch.float16)

    s = torch.cuda.current_stream().cuda_stream
    status = 0
    if args.op == "norm":
        x, y, out, norm = tensor(C), tensor(C), tensor(C), tensor(C)
        w = np.ones(C, dtype=np.float32)
        op = TokenNorm(C, post_norm="rms", pre_norm="rms", post_weight=w, pre_weight=w, layer_scale=0.5 * w)
        label, flops, nbytes = f"norm {C} {H}x{W}", 12.0 * n * C, 8.0 * n * C + 12.0 * C

        def launch():
            op.run(n, x.data_ptr(), out.data_ptr(), norm.data_ptr(), y.data_ptr(), stream=s)
    else:
        if C % d or d % 16:
            ap.error("--C must be a multiple of --head-dim, and that of 16")
        heads = C // d
        yy, xx = torch.meshgrid(torch.arange(H, device="cuda"), torch.arange(W, device="cuda"), indexing="ij")
        if args.op == "rope":
            q, k, q_out, k_out = tensor(C), tensor(C), tensor(C), tensor(C)
            pos = torch.stack([yy.flatten(), xx.flatten()]).float().contiguous()
            op = AxisRotary(d, [d // 2, d // 2])
            label, flops, nbytes = f"rope {heads}x{d} {H}x{W}", 6.0 * n * C, 8.0 * n * C + 8.0 * n

            def launch():
                op.run(n, pos.data_ptr(), q.data_ptr(), heads, q_out.data_ptr(), k.data_ptr(), heads,
                       k_out.data_ptr(), stream=s)
        else:
            b = args.window
            if b < 0 or (b and (H % b or W % b)):
                ap.error("--window must divide --H and --W")

            def windows(t):  # tokens of one window after those of another
                return t.flatten() if b == 0 else t.view(H // b, b, W // b, b).permute(0, 2, 1, 3).reshape(-1)

            pos = torch.stack([windows(yy), windows(xx)]).float().contiguous()
            q, k, v, out = tensor(C), tensor(C), tensor(C), tensor(C)
            each = b * b if b else n
            off = np.arange(0, n + 1, each)
            op = TokenAttention(off, off, heads, heads, d, slopes=np.full((heads, 2), 0.05, dtype=np.float32))
            label = f"attention {heads}x{d} {'whole' if b == 0 else f'{b}x{b} windows'} {H}x{W}"
            flops, nbytes = 4.0 * n * each * C, 8.0 * n * C + 16.0 * n

            def launch():
                op.run(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), pos.data_ptr(), pos.data_ptr(),
                       stream=s)

    for _ in range(max(1, args.warmup)):
        launch()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(args.iters):
        launch()
    e1.record()
    torch.cuda.synchronize()
    if args.op == "attention":
        status = op.status()
    ms = e0.elapsed_time(e1) / args.iters
    peaks, src = _peaks()
    roof_ms = max(flops / (peaks["bf16_tflops"] * 1e12), nbytes / (peaks["hbm_gbs"] * 1e9)) * 1e3
    print(json.dumps({
        "layer": label, "us_per_launch": ms * 1e3, "tflops": flops / (ms * 1e-3) / 1e12,
        "gbs": nbytes / (ms * 1e-3) / 1e9, "algorithmic_flops": flops, "algorithmic_bytes": nbytes,
        "roofline_us": roof_ms * 1e3, "roofline_frac": roof_ms / ms, "peaks": src, "iters": args.iters,
        "status": status,
    }))
    op.close()
    return 0 if status == 0 else 1


def _model_frames(args) -> int:
    import tempfile
    import time

    import torch

    from arthip_b200 import modelgen, onnx_proto as op
    from arthip_b200.engine import Engine

    H, W = args.H, args.W
    with tempfile.TemporaryDirectory() as td:
        cm = modelgen.conv_chain(modelgen.CONFIGS[args.model], seed=args.seed)
        path = Path(td) / f"{args.model}.onnx"
        op.save_model(cm.model, path)
        eng = Engine(path)
        eng.set_conv_algo(args.algo)
        in_ptr, _, in_bytes, _ = eng.prepare(1, H, W)
        dev = torch.device("cuda:0")
        frame = torch.from_numpy(modelgen.synthetic_frame(args.seed, 1, H, W).reshape(-1)).to(dev)
        torch.cuda.synchronize()

        class _B:  # the engine's input buffer as a torch view
            __cuda_array_interface__ = {"shape": (in_bytes // 2,), "typestr": "<f2", "data": (in_ptr, False),
                                        "version": 3}
        torch.as_tensor(_B(), device=dev).copy_(frame)
        torch.cuda.synchronize()
        for _ in range(max(1, args.warmup)):
            eng.enqueue()
        eng.synchronize()
        t0 = time.perf_counter()
        for _ in range(args.iters):
            eng.enqueue()
        eng.synchronize()
        ms = (time.perf_counter() - t0) * 1e3 / args.iters
        print(json.dumps({"model": f"{args.model} {H}x{W}", "algo": args.algo, "ms_per_frame": ms, "fps": 1e3 / ms,
                          "iters": args.iters, "timing": "host wall clock around enqueued graph replays"}))
        eng.close()
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
