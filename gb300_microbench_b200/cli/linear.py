"""Sweep of the quantised linear layer: the quantiser of its activations and
its product, per format and number of tokens, on one GPU.

    python -m gb300_microbench_b200.cli.linear [--formats F,F] [--tokens M,M] [--n N] [--k K]
                                               [--iterations N] [--warmup-iterations N] [--output FILE]

Formats: fp8 (RMS norm with the residual's addition to FP8, FP8 product),
nvfp4 and mxfp4 (4-bit quantisation and product). Weights are N(0, 0.02),
tokens N(0, 1) BF16, both from torch.Generator seed 0. Each step is timed with
CUDA events after a 256 MiB write outside them (L2 flushed), and the layer
as a whole back to back (hot). D is checked against the FP64 product of the
decoded operands on up to 64 rows (relative Frobenius <= 5e-3: BF16 rounding
is 1.7e-3). One CSV row per (format, tokens).
"""
from __future__ import annotations

import argparse
import csv
import statistics
import sys

from . import common as cm

FORMATS = ("fp8", "nvfp4", "mxfp4")
TOKENS = (1, 16, 64, 256, 1024, 8192)
TOL = 5e-3
FIELDS = ("format", "m", "n", "k", "quantizer_us", "product_us", "layer_us_hot", "product_tflops", "product_weight_gbs",
          "few_rows", "tile_m", "tile_n", "grid_ctas", "rel_frobenius_sampled", "correctness", "gpu_name", "git_commit")


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="linear")
    ap.add_argument("--formats", default=",".join(FORMATS))
    ap.add_argument("--tokens", default=",".join(map(str, TOKENS)))
    ap.add_argument("--n", type=int, default=8192)
    ap.add_argument("--k", type=int, default=8192)
    ap.add_argument("--iterations", type=int, default=20)
    ap.add_argument("--warmup-iterations", type=int, default=5)
    ap.add_argument("--output", default="-")
    try:
        args = ap.parse_args(sys.argv[1:] if argv is None else argv)
    except SystemExit as exc:
        return int(exc.code or 0)
    formats = args.formats.split(",")
    try:
        tokens = [int(t) for t in args.tokens.split(",")]
    except ValueError:
        tokens = [0]
    if set(formats) - set(FORMATS) or min(tokens) < 1 or args.n < 1 or args.k < 32 or args.k % 32:
        cm.eprint(f"linear: --formats from {','.join(FORMATS)}, --tokens and --n positive, --k a multiple of 32")
        return 2
    if args.iterations < 1 or args.warmup_iterations < 0:
        cm.eprint("linear: --iterations must be >= 1 and --warmup-iterations >= 0")
        return 2

    import torch

    from .. import lowp, quantize

    dev = torch.device("cuda", 0)
    stream = torch.cuda.Stream(device=dev)
    flush = torch.empty(64 << 20, dtype=torch.float32, device=dev)
    gpu, commit = cm.query_gpu(), cm.git_commit_hash()
    n, k = args.n, args.k

    def flushed_us(plan) -> float:
        pairs = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
                 for _ in range(args.iterations)]
        for e0, e1 in pairs:
            with torch.cuda.stream(stream):
                flush.zero_()
            e0.record(stream)
            plan.run()
            e1.record(stream)
        stream.synchronize()
        return statistics.median(e0.elapsed_time(e1) for e0, e1 in pairs) * 1e3

    rows, failed = [], False
    gen = torch.Generator().manual_seed(0)
    weights = (torch.randn(n, k, generator=gen) * 0.02).to(dev)
    for fmt in formats:
        w = {"fp8": lowp.Fp8BlockOperand, "nvfp4": lowp.Nvfp4Operand, "mxfp4": lowp.Mxfp4Operand}[fmt](weights)
        for m in tokens:
            x = torch.randn(m, k, generator=gen).to(torch.bfloat16).to(dev)
            if fmt == "fp8":
                a = lowp.Fp8GroupOperand.empty(m, k, device=dev)
                quant = quantize.RmsNormFp8Plan(x, torch.ones(k, dtype=torch.bfloat16, device=dev), a,
                                                residual=torch.zeros_like(x), residual_out=torch.empty_like(x),
                                                stream=stream)
            else:
                a = (lowp.Nvfp4Operand if fmt == "nvfp4" else lowp.Mxfp4Operand).empty(m, k, device=dev)
                quant = quantize.Fp4QuantPlan(x, a, stream=stream)
            d = torch.empty(m, n, dtype=torch.bfloat16, device=dev)
            product = lowp.LowpLinearPlan(a, w, d, stream=stream)
            stream.wait_stream(torch.cuda.current_stream(dev))
            for _ in range(1 + args.warmup_iterations):
                quant.run()
                product.run()
            product.synchronize()
            quant_us, product_us = flushed_us(quant), flushed_us(product)
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record(stream)
            for _ in range(args.iterations):
                quant.run()
                product.run()
            e1.record(stream)
            product.synchronize()
            layer_us = e0.elapsed_time(e1) / args.iterations * 1e3
            pick = torch.arange(0, m, max(1, -(-m // 64)), device=dev)
            ref = a.dequantize()[pick].double() @ w.dequantize().double().T
            err = ((d[pick].double() - ref).norm() / ref.norm()).item()
            ok = err <= TOL
            failed |= not ok
            weight_bytes = w.data.numel() + (w.scales.numel() * 4 if fmt == "fp8" else w.atoms.numel())
            info = product.info
            rows.append({
                "format": fmt, "m": m, "n": n, "k": k, "quantizer_us": cm.fixed6(quant_us),
                "product_us": cm.fixed6(product_us), "layer_us_hot": cm.fixed6(layer_us),
                "product_tflops": cm.fixed6(product.flops / product_us / 1e6),
                "product_weight_gbs": cm.fixed6(weight_bytes / product_us / 1e3), "few_rows": info["few_rows"],
                "tile_m": info["tile_m"], "tile_n": info["tile_n"], "grid_ctas": info["grid_ctas"],
                "rel_frobenius_sampled": f"{err:.6e}", "correctness": "pass" if ok else "fail", "gpu_name": gpu.name,
                "git_commit": commit})
            quant.close()
            product.close()

    out = sys.stdout if args.output == "-" else open(args.output, "w", newline="")
    writer = csv.DictWriter(out, fieldnames=FIELDS, lineterminator="\n")
    writer.writeheader()
    writer.writerows(rows)
    if out is not sys.stdout:
        out.close()
    return 1 if failed else 0


if __name__ == "__main__":
    raise SystemExit(main())
