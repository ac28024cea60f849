"""The operators of a quantised linear layer, as they are measured: RMS norm
with the residual's addition and FP8 output, the FP8 product of activations
scaled per row and 128 columns, the quantisation to 4-bit microscaled formats
(NVFP4, MXFP4) and the 4-bit product behind it.

Every operator has its plain form here (elementary torch operations in 32
bits) and the framework's own calls; ``own`` says which of them ``run`` makes.
"""
import math

import torch

own = False

E4M3_MAX = 448.0
E2M1_MAX = 6.0
GROUP = 128  # columns that share one FP8 scale
EPS = 1e-6

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One token of a decoding step: latency of one launch.
        {"name": "norm_fp8_one_token", "op": "norm_fp8", "rows": 1, "cols": 4096, "dtype": "bf16"},
        # A batch of short requests; the last scale group of a row is half full.
        {"name": "norm_fp8_batch", "op": "norm_fp8", "rows": 333, "cols": 2880, "dtype": "fp16"},
        # A long prompt: all tokens of a prefill chunk at once.
        {"name": "norm_fp8_prompt", "op": "norm_fp8", "rows": 16384, "cols": 8192, "dtype": "bf16"},
        # One token against a wide projection: the weights' bytes are the work.
        {"name": "fp8_linear_one_token", "op": "fp8_linear", "m": 1, "n": 14336, "k": 4096},
        # A decoding batch, an output width no tile divides and a K that ends inside a scale block.
        {"name": "fp8_linear_batch", "op": "fp8_linear", "m": 61, "n": 5000, "k": 2896},
        # A prefill at this repository's own largest GEMM size.
        {"name": "fp8_linear_prompt", "op": "fp8_linear", "m": 8192, "n": 8192, "k": 8192},
        # A decoding batch's activations, tensor scale known from calibration.
        {"name": "nvfp4_quantize_batch", "op": "fp4_quantize", "fmt": "nvfp4", "rows": 77, "cols": 4096,
         "dtype": "bf16", "scale": "given"},
        # A prefill's activations.
        {"name": "mxfp4_quantize_prompt", "op": "fp4_quantize", "fmt": "mxfp4", "rows": 16384, "cols": 8192,
         "dtype": "bf16", "scale": "none"},
        # A weight matrix at load time: the tensor scale is found from the data.
        {"name": "nvfp4_quantize_weights", "op": "fp4_quantize", "fmt": "nvfp4", "rows": 14336, "cols": 4096,
         "dtype": "fp32", "scale": "found"},
        # One token: its quantisation and the product with a square projection.
        {"name": "nvfp4_linear_one_token", "op": "fp4_linear", "fmt": "nvfp4", "m": 1, "n": 8192, "k": 8192},
        # A ragged batch between decoding and prefill.
        {"name": "mxfp4_linear_batch", "op": "fp4_linear", "fmt": "mxfp4", "m": 200, "n": 5000, "k": 2880},
        # A prefill: quantisation of the activations and the product.
        {"name": "mxfp4_linear_prompt", "op": "fp4_linear", "fmt": "mxfp4", "m": 8192, "n": 8192, "k": 8192},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_fp8", "fp8_linear", "fp4_quantize", "fp4_linear"])
    if op == "norm_fp8":
        rows = _log_int(rng, 1, 16384)
        cols = _log_int(rng, 256, 12288)
        if rng.random() < 0.75:  # models' widths are mostly multiples of 16
            cols = max(16, cols // 16 * 16)
        rows = max(1, min(rows, 16384 * 8192 // cols))
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])
                if rows * cols <= 16384 * 4096 else "bf16"}
    if op == "fp4_quantize":
        rows = _log_int(rng, 1, 16384)
        cols = 32 * _log_int(rng, 4, 400)
        rows = max(1, min(rows, 16384 * 4096 // cols))
        fmt = rng.choice(["nvfp4", "mxfp4"])
        return {"op": op, "fmt": fmt, "rows": rows, "cols": cols, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "scale": "none" if fmt == "mxfp4" else rng.choice(["given", "found"])}
    m = _log_int(rng, 1, 8192)
    n = _log_int(rng, 64, 16384)
    if rng.random() < 0.75:
        n = max(8, n // 8 * 8)
    step = 16 if op == "fp8_linear" else 32
    k = step * _log_int(rng, 256 // step, 14336 // step)
    m = max(1, min(m, 8192 ** 3 // (n * k)))
    if op == "fp8_linear":
        return {"op": op, "m": m, "n": n, "k": k}
    return {"op": op, "fmt": rng.choice(["nvfp4", "mxfp4"]), "m": m, "n": n, "k": k}


# ------------------------------------------------------------------ formats, in 32 bits
def _e2m1_round(y):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), signed; |y| is cut at 6."""
    a = y.abs().clamp(max=E2M1_MAX)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, y)


def _pad_cols(t, width):
    return torch.nn.functional.pad(t, (0, width - t.shape[1])) if width != t.shape[1] else t


def _fp8_group_scales(y):
    """(R, ceil(C / 128)) scales amax / 448, 1 where a group is all zeros."""
    groups = -(-y.shape[1] // GROUP)
    amax = _pad_cols(y, groups * GROUP).view(y.shape[0], groups, GROUP).abs().amax(dim=2)
    return torch.where(amax > 0, amax / torch.full_like(amax, E4M3_MAX), torch.ones_like(amax))


def _spread(scales, block, cols):
    return scales.repeat_interleave(block, dim=1)[:, :cols]


def _fp4_blocks(x, fmt, tensor_scale):
    """(scales as stored, values / (tensor scale), tensor scale as a tensor) of x in 32 bits."""
    x = x.float()
    rows, cols = x.shape
    if fmt == "mxfp4":
        blocks = x.view(rows, cols // 32, 32)
        amax = blocks.abs().amax(dim=2)
        _, e = torch.frexp(amax)  # amax = f * 2^e with f in [0.5, 1)
        e = torch.where(amax > 0, e - 3, torch.full_like(e, -127)).clamp(-127, 127)
        # 2^e by its bits (2^-127 lies below the normal numbers).
        scale = torch.where(e > -127, (e + 127) << 23, torch.full_like(e, 1 << 22)).to(torch.int32).view(torch.float32)
        q = _e2m1_round(blocks / scale.unsqueeze(2))
        return (e + 127).to(torch.uint8), (q * scale.unsqueeze(2)).view(rows, cols), None
    blocks = x.view(rows, cols // 16, 16)
    # Divisors are tensors: a division by a number multiplies by its rounded reciprocal on a GPU, which moves
    # values that lie next to a border of the 8- or 4-bit grid.
    if tensor_scale is None:
        amax = x.abs().amax()
        tensor_scale = torch.where(amax > 0, amax / torch.full_like(amax, E4M3_MAX * E2M1_MAX), torch.ones_like(amax))
    else:
        tensor_scale = torch.full((), tensor_scale, device=x.device)
    amax = blocks.abs().amax(dim=2)
    scale8 = (amax / torch.full_like(amax, E2M1_MAX) / tensor_scale).clamp(max=E4M3_MAX).to(torch.float8_e4m3fn)
    scale = scale8.float()
    denom = (scale * tensor_scale).unsqueeze(2)
    y = torch.where(denom > 0, blocks / torch.where(denom > 0, denom, torch.ones_like(denom)),
                    torch.zeros_like(blocks))
    q = _e2m1_round(y)
    return scale8.view(torch.uint8), (q * scale.unsqueeze(2)).view(rows, cols), tensor_scale


def _atoms(scales):
    """(R, S) scale bytes -> (ceil(R / 128), ceil(S / 4), 512): the layout in which the tensor core reads
    them, scale j of row r at byte (r % 32) * 16 + (r / 32) * 4 + j of its atom, padding zero."""
    r, s = scales.shape
    rb, sg = -(-r // 128), -(-s // 4)
    padded = torch.nn.functional.pad(scales, (0, sg * 4 - s, 0, rb * 128 - r))
    return padded.view(rb, 4, 32, sg, 4).permute(0, 3, 2, 1, 4).reshape(rb, sg, 512)


def _as_scale_values(atoms, fmt):
    return atoms.view(torch.float8_e8m0fnu if fmt == "mxfp4" else torch.float8_e4m3fn)


def _pack_e2m1(q):
    """Values on the E2M1 grid -> two codes a byte, element 2i in the low nibble."""
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | ((q < 0) & (a > 0)).to(torch.uint8) << 3
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous()


def _unpack_e2m1(packed):
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=packed.device)
    return torch.stack((grid[(packed & 15).long()], grid[(packed >> 4).long()]), dim=2).view(packed.shape[0], -1)


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(g, rows, cols, dtype):
    """Activations as a residual stream has them: channels of different size, a few of them large."""
    channel = torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))
    channel[torch.randint(0, cols, (max(1, cols // 256),), generator=g, device="cuda")] *= 12
    return (torch.randn(rows, cols, generator=g, device="cuda") * channel).to(dtype)


def _fp8_block_weights(g, n, k):
    """(N, K) E4M3 weights and FP32 scales of their 128 x 128 blocks."""
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    nb, kb = -(-n // 128), -(-k // 128)
    blocks = torch.nn.functional.pad(w, (0, kb * 128 - k, 0, nb * 128 - n)).view(nb, 128, kb, 128)
    scale = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(nb * 128, kb * 128)[:n, :k].contiguous(), scale


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    s = {"case": case}
    if op == "norm_fp8":
        dtype = DTYPES[case["dtype"]]
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(g, rows, cols, dtype)
        s["residual"] = (3 * torch.randn(rows, cols, generator=g, device="cuda")).to(dtype)
        s["weight"] = (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(dtype)
        if own:
            from gb300_microbench_b200 import lowp, quantize

            s["out"] = lowp.Fp8GroupOperand.empty(rows, cols, device="cuda")
            s["residual_out"] = torch.empty_like(s["residual"])
            s["plan"] = quantize.RmsNormFp8Plan(s["x"], s["weight"], s["out"], residual=s["residual"],
                                                residual_out=s["residual_out"], eps=EPS)
    elif op == "fp8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = _activations(g, m, k, torch.float32)
        # The scales of one K block side by side, as the norm in front writes them.
        s["sx"] = _fp8_group_scales(x).t().contiguous().t()
        s["x"] = (x / _spread(s["sx"], GROUP, k)).to(torch.float8_e4m3fn)
        s["w"], s["sw"] = _fp8_block_weights(g, n, k)
        if own:
            from gb300_microbench_b200 import lowp

            a = lowp.Fp8GroupOperand.from_parts(s["x"], s["sx"])
            b = lowp.Fp8BlockOperand.from_parts(s["w"].view(torch.uint8), s["sw"])
            s["d"] = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
            s["plan"] = lowp.LowpLinearPlan(a, b, s["d"])
    elif op == "fp4_quantize":
        rows, cols, fmt = case["rows"], case["cols"], case["fmt"]
        s["x"] = _activations(g, rows, cols, DTYPES[case["dtype"]])
        # A calibrated scale: from another draw of the same distribution.
        s["tensor_scale"] = float(_activations(g, 64, cols, torch.float32).abs().max()) / (E4M3_MAX * E2M1_MAX) \
            if case["scale"] == "given" else None
        if own:
            from gb300_microbench_b200 import lowp, quantize

            if fmt == "mxfp4":
                s["out"] = lowp.Mxfp4Operand.empty(rows, cols, device="cuda")
            else:
                s["out"] = lowp.Nvfp4Operand.empty(rows, cols, device="cuda", tensor_scale=s["tensor_scale"])
            s["values"] = torch.empty_like(s["x"])
            s["plan"] = quantize.Fp4QuantPlan(s["x"], s["out"], values=s["values"])
    else:
        m, n, k, fmt = case["m"], case["n"], case["k"], case["fmt"]
        s["x"] = _activations(g, m, k, torch.bfloat16)
        s["tensor_scale"] = float(_activations(g, 64, k, torch.float32).abs().max()) / (E4M3_MAX * E2M1_MAX) \
            if fmt == "nvfp4" else None
        w = torch.randn(n, k, generator=g, device="cuda") * 0.02
        scales, values, w_scale = _fp4_blocks(w, fmt, None)
        unit = _spread(_as_scale_values(scales, fmt).float(), 32 if fmt == "mxfp4" else 16, k)
        q = torch.where(unit > 0, values / unit, 0.0)
        s["w"], s["sw"], s["w_scale"] = _pack_e2m1(q), scales, None if w_scale is None else float(w_scale)
        if own:
            from gb300_microbench_b200 import lowp, quantize

            if fmt == "mxfp4":
                a = lowp.Mxfp4Operand.empty(m, k, device="cuda")
                b = lowp.Mxfp4Operand.from_parts(s["w"], s["sw"])
            else:
                a = lowp.Nvfp4Operand.empty(m, k, device="cuda", tensor_scale=s["tensor_scale"])
                b = lowp.Nvfp4Operand.from_parts(s["w"], s["sw"], s["w_scale"])
            s["d"] = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
            s["quantize"] = quantize.Fp4QuantPlan(s["x"], a)
            s["plan"] = lowp.LowpLinearPlan(a, b, s["d"])
    if own:
        s["device"], s["stream"] = s["plan"].stream.device_index, s["plan"].stream.cuda_stream
    return s


# ------------------------------------------------------------------ one pass
def _on_the_plans_stream(s):
    """The pass behind what is queued on the current stream, and what is queued there next behind the pass."""
    current, stream = torch.cuda.current_stream(), s["plan"].stream
    stream.wait_stream(current)
    with torch.cuda.stream(stream):
        out = run(s)
    current.wait_stream(stream)
    return out


def run(s):
    # A plan runs on the stream that it was made for. (The current one's handle is read as it is: asking for a
    # stream object takes 1 to 3 us, as long as the smallest pass.)
    if own and torch._C._cuda_getCurrentRawStream(s["device"]) != s["stream"]:
        return _on_the_plans_stream(s)
    case = s["case"]
    op = case["op"]
    if op == "norm_fp8":
        if own:
            s["plan"].run()
            return {"residual": s["residual_out"], "q": s["out"].values, "scales": s["out"].scales}
        h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
        f = h.float()
        y = f * torch.rsqrt((f * f).mean(dim=1, keepdim=True) + EPS) * s["weight"].float()
        scales = _fp8_group_scales(y)
        q = (y / _spread(scales, GROUP, y.shape[1])).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        return {"residual": h, "q": q, "scales": scales}
    if op == "fp8_linear":
        if own:
            s["plan"].run()
            return {"d": s["d"]}
        n, k = s["w"].shape
        x = s["x"].float() * _spread(s["sx"], GROUP, k)
        w = s["w"].float() * _spread(s["sw"], 128, k).repeat_interleave(128, dim=0)[:n]
        return {"d": (x @ w.t()).to(torch.bfloat16)}
    if op == "fp4_quantize":
        if own:
            s["plan"].run()
            out = {"values": s["values"], "scales": _as_scale_values(s["out"].atoms, case["fmt"])}
            return {**out, "tensor_scale": s["out"].tensor_scale_out} if case["scale"] == "found" else out
        scales, values, tensor_scale = _fp4_blocks(s["x"], case["fmt"], s["tensor_scale"])
        if tensor_scale is not None:
            values = values * tensor_scale
        out = {"values": values.to(s["x"].dtype), "scales": _as_scale_values(_atoms(scales), case["fmt"])}
        return {**out, "tensor_scale": tensor_scale.view(1)} if case["scale"] == "found" else out
    if own:
        s["quantize"].run()
        s["plan"].run()
        return {"d": s["d"]}
    fmt = case["fmt"]
    _, x, x_scale = _fp4_blocks(s["x"], fmt, s["tensor_scale"])
    w = _unpack_e2m1(s["w"]) * _spread(_as_scale_values(s["sw"], fmt).float(), 32 if fmt == "mxfp4" else 16, case["k"])
    d = x @ w.t()
    return {"d": (d if x_scale is None else d * (x_scale * s["w_scale"])).to(torch.bfloat16)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm_fp8":
        t, c = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": t * c * (3 * size + 1) + t * -(-c // GROUP) * 4 + c * size, "flops": 8 * t * c}
    if op == "fp8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // 128)
        return {"bytes": m * k + n * k + 2 * m * n + 4 * kb * (m + -(-n // 128)), "flops": 2 * m * n * k}
    block = 32 if case["fmt"] == "mxfp4" else 16
    if op == "fp4_quantize":
        t, c = case["rows"], case["cols"]
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": 2 * t * c * size + t * c // 2 + -(-t // 128) * 128 * c // block, "flops": 4 * t * c}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": 2 * m * k + n * k // 2 + n * k // block + 2 * m * n, "flops": 2 * m * n * k}


# ------------------------------------------------------------------ the definitions in 64 bits
def _power_of_two(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _grid_round(v, mantissa, least, most):
    """v (float64) to the nearest value with `mantissa` fraction bits, steps no finer than 2^(least - mantissa),
    magnitude at most `most`; ties to even."""
    _, e = torch.frexp(v.abs())
    step = _power_of_two(torch.clamp(e - 1, min=least) - mantissa)
    return (torch.round(v / step) * step).clamp(-most, most)


def _exact_fp4(x, fmt, tensor_scale):
    """(scales' values (R, S), dequantised values, tensor scale) in 64 bits."""
    r, c = x.shape
    x = x.double()
    if fmt == "mxfp4":
        b = x.reshape(r, -1, 32)
        top = b.abs().max(dim=2).values
        e = torch.frexp(top).exponent - 3  # floor(log2) - 2: frexp's mantissa lies in [0.5, 1)
        scale = _power_of_two(torch.where(top > 0, e, torch.full_like(e, -127)).clamp(-127, 127))
        return scale, (_grid_round(b / scale[..., None], 1, 0, 6.0) * scale[..., None]).reshape(r, c), None
    g = x.abs().max() / (448 * 6) if tensor_scale is None else torch.tensor(tensor_scale, dtype=torch.float64, device=x.device)
    b = x.reshape(r, -1, 16)
    scale = _grid_round(b.abs().max(dim=2).values / (6 * g), 3, -6, 448.0)
    d = (scale * g)[..., None]
    q = torch.where(d > 0, _grid_round(b / torch.where(d > 0, d, 1.0), 1, 0, 6.0), 0.0)
    return scale, (q * d).reshape(r, c), g


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm_fp8":
        t, c = case["rows"], case["cols"]
        h = (s["x"].double() + s["residual"].double()).to(s["x"].dtype).double()
        y = h / torch.sqrt((h ** 2).sum(dim=1, keepdim=True) / c + EPS) * s["weight"].double()
        scales = torch.stack([y[:, i:i + GROUP].abs().max(dim=1).values for i in range(0, c, GROUP)], dim=1) / 448
        scales = torch.where(scales > 0, scales, 1.0)
        return {"residual": h, "q": _grid_round(y / scales[:, torch.arange(c, device=y.device) // GROUP], 3, -6, 448.0),
                "scales": scales}
    if op == "fp8_linear":
        m, n, k = case["m"], case["n"], case["k"]
        at_k = torch.arange(k, device="cuda") // 128
        w = s["w"].double() * s["sw"].double()[torch.arange(n, device="cuda") // 128][:, at_k]
        return {"d": torch.matmul(s["x"].double() * s["sx"].double()[:, at_k], w.T)}
    if op == "fp4_quantize":
        scale, values, g = _exact_fp4(s["x"], case["fmt"], s["tensor_scale"])
        r, c = scale.shape
        low = 2.0 ** -127 if case["fmt"] == "mxfp4" else 0.0  # what a zero byte stands for
        atoms = torch.full((-(-r // 128), -(-c // 4), 32, 4, 4), low, dtype=torch.float64, device="cuda")
        row, col = torch.arange(r, device="cuda")[:, None], torch.arange(c, device="cuda")[None, :]
        atoms[row // 128, col // 4, row % 32, row % 128 // 32, col % 4] = scale
        out = {"values": values, "scales": atoms.reshape(atoms.shape[0], atoms.shape[1], 512)}
        return {**out, "tensor_scale": g.reshape(1)} if case["scale"] == "found" else out
    fmt = case["fmt"]
    _, x, _ = _exact_fp4(s["x"], fmt, s["tensor_scale"])
    unit = _as_scale_values(s["sw"], fmt).double()
    w = _unpack_e2m1(s["w"]).double() * unit[:, torch.arange(case["k"], device="cuda") // (32 if fmt == "mxfp4" else 16)]
    return {"d": torch.matmul(x, w.T) * (1.0 if s["w_scale"] is None else s["w_scale"])}
