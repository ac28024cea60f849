"""The quantised linear layer's product (LowpLinearPlan) on the GPU: against
64-bit products of the decoded operands, from one row to several tiles, at
odd widths and K, into strided and differently typed D; and the layer as it is
used, from the residual stream through quantiser and product."""
import pytest
import torch

from gb300_microbench_b200 import lowp, quantize

pytestmark = pytest.mark.gpu

KINDS = ["nvfp4", "mxfp4", "fp8"]
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _exact_operand(kind, rows, k, gen, weights):
    """Small integers with power-of-two scales: every product and sum is exact in FP32."""
    if kind == "fp8":
        q = torch.randint(-15, 16, (rows, k), generator=gen).float().to(torch.float8_e4m3fn).view(torch.uint8)
        kb = -(-k // 128)
        s = torch.exp2(torch.randint(-1, 2, (-(-rows // 128) if weights else rows, kb), generator=gen).float())
        return lowp.Fp8BlockOperand.from_parts(q, s) if weights else lowp.Fp8GroupOperand.from_parts(q, s)
    codes = torch.randint(0, 256, (rows, k // 2), generator=gen, dtype=torch.uint8)
    if kind == "mxfp4":
        return lowp.Mxfp4Operand.from_parts(codes, torch.randint(126, 129, (rows, k // 32), generator=gen).to(torch.uint8))
    bits = ((torch.randint(-1, 2, (rows, k // 16), generator=gen) + 7) << 3).to(torch.uint8)
    return lowp.Nvfp4Operand.from_parts(codes, bits, 0.5 if weights else 2.0)


def _quantised_operand(kind, rows, k, gen, weights):
    x = torch.randn(rows, k, generator=gen) * torch.exp(torch.randn(k, generator=gen) * 0.3)
    if kind == "fp8":
        return lowp.Fp8BlockOperand(x) if weights else lowp.Fp8GroupOperand(x)
    return lowp.Mxfp4Operand(x) if kind == "mxfp4" else lowp.Nvfp4Operand(x)


def _decode(op):
    if isinstance(op, lowp.Fp8BlockOperand):
        s = op.scales.double().repeat_interleave(128, 0).repeat_interleave(128, 1)[:op.rows, :op.k]
        return op.data.view(torch.float8_e4m3fn).double() * s
    if isinstance(op, lowp.Fp8GroupOperand):
        return op.values.double() * op.scales.double().repeat_interleave(128, 1)[:, :op.k]
    if isinstance(op, lowp.Mxfp4Operand):
        return lowp.mxfp4_dequantize(op.data, lowp.unpack_scale_atoms(op.atoms, op.rows, op.k // 32)).double()
    g = op.tensor_scale if op.tensor_scale is not None else float(op.tensor_scale_out)
    bits = lowp.unpack_scale_atoms(op.atoms, op.rows, op.k // 16)
    return lowp.nvfp4_dequantize(op.data, bits, 1.0).double() * g


def _run(x, w, dev, dtype=torch.bfloat16, d=None):
    if d is None:
        d = torch.full((x.rows, w.rows), float("nan"), dtype=dtype, device=dev)
    plan = lowp.LowpLinearPlan(x.to(dev), w.to(dev), d)
    plan.run()
    plan.synchronize()
    assert plan.launches >= (1 if x.rows else 0)
    first = d.clone()
    plan.run()
    plan.synchronize()
    assert torch.equal(first.view(torch.uint8), d.view(torch.uint8)) if d.is_contiguous() else torch.equal(first, d)
    plan.close()
    return d.cpu()


def _check(x, w, d):
    """Half a step of D's type, and FP32 accumulation: K / 32 + 32 additions (one instruction adds 32 or 64
    products to the running sum) that lose at most a quarter step 2^-22 of the sum of magnitudes each, and the
    scales' products."""
    a, b = _decode(x), _decode(w)
    want = a @ b.T
    bound = HALF_STEP[d.dtype] * want.abs() * (1 + 2.0 ** -8) + (x.k / 32 + 32) * 2.0 ** -22 * (a.abs() @ b.abs().T)
    if d.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # its subnormal step
    err = (d.double() - want).abs()
    assert (err <= bound).all(), float((err / bound.clamp(min=1e-300)).max())


def _round_up(k, kind):
    step = 16 if kind == "fp8" else 32
    return -(-k // step) * step


ROWS = [1, 2, 7, 15, 16, 17, 32, 33, 61, 64, 65, 127, 128, 129, 200, 256, 257, 300, 520]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", ROWS)
def test_exact_rows(cuda_device, kind, m):
    gen = torch.Generator().manual_seed(m)
    n, k = 264, 544
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    want = _decode(x) @ _decode(w).T
    assert torch.equal(_run(x, w, cuda_device, torch.float32).double(), want)
    d = _run(x, w, cuda_device)
    assert torch.equal(d, want.float().to(torch.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 40, 130])
@pytest.mark.parametrize("n", [1, 7, 8, 100, 127, 128, 129, 255, 257, 1000, 2052])
def test_exact_widths(cuda_device, kind, m, n):
    gen = torch.Generator().manual_seed(n)
    k = 288
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    want = _decode(x) @ _decode(w).T
    assert torch.equal(_run(x, w, cuda_device), want.float().to(torch.bfloat16))


# Token tiles of the FP8 kernel for few rows, with and without K split: several tiles of 16 or 32 tokens,
# the last one with a single token, and 128 tokens.
@pytest.mark.parametrize("m,n,k,tile,split", [
    (17, 264, 544, 16, True), (129, 1000, 288, 16, False), (100, 264, 1040, 16, True), (513, 264, 528, 16, False),
    (257, 140, 4096, 32, True), (193, 777, 1056, 32, True), (1281, 264, 528, 32, False), (65, 12000, 528, 32, False),
    (513, 640, 2048, 128, True), (600, 1100, 4096, 128, True), (300, 6000, 528, 128, False), (1000, 500, 8192, 128, True)])
def test_exact_fp8_tiles(cuda_device, m, n, k, tile, split):
    gen = torch.Generator().manual_seed(m)
    x, w = _exact_operand("fp8", m, k, gen, False), _exact_operand("fp8", n, k, gen, True)
    want = _decode(x) @ _decode(w).T
    d = torch.full((m + 2, n + 3), 7.0, device=cuda_device)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d[:m, :n])
    assert plan.info["few_rows"] and plan.info["tile_m"] == tile and (plan.info["k_splits"] > 1) == split
    plan.run(3)
    plan.synchronize()
    assert torch.equal(d[:m, :n].cpu().double(), want)
    assert (d[m:] == 7).all() and (d[:, n:] == 7).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 24, 257])
@pytest.mark.parametrize("k", [16, 32, 64, 96, 128, 144, 160, 256, 272, 512, 1040, 2880, 4096])
def test_exact_depths(cuda_device, kind, m, k):
    gen = torch.Generator().manual_seed(k)
    k = _round_up(k, kind)
    n = 140
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    want = _decode(x) @ _decode(w).T
    # Sums of K products of at most 15 * 15 * 4: exact in FP32 below 2^24 half-units.
    assert torch.equal(_run(x, w, cuda_device, torch.float32).double(), want)


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (5, 1000, 2880), (61, 5000, 2912), (128, 256, 8192), (200, 777, 1056),
                                   (513, 640, 2048), (1024, 1032, 1024)])
def test_quantised_normal(cuda_device, kind, dtype, m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    x, w = _quantised_operand(kind, m, k, gen, False), _quantised_operand(kind, n, k, gen, True)
    _check(x, w, _run(x, w, cuda_device, dtype))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("n,pad,shift", [(264, 8, 0), (264, 3, 1), (96, 8, 8), (131, 0, 0)])
def test_strided_output(cuda_device, kind, dtype, m, n, pad, shift):
    """D inside a wider tensor; what lies beside and behind it stays as it was."""
    gen = torch.Generator().manual_seed(n)
    k = 160
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    full = torch.full((m + 2, n + pad + shift), -7.0, dtype=dtype, device=cuda_device)
    _run(x, w, cuda_device, d=full[1:1 + m, shift:shift + n])
    want = torch.full(full.shape, -7.0, dtype=dtype)
    want[1:1 + m, shift:shift + n] = (_decode(x) @ _decode(w).T).float().to(dtype)
    assert torch.equal(full.cpu(), want)


# More than one tile of 128 x 128 per SM: the kernel of 256 x 256 tiles.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1921, 1300, 288), (257, 12808, 144), (2048, 2048, 1040), (16100, 200, 96),
                                   (1400, 1801, 32)])
def test_exact_many_tiles(cuda_device, kind, m, n, k):
    gen = torch.Generator().manual_seed(m)
    k = _round_up(k, kind)
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    want = _decode(x) @ _decode(w).T
    d = torch.full((m, n), float("nan"), dtype=torch.bfloat16, device=cuda_device)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d)
    assert plan.info["few_rows"] == 0
    plan.run()
    plan.synchronize()
    assert torch.equal(d.cpu(), want.float().to(torch.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("pad,shift", [(0, 0), (3, 1), (8, 8)])
def test_many_tiles_strided_output(cuda_device, kind, dtype, pad, shift):
    gen = torch.Generator().manual_seed(pad)
    m, n, k = 1500, 1700, 160
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    full = torch.full((m + 2, n + pad + shift), -7.0, dtype=dtype, device=cuda_device)
    d = full[1:1 + m, shift:shift + n]
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d)
    assert plan.info["few_rows"] == 0
    plan.run()
    plan.synchronize()
    want = torch.full(full.shape, -7.0, dtype=dtype)
    want[1:1 + m, shift:shift + n] = (_decode(x) @ _decode(w).T).float().to(dtype)
    assert torch.equal(full.cpu(), want)


# Token tiles of the 4-bit kernels for few rows with K split over clusters, and of 128 tokens on shared SMs.
@pytest.mark.parametrize("kind", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("m,n,k,tile", [(9, 300, 8192, 16), (30, 129, 8192, 32), (51, 300, 8192, 64), (64, 1000, 14336, 64),
                                        (100, 300, 8192, 128), (257, 700, 12320, 128), (190, 9217, 8192, 128)])
def test_exact_fp4_splits(cuda_device, kind, m, n, k, tile):
    gen = torch.Generator().manual_seed(m)
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    want = (_decode(x).to(cuda_device) @ _decode(w).to(cuda_device).T).float()
    d = torch.full((m + 2, n + 3), 7.0, device=cuda_device)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d[:m, :n])
    assert plan.info["few_rows"] and plan.info["tile_m"] == tile and plan.info["k_splits"] > 1
    plan.run(3)
    plan.synchronize()
    assert torch.equal(d[:m, :n], want)
    assert (d[m:] == 7).all() and (d[:, n:] == 7).all()


# Three waves of 256 x 256 tiles and a long K: CTA pairs for every kind; a few K: one CTA per tile.
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,pad,dtype,pairs", [
    (2300, 4304, 8192, 0, torch.bfloat16, True), (2300, 4303, 8192, 2, torch.float32, True),
    (2300, 4301, 8192, 0, torch.float16, True), (1400, 3304, 576, 0, torch.bfloat16, False),
    (1400, 3303, 576, 2, torch.bfloat16, False), (2304, 4304, 1040, 0, torch.bfloat16, True)])
def test_tiles_of_pairs_and_single_ctas(cuda_device, kind, m, n, k, pad, dtype, pairs):
    gen = torch.Generator().manual_seed(n)
    k = _round_up(k, kind)
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    rows = torch.cat([torch.arange(0, m, 37), torch.arange(m - 4, m)])
    want = (_decode(x)[rows].float().to(cuda_device).double() @ _decode(w).float().to(cuda_device).double().T).float()
    full = torch.full((m, n + pad), -7.0, dtype=dtype, device=cuda_device)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), full[:, :n])
    assert plan.info["few_rows"] == 0 and plan.info["cta_group"] == (2 if pairs else 1)
    plan.run(2)
    plan.synchronize()
    assert torch.equal(full[rows.to(cuda_device), :n], want.to(dtype))
    assert (full[:, n:] == -7).all()


@pytest.mark.parametrize("dtype", list(HALF_STEP))
@pytest.mark.parametrize("kind", KINDS)
def test_many_tiles_quantised(cuda_device, kind, dtype):
    gen = torch.Generator().manual_seed(77)
    x, w = _quantised_operand(kind, 2100, 2080, gen, False), _quantised_operand(kind, 1430, 2080, gen, True)
    _check(x, w, _run(x, w, cuda_device, dtype))


@pytest.mark.parametrize("kind", KINDS)
def test_weights_written_just_before(cuda_device, kind):
    """Launches overlap the ones before them: weights and tokens filled by the launch right in front must
    be the ones multiplied, every time."""
    gen = torch.Generator().manual_seed(3)
    for m, n, k in ((1, 2048, 1024), (40, 1000, 512), (2000, 1664, 256)):
        x = _quantised_operand(kind, m, k, gen, False).to(cuda_device)
        sets = [_quantised_operand(kind, n, k, gen, True).to(cuda_device) for _ in range(4)]
        w = _quantised_operand(kind, n, k, gen, True).to(cuda_device)
        scales = (lambda op: op.scales) if kind == "fp8" else (lambda op: op.atoms)
        if kind == "nvfp4":
            for op in sets:
                op.tensor_scale = w.tensor_scale
        outs = [torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device) for _ in sets]
        plans = [lowp.LowpLinearPlan(x, w, d) for d in outs]
        own = [lowp.LowpLinearPlan(x, op, torch.empty_like(outs[0])) for op in sets]
        for _ in range(3):
            for op, plan in zip(sets, plans):
                w.data.copy_(op.data)
                scales(w).copy_(scales(op))
                plan.run()
        for p in own:
            p.run()
        torch.cuda.synchronize(cuda_device)
        for d, p in zip(outs, own):
            assert torch.equal(d, p.d)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_weights_quantised_just_before(cuda_device, fmt):
    """A weight update: new weights quantised by the plan in front of the product, which starts early."""
    gen = torch.Generator().manual_seed(4)
    make = lowp.Mxfp4Operand if fmt == "mxfp4" else lowp.Nvfp4Operand
    n, k = 1536, 2048
    src = torch.empty(n, k, dtype=torch.bfloat16, device=cuda_device)
    w = make.empty(n, k, device=cuda_device)
    x = _quantised_operand(fmt, 3, k, gen, False).to(cuda_device)
    d = torch.empty(3, n, dtype=torch.float32, device=cuda_device)
    fill, product = quantize.Fp4QuantPlan(src, w), lowp.LowpLinearPlan(x, w, d)
    new = [torch.randn(n, k, generator=gen).to(torch.bfloat16).to(cuda_device) * (1 + i) for i in range(5)]
    got = []
    for t in new:
        src.copy_(t)
        for _ in range(2):
            fill.run()
            product.run()
        got.append(d.clone())
    torch.cuda.synchronize(cuda_device)
    for t, g in zip(new, got):
        ref = make(t.cpu())
        want = _decode(x.to("cpu")) @ _decode(ref).T
        bound = 2.0 ** -24 * want.abs() + (k / 32 + 32) * 2.0 ** -22 * (_decode(x.to("cpu")).abs() @ _decode(ref).abs().T)
        assert ((g.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k,pairs", [(2300, 4304, 8192, True), (1400, 3304, 576, False)])
def test_activations_quantised_just_before(cuda_device, kind, m, n, k, pairs):
    """Quantiser and tile kernel in turn with nothing between them, each launch starting before the one in
    front has ended: every product is of its own step's tokens and scales, which lie at one address."""
    gen = torch.Generator(device=cuda_device).manual_seed(9)
    w = {"fp8": lowp.Fp8BlockOperand, "mxfp4": lowp.Mxfp4Operand, "nvfp4": lowp.Nvfp4Operand}[kind](
        torch.randn(n, k, generator=gen, device=cuda_device))
    empty = {"fp8": lowp.Fp8GroupOperand, "mxfp4": lowp.Mxfp4Operand, "nvfp4": lowp.Nvfp4Operand}[kind].empty
    weight = torch.ones(k, device=cuda_device)

    def quantiser(x, a, i):
        return quantize.RmsNormFp8Plan(x, weight * 4.0 ** i, a) if kind == "fp8" else quantize.Fp4QuantPlan(x, a)

    shared = empty(m, k, device=cuda_device)
    steps, want = [], []
    for i in range(5):
        x = torch.randn(m, k, generator=gen, device=cuda_device) * 4.0 ** (i - 2)
        x *= torch.exp(torch.randn(m, 1, generator=gen, device=cuda_device))
        x = x.to(torch.bfloat16)
        alone = empty(m, k, device=cuda_device)
        plans = [quantiser(x, alone, i)] + [lowp.LowpLinearPlan(alone, w, torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device))]
        for p in plans:
            p.run()
            p.synchronize()
        want.append(plans[1].d)
        rows = torch.randint(0, m, (16,), generator=gen, device=cuda_device)
        _check(_rows_of(alone.to("cpu"), rows.cpu()), w.to("cpu"), plans[1].d[rows].cpu())
        product = lowp.LowpLinearPlan(shared, w, torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device))
        assert product.info["few_rows"] == 0 and product.info["cta_group"] == (2 if pairs else 1)
        steps.append((quantiser(x, shared, i), product))
    torch.cuda.synchronize(cuda_device)
    for _ in range(4):
        for _, product in steps:
            product.d.zero_()
        for quantiser_, product in steps:
            quantiser_.run()
            product.run()
        torch.cuda.synchronize(cuda_device)
        for (_, product), d in zip(steps, want):
            product.synchronize()
            assert torch.equal(product.d, d)


def _rows_of(op, rows):
    """The operand of some of its rows."""
    if isinstance(op, lowp.Fp8GroupOperand):
        return lowp.Fp8GroupOperand.from_parts(op.data[rows], op.scales[rows])
    mx = isinstance(op, lowp.Mxfp4Operand)
    bits = lowp.unpack_scale_atoms(op.atoms, op.rows, op.k // (32 if mx else 16))[rows]
    return lowp.Mxfp4Operand.from_parts(op.data[rows], bits) if mx else \
        lowp.Nvfp4Operand.from_parts(op.data[rows], bits, float(op.tensor_scale_out))


@pytest.mark.parametrize("kind", KINDS)
def test_nan_stays_in_its_row(cuda_device, kind):
    gen = torch.Generator().manual_seed(5)
    k, n = 256, 136
    for m in (3, 200):
        x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
        want = (_decode(x) @ _decode(w).T).float().to(torch.bfloat16)
        if kind == "fp8":
            x.data[m - 2, 7] = 0x7F
        else:
            bits = lowp.unpack_scale_atoms(x.atoms, m, k // (32 if kind == "mxfp4" else 16))
            bits[m - 2, 1] = 0xFF if kind == "mxfp4" else 0x7F
            x.atoms = lowp.pack_scale_atoms(bits)
            if kind == "nvfp4":
                x.scales = bits  # what .to() lays the atoms out from
        d = _run_once(x, w, cuda_device)
        assert torch.isnan(d[m - 2]).all()
        keep = [i for i in range(m) if i != m - 2]
        assert torch.equal(d[keep], want[keep])


def _run_once(x, w, dev):
    d = torch.empty(x.rows, w.rows, dtype=torch.bfloat16, device=dev)
    plan = lowp.LowpLinearPlan(x.to(dev), w.to(dev), d)
    plan.run()
    plan.synchronize()
    return d.cpu()


@pytest.mark.parametrize("kind", KINDS)
def test_no_rows(cuda_device, kind):
    gen = torch.Generator().manual_seed(0)
    w = _exact_operand(kind, 40, 64, gen, True)
    x = {"fp8": lowp.Fp8GroupOperand, "mxfp4": lowp.Mxfp4Operand, "nvfp4": lowp.Nvfp4Operand}[kind].empty(0, 64, device="cpu")
    assert _run(x, w, cuda_device).shape == (0, 40)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [1, 64, 260])
def test_layer_chain(cuda_device, kind, m):
    """Residual stream -> quantiser -> product, captured once and replayed on new tokens, beside a second
    layer that runs on another stream at the same time."""
    k, n = 512, 1000
    gen = torch.Generator().manual_seed(m)
    layers = []
    for _ in range(2):
        stream = torch.cuda.Stream(device=cuda_device)
        w = _quantised_operand(kind, n, k, gen, True).to(cuda_device)
        x = torch.empty(m, k, dtype=torch.bfloat16, device=cuda_device)
        d = torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device)
        if kind == "fp8":
            a = lowp.Fp8GroupOperand.empty(m, k, device=cuda_device)
            res = torch.empty_like(x)
            first = quantize.RmsNormFp8Plan(x, torch.ones(k, device=cuda_device), a, residual=res, residual_out=res,
                                            stream=stream)
        else:
            a = (lowp.Mxfp4Operand if kind == "mxfp4" else lowp.Nvfp4Operand).empty(m, k, device=cuda_device)
            res = None
            first = quantize.Fp4QuantPlan(x, a, stream=stream)
        layers.append((stream, x, res, a, w, d, first, lowp.LowpLinearPlan(a, w, d, stream=stream)))
    torch.cuda.synchronize(cuda_device)
    graphs = []
    for stream, *_, first, product in layers:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            first.run()
            product.run()
        graphs.append(graph)
    for step in range(3):
        for i, (stream, x, res, *_) in enumerate(layers):
            x.copy_(torch.randn(m, k, generator=gen).to(torch.bfloat16) * (1 + step + i))
            if res is not None:
                res.copy_(torch.randn(m, k, generator=gen).to(torch.bfloat16))
        torch.cuda.synchronize(cuda_device)
        for (stream, *_), graph in zip(layers, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize(cuda_device)
        for stream, x, res, a, w, d, first, product in layers:
            first.synchronize()
            product.synchronize()
            if kind == "fp8":  # res holds the sum now: the norm of it is what was quantised
                y = res.double() / torch.sqrt((res.double() ** 2).mean(1, keepdim=True) + 1e-6)
                got = _decode(a)
                assert ((got - y).abs() <= y.abs() * 2.0 ** -4 * (1 + 2.0 ** -8)
                        + a.scales.double().repeat_interleave(128, 1) * 2.0 ** -10).all()
            else:
                ref = (lowp.mxfp4_quantize if kind == "mxfp4" else lowp.nvfp4_quantize)(x.cpu())
                assert torch.equal(a.data.cpu(), ref[0])
            _check(a.to("cpu"), w.to("cpu"), d.cpu())


def test_refusals_on_the_gpu(cuda_device):
    gen = torch.Generator().manual_seed(1)
    x, w = _exact_operand("mxfp4", 4, 64, gen, False), _exact_operand("mxfp4", 8, 64, gen, True)
    d = torch.empty(4, 8, dtype=torch.bfloat16, device=cuda_device)
    with pytest.raises(ValueError, match="CUDA"):
        lowp.LowpLinearPlan(x, w.to(cuda_device), d)
    w2 = w.to(cuda_device)
    w2.atoms = w2.atoms[:, :0]
    with pytest.raises(ValueError, match="scales"):
        lowp.LowpLinearPlan(x.to(cuda_device), w2, d)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d)
    from gb300_microbench_b200 import _native as nat
    with pytest.raises(nat.NativeCallError):
        plan.run(-1)
    plan.run(0)
    assert plan.launches == 0


@pytest.mark.parametrize("kind", KINDS)
def test_output_stride_past_32_bits(cuda_device, kind):
    """Rows of D 2^31 elements apart."""
    gen = torch.Generator().manual_seed(6)
    m, n, k = 3, 200, 96
    x, w = _exact_operand(kind, m, k, gen, False), _exact_operand(kind, n, k, gen, True)
    big = torch.empty(2 * (1 << 31) + n, dtype=torch.bfloat16, device=cuda_device)
    d = big.as_strided((m, n), (1 << 31, 1))
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w.to(cuda_device), d)
    plan.run()
    plan.synchronize()
    assert torch.equal(d.cpu(), (_decode(x) @ _decode(w).T).float().to(torch.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
def test_large_output(cuda_device, kind):
    """More than 2^32 elements of D (the tile kernel): identical rows of x give identical rows of D."""
    gen = torch.Generator().manual_seed(7)
    m, n, k = 66000, 65600, 64
    base = _exact_operand(kind, 200, k, gen, False)
    w = _exact_operand(kind, n, k, gen, True).to(cuda_device)
    reps = m // 200
    if kind == "fp8":
        x = lowp.Fp8GroupOperand.from_parts(base.data.repeat(reps, 1), base.scales.repeat(reps, 1))
    else:
        bits = lowp.unpack_scale_atoms(base.atoms, 200, k // (32 if kind == "mxfp4" else 16))
        parts = (base.data.repeat(reps, 1), bits.repeat(reps, 1))
        x = lowp.Mxfp4Operand.from_parts(*parts) if kind == "mxfp4" else lowp.Nvfp4Operand.from_parts(*parts, base.tensor_scale)
    d = torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device)
    plan = lowp.LowpLinearPlan(x.to(cuda_device), w, d)
    assert plan.info["few_rows"] == 0
    plan.run()
    plan.synchronize()
    first = (_decode(base) @ _decode(w.to("cpu")).T).float().to(torch.bfloat16).to(cuda_device)
    for rep in (0, reps // 2, reps - 1):
        assert torch.equal(d[200 * rep:200 * rep + 200], first)


@pytest.mark.parametrize("kind", ["mxfp4", "fp8"])
def test_captured_fork_and_join(cuda_device, kind):
    """The layer inside a graph whose streams fork and join around it: copies and kernels of other streams
    in front of it, readers behind it."""
    gen = torch.Generator().manual_seed(8)
    m, k, n = 20, 512, 640
    main, side = torch.cuda.Stream(device=cuda_device), torch.cuda.Stream(device=cuda_device)
    w = _quantised_operand(kind, n, k, gen, True).to(cuda_device)
    src = torch.empty(m, k, dtype=torch.bfloat16, device=cuda_device)
    x, res = torch.empty_like(src), torch.empty_like(src)
    d, behind = (torch.empty(m, n, dtype=torch.bfloat16, device=cuda_device) for _ in range(2))
    if kind == "fp8":
        a = lowp.Fp8GroupOperand.empty(m, k, device=cuda_device)
        first = quantize.RmsNormFp8Plan(x, torch.ones(k, device=cuda_device), a, residual=res, stream=main)
    else:
        a = lowp.Mxfp4Operand.empty(m, k, device=cuda_device)
        first = quantize.Fp4QuantPlan(x, a, stream=main)
    product = lowp.LowpLinearPlan(a, w, d, stream=main)
    torch.cuda.synchronize(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        side.wait_stream(main)
        with torch.cuda.stream(side):
            x.copy_(src)
            res.copy_(src)
            res.mul_(0.5)
        main.wait_stream(side)
        first.run()
        product.run()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            behind.copy_(d)
        product.run()
        main.wait_stream(side)
        d.zero_()
    for i in range(3):
        src.copy_(torch.randn(m, k, generator=gen).to(torch.bfloat16) * (i + 1))
        torch.cuda.synchronize(cuda_device)
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        assert not d.any()
        _check(a.to("cpu"), w.to("cpu"), behind.cpu())
        if kind == "mxfp4":
            assert torch.equal(a.data.cpu(), lowp.mxfp4_quantize(src.cpu())[0])


@pytest.mark.parametrize("op", ["norm_fp8", "fp4_quantize", "fp4_linear"])
def test_measured_pass_under_another_stream(cuda_device, op, monkeypatch):
    """A pass of perf/operators.py under a stream that is not its plans': behind the copy that fills x there,
    and before what reads the outputs there."""
    from perf import operators

    monkeypatch.setattr(operators, "own", True)
    case = next(c for c in operators.listed() if c["op"] == op)
    s, other = operators.prepare(case, 1), operators.prepare(case, 2)
    first = {k: v.clone() for k, v in operators.run(s).items()}
    x = s["x"].clone()
    s["x"].copy_(other["x"])
    operators.run(s)  # what stale outputs would hold
    torch.cuda.synchronize(cuda_device)
    side = torch.cuda.Stream(device=cuda_device)
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.cuda._sleep(20_000_000)  # about 10 ms
            s["x"].copy_(x)
            got = {k: v.clone() for k, v in operators.run(s).items()}
            s["x"].copy_(other["x"])
    torch.cuda.synchronize(cuda_device)
    for k, v in first.items():
        assert torch.equal(got[k].contiguous().view(torch.uint8), v.contiguous().view(torch.uint8))
