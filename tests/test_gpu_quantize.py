"""The quantisers on the GPU: RMS norm to FP8 against the formula in 64 bits,
the 4-bit formats against the torch definitions on the CPU bit for bit and
against 64 bits, at odd sizes, strides, empty and non-finite rows, on other
streams and in captured graphs."""
import pytest
import torch

from gb300_microbench_b200 import lowp, quantize

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24  # half a step of FP32, relative


def _x(rows, cols, dtype, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(0.5 * torch.randn(cols, generator=g)) * scale
    return x.to(dtype)


# ------------------------------------------------------------------ RMS norm -> FP8
def _norm_check(x, res, weight, eps, h_got, q_got, s_got):
    """x, res, weight on the CPU. The bounds: the sum of squares of positive terms is added in at most
    64 + 10 + 5 steps of half a step each, the root halves that; division by the width, the added eps and
    CUDA's rsqrtf (2 steps) and the two products of y add 2 + 4 + 2 half steps; a scale's division one more."""
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    if h_got is not None:
        assert torch.equal(h_got, h)
    f = h.double()
    cols = f.shape[1]
    y = f / torch.sqrt((f * f).sum(1, keepdim=True) / cols + eps) * weight.double()
    groups = -(-cols // 128)
    amax = torch.nn.functional.pad(y, (0, groups * 128 - cols)).view(-1, groups, 128).abs().amax(2)
    s = torch.where(amax > 0, amax / 448, 1.0)
    rel = (79 / 2 + 8 + 1) * U
    assert ((s_got.double() - s).abs() <= rel * s).all()
    # q is e4m3(y / s): half a step of E4M3 around a quotient that is off by what y and s are.
    want = y / s.repeat_interleave(128, 1)[:, :cols]
    half = torch.maximum(want.abs() * 2.0 ** -4, torch.full_like(want, 2.0 ** -10))
    err = (q_got.double() - want).abs()
    assert (err <= half * (1 + 2.0 ** -10) + 2 * rel * want.abs()).all(), float((err / half).max())


def _norm(x, weight, dev, res=None, eps=1e-6, store=True, stream=None):
    out = lowp.Fp8GroupOperand.empty(*x.shape, device=dev)
    xd, rd = x.to(dev), None if res is None else res.to(dev)
    ro = torch.empty_like(xd) if store else None
    plan = quantize.RmsNormFp8Plan(xd, weight.to(dev), out, residual=rd, residual_out=ro, eps=eps, stream=stream)
    plan.run()
    plan.synchronize()
    assert plan.launches == (1 if x.shape[0] else 0)
    plan.close()
    return None if ro is None else ro.cpu(), out.values.float().cpu(), out.scales.cpu()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 128), (5, 129), (4, 255), (1, 4096), (33, 2880),
                                       (7, 2900), (3, 8192), (2, 12288), (1, 32768), (2, 32776), (1, 65536),
                                       (1, 65535), (300, 257)])
def test_norm_sizes(cuda_device, dtype, rows, cols):
    x, res = _x(rows, cols, dtype), _x(rows, cols, dtype, seed=1, scale=3.0)
    w = (1 + 0.1 * torch.randn(cols, generator=torch.Generator().manual_seed(2))).to(dtype)
    _norm_check(x, res, w, 1e-6, *_norm(x, w, cuda_device, res))


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_without_residual_and_fp32_weight(cuda_device, dtype):
    x, w = _x(9, 520, dtype), torch.linspace(-2, 2, 520)
    _, q, s = _norm(x, w, cuda_device, store=False, eps=0.0)
    _norm_check(x, None, w, 0.0, None, q, s)


@pytest.mark.parametrize("pad,shift", [(8, 0), (1, 0), (3, 1), (8, 4)])
def test_norm_strides(cuda_device, pad, shift):
    """Rows inside wider tensors, aligned and not; what lies beside them stays."""
    rows, cols = 6, 264
    full = _x(rows, cols + pad + shift, torch.bfloat16, seed=4).to(cuda_device)
    res_full = _x(rows, cols + pad + shift, torch.bfloat16, seed=5).to(cuda_device)
    before = res_full.clone()
    x, res = full[:, shift:shift + cols], res_full[:, shift:shift + cols]
    w = torch.ones(cols, dtype=torch.bfloat16, device=cuda_device)
    out = lowp.Fp8GroupOperand.empty(rows, cols, device=cuda_device)
    x0, r0 = x.cpu().clone(), res.cpu().clone()
    plan = quantize.RmsNormFp8Plan(x, w, out, residual=res, residual_out=res)  # in place
    plan.run()
    plan.synchronize()
    _norm_check(x0, r0, w.cpu(), 1e-6, res.cpu().clone(), out.values.float().cpu(), out.scales.cpu())
    side = torch.ones(cols + pad + shift, dtype=torch.bool)
    side[shift:shift + cols] = False
    assert torch.equal(res_full[:, side.to(cuda_device)], before[:, side.to(cuda_device)])


def test_norm_zero_and_non_finite_rows(cuda_device):
    x = _x(5, 300, torch.float32)
    x[1] = 0
    x[2, 130] = float("nan")
    x[3, 5] = float("inf")
    w = torch.ones(300)
    _, q, s = _norm(x, w, cuda_device, store=False)
    for r in (0, 4):
        _norm_check(x[r:r + 1], None, w, 1e-6, None, q[r:r + 1], s[r:r + 1])
    assert (q[1] == 0).all() and (s[1] == 1).all()
    assert torch.isnan(q[2]).all() and torch.isnan(s[2]).all()
    assert torch.isnan(q[3, 5]) and torch.isnan(s[3, 0])


def _round_once(x, dtype):
    """FP64 to the nearest number of a 16-bit type, ties to even. (Tensor.to goes by way of FP32.)"""
    digits, least = (8, -133) if dtype == torch.bfloat16 else (11, -24)
    step = torch.exp2((torch.frexp(x).exponent - digits).clamp(min=least).double())
    return (torch.round(x / step) * step).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [4096, 4095])
def test_norm_sums_of_every_magnitude(cuda_device, dtype, cols):
    """h is x + residual rounded once, to the bit: all finite patterns, subnormal numbers and signed zeros
    among them, with sums at every distance of exponents."""
    g = torch.Generator().manual_seed(10)
    bits = [torch.randint(-2 ** 15, 2 ** 15, (64, cols), generator=g).to(torch.int16) for _ in range(2)]
    near = torch.randint(-2 ** 10, 2 ** 10, (32, cols), generator=g).to(torch.int16)  # exponents close by
    bits[1][:32] = bits[0][:32] ^ near
    bits[0][40:48] &= 0xFF  # subnormal and small numbers
    bits[1][44:52] &= 0x1FF
    x, res = (torch.where(torch.isfinite(b.view(dtype).float()), b, 0).view(dtype) for b in bits)
    h, _, _ = _norm(x, torch.ones(cols), cuda_device, res)
    want = _round_once(x.double() + res.double(), dtype)
    assert torch.equal(h.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [640, 637])
def test_norm_infinite_rows(cuda_device, dtype, cols):
    """The whole row: NaN in the infinity's group of 128, 0 with scale 1 in the others; by the residual's
    addition too."""
    big = torch.finfo(dtype).max
    x, res = _x(4, cols, dtype, seed=7), torch.zeros(4, cols, dtype=dtype)
    x[1, 200], x[2, cols - 1] = float("inf"), -float("inf")
    x[3, 5] = res[3, 5] = big
    w = torch.ones(cols)
    h, q, s = _norm(x, w, cuda_device, res)
    _norm_check(x[:1], res[:1], w, 1e-6, h[:1], q[:1], s[:1])
    assert torch.isinf(h[3, 5])
    for r, group in ((1, 1), (2, 4), (3, 0)):
        inside = torch.zeros(cols, dtype=torch.bool)
        at = {1: 200, 2: cols - 1, 3: 5}[r]
        inside[128 * group:128 * (group + 1)] = True
        # The group's scale is NaN, and so are all its codes.
        assert torch.isnan(q[r, at]) and torch.isnan(q[r, inside]).all() and torch.isnan(s[r, group])
        assert not q[r, ~inside].any()
        assert torch.equal(s[r, torch.arange(5) != group], torch.ones(4))


# Rows whose squares leave FP32, upwards and (with eps 0, which does not cover them) downwards.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [300, 4096, 12288, 32776, 65536])
@pytest.mark.parametrize("magnitude,eps", [(3e38, 1e-6), (1e30, 0.0), (1e19, 1e-6), (1e18, 1e-6), (1e-14, 0.0), (1e-16, 0.0),
                                           (1e-16, 1e-32), (1e-22, 1e-33), (1e-30, 0.0), (1e-37, 0.0)])
def test_norm_squares_outside_fp32(cuda_device, dtype, cols, magnitude, eps):
    x = _x(3, cols, torch.float32, seed=8)
    x = (x / x.abs().max() * magnitude).to(dtype)
    x[1, cols // 2:] = 0
    x[1, -1] = magnitude / 1024
    x[2] = _x(1, cols, dtype, seed=9)[0]  # an ordinary row beside them
    w = torch.linspace(0.5, 2, cols)
    assert torch.isfinite(x).all()
    h, q, s = _norm(x, w, cuda_device, store=True, eps=eps)
    _norm_check(x, None, w, eps, h, q, s)


def test_norm_least_numbers(cuda_device):
    """Rows of the types' least numbers: 1 / rms lies outside FP32, the result does not."""
    for dtype, least in ((torch.bfloat16, 2.0 ** -133), (torch.float32, 2.0 ** -149), (torch.float16, 2.0 ** -24)):
        x = torch.full((2, 384), least, dtype=dtype)
        x[1, 1::2] = 0
        _, q, s = _norm(x, torch.ones(384), cuda_device, store=False, eps=0.0)
        _norm_check(x, None, torch.ones(384), 0.0, None, q, s)
        assert (q[0] == 448).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [640, 637])
def test_norm_groups_below_the_scales_range(cuda_device, dtype, cols):
    """Groups whose max|y| / 448 is 0 in FP32 beside ordinary ones: scale 1, codes 0. Weights below 2^-10 take BF16's
    least numbers there too. A group a little above has a subnormal scale and finite codes."""
    x = torch.zeros(4, cols, dtype=dtype)
    x[:, 512:] = _x(4, cols - 512, dtype, seed=6)
    w = torch.ones(cols)
    w[:512] = 2.0 ** -13
    _, q0, s0 = _norm(x, w, cuda_device, store=False)
    _norm_check(x, None, w, 1e-6, None, q0, s0)
    x[:, 3] = 2.0 ** -133  # y is about 2^-145, less than 448 * 2^-150
    x[1:, 129] = -2.0 ** -133
    x[2, 260], x[3, 300] = 2.0 ** -125, 2.0 ** -133
    _, q, s = _norm(x, w, cuda_device, store=False)
    assert torch.equal(q[:, 512:], q0[:, 512:]) and torch.equal(s[:, 4], s0[:, 4])  # their squares are 0
    assert torch.isfinite(q).all() and torch.isfinite(s).all()
    low = torch.ones(4, 512, dtype=torch.bool)
    low[2, 256:384] = False
    assert not q[:, :512][low].any()
    assert torch.equal(s[:, :2], torch.ones(4, 2)) and torch.equal(s[:, 3], torch.ones(4))
    assert s[2, 2] > 0 and s[2, 2] < 2.0 ** -126 and torch.equal(s[[0, 1, 3], 2], torch.ones(3))
    assert (q[2, 256:384] != 0).nonzero().flatten().tolist() == [4]


def test_norm_no_rows(cuda_device):
    x = torch.empty(0, 64, dtype=torch.bfloat16)
    h, q, s = _norm(x, torch.ones(64), cuda_device)
    assert h.shape == (0, 64) and q.shape == (0, 64) and s.shape == (0, 1)


def test_norm_rows_of_few_steps_are_exact(cuda_device):
    """One non-zero element a row: y = sqrt(cols) * sign * w, q = +-448."""
    x = torch.zeros(64, 64, dtype=torch.float16)
    x.fill_diagonal_(-3.0)
    _, q, s = _norm(x, torch.ones(64), cuda_device, store=False, eps=0.0)
    assert torch.equal(q, torch.eye(64) * -448)
    assert ((s.double() - 8 / 448).abs() <= 10 * U * 8 / 448).all()


# ------------------------------------------------------------------ 4-bit formats
def _operand(fmt, rows, k, dev, scale):
    if fmt == "mxfp4":
        return lowp.Mxfp4Operand.empty(rows, k, device=dev)
    return lowp.Nvfp4Operand.empty(rows, k, device=dev, tensor_scale=scale)


def _fp4(fmt, x, dev, scale=None, values=True, stream=None):
    op = _operand(fmt, *x.shape, dev, scale)
    op.data.fill_(0xAA)
    op.atoms.fill_(0xAA)
    xd = x.to(dev)
    v = torch.full_like(xd, float("nan")) if values else None
    plan = quantize.Fp4QuantPlan(xd, op, values=v, stream=stream)
    plan.run()
    plan.synchronize()
    plan.close()
    return op.to("cpu"), None if v is None else v.cpu()


def _fp4_reference(fmt, x, scale=None):
    if fmt == "mxfp4":
        packed, bits = lowp.mxfp4_quantize(x)
        return packed, bits, None, lowp.mxfp4_dequantize(packed, bits)
    packed, bits, g = lowp.nvfp4_quantize(x, scale)
    return packed, bits, g, lowp.nvfp4_dequantize(packed, bits, g)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,scale", [("mxfp4", None), ("nvfp4", None), ("nvfp4", 0.003)])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 64), (2, 96), (127, 160), (129, 32), (77, 4096), (300, 288), (5, 2880)])
def test_fp4_equals_definition(cuda_device, fmt, scale, dtype, rows, k):
    x = _x(rows, k, dtype, seed=rows)
    packed, bits, g, deq = _fp4_reference(fmt, x, scale)
    op, v = _fp4(fmt, x, cuda_device, scale)
    assert torch.equal(op.atoms, lowp.pack_scale_atoms(bits))  # padding rows and columns zero
    assert torch.equal(op.data, packed)
    assert torch.equal(v, deq.to(dtype))
    if fmt == "nvfp4" and scale is None:
        assert float(op.tensor_scale_out) == float(torch.tensor(g, dtype=torch.float32))
    assert torch.equal(op.dequantize(), deq)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_fp4_against_64_bits(cuda_device, fmt):
    """Each value is the nearest of the block's grid: half a step around a quotient whose divisor and
    result were rounded once each (nvfp4; mxfp4 divides exactly)."""
    x = _x(130, 512, torch.float32, seed=9)
    op, v = _fp4(fmt, x, cuda_device, values=True)
    block, bits = (32, None) if fmt == "mxfp4" else (16, None)
    width = 512 // block
    bits = lowp.unpack_scale_atoms(op.atoms, 130, width)
    unit = lowp.mxfp4_scale_values(bits).double() if fmt == "mxfp4" else \
        bits.view(torch.float8_e4m3fn).double() * float(op.tensor_scale_out)
    unit = unit.repeat_interleave(block, 1)
    y = (x.double() / unit).abs()
    # The block's scale may leave amax / scale above 6 by its own rounding (mxfp4: below 8); cut there.
    q = (v.double() / unit).abs()
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    slack = 0.0 if fmt == "mxfp4" else 4 * U
    ok = ((q - y).abs() <= step / 2 + slack * y) | ((y > 6) & ((q - 6).abs() <= slack * 6))
    assert ok.all()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("magnitude", [1e-42, 1e-36, 1e-20, 1e20, 1e37])
def test_fp4_range(cuda_device, fmt, magnitude):
    x = _x(40, 128, torch.float32, seed=11)
    x = x / x.abs().max() * magnitude
    x[3, :64] = 0
    x[4] = 0
    packed, bits, g, deq = _fp4_reference(fmt, x)
    op, v = _fp4(fmt, x, cuda_device)
    assert torch.equal(op.atoms, lowp.pack_scale_atoms(bits))
    assert torch.equal(op.data, packed) and torch.equal(v, deq)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_fp4_non_finite(cuda_device, fmt):
    x = _x(4, 96, torch.float32, seed=12)
    x[0, 3], x[1, 40], x[2, 95] = float("nan"), float("inf"), float("-inf")
    packed, bits, g, deq = _fp4_reference(fmt, x, 0.01)
    op, v = _fp4(fmt, x, cuda_device, scale=0.01 if fmt == "nvfp4" else None)
    assert torch.equal(op.atoms, lowp.pack_scale_atoms(bits))
    assert torch.equal(op.data, packed)
    assert torch.equal(torch.isnan(v), torch.isnan(deq)) and torch.equal(v.nan_to_num(), deq.nan_to_num())
    assert not torch.isnan(v[3]).any()


def test_fp4_borders(cuda_device):
    """Quotients on and one step beside every border of the grid."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    rows = []
    for scale in (1.0, 3.0, 0.7, 1.3e-5, 7.7e4):
        for direction in (0.0, 1e9, -1e9):
            m = mids * scale
            m = torch.nextafter(m, torch.full_like(m, direction)) if direction else m
            m[-1] = 6 * scale
            rows.append(torch.cat((m, -m)).repeat(4))
    x = torch.stack(rows)
    for fmt, scale in (("mxfp4", None), ("nvfp4", None), ("nvfp4", 1e-3), ("nvfp4", 0.37)):
        packed, bits, _, deq = _fp4_reference(fmt, x, scale)
        op, v = _fp4(fmt, x, cuda_device, scale)
        assert torch.equal(op.atoms, lowp.pack_scale_atoms(bits))
        assert torch.equal(op.data, packed) and torch.equal(v, deq)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_fp4_strides_and_in_place(cuda_device, fmt, shift):
    full = _x(20, 96 + 16, torch.bfloat16, seed=13).to(cuda_device)
    keep = full.clone()
    x = full[:, shift:shift + 96]
    packed, bits, _, deq = _fp4_reference(fmt, x.cpu(), 0.01)
    op = _operand(fmt, 20, 96, cuda_device, 0.01)
    plan = quantize.Fp4QuantPlan(x, op, values=x)
    plan.run()
    plan.synchronize()
    assert torch.equal(op.data.cpu(), packed) and torch.equal(op.atoms.cpu(), lowp.pack_scale_atoms(bits))
    assert torch.equal(x.cpu(), deq.to(torch.bfloat16))
    assert torch.equal(full[:, :shift], keep[:, :shift]) and torch.equal(full[:, shift + 96:], keep[:, shift + 96:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 4096), (1, 16384), (1, 32800), (3, 4096), (8, 512), (9, 512), (5, 2880)])
@pytest.mark.parametrize("shift", [0, 3])
def test_fp4_found_scale_of_few_rows(cuda_device, dtype, rows, k, shift):
    """The scale of a few rows, found with and without a launch of its own: the maximum in the last row's
    last block, no values, then values over x itself (no CTA may read x after another wrote it)."""
    full = torch.zeros(rows, k + 16, dtype=dtype, device=cuda_device)
    x = full[:, shift:shift + k]
    x.copy_(_x(rows, k, dtype, seed=rows + k).to(cuda_device))
    x[-1, -1] = -900.0
    packed, bits, g, deq = _fp4_reference("nvfp4", x.cpu())
    atoms = lowp.pack_scale_atoms(bits)
    for values in (None, x):
        op = lowp.Nvfp4Operand.empty(rows, k, device=cuda_device)
        plan = quantize.Fp4QuantPlan(x, op, values=values)
        plan.run()
        plan.synchronize()
        assert torch.equal(op.data.cpu(), packed) and torch.equal(op.atoms.cpu(), atoms)
        assert float(op.tensor_scale_out) == float(torch.tensor(g, dtype=torch.float32))
        plan.close()
    assert torch.equal(x.cpu(), deq.to(dtype))


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("fill", [0.0, float("nan"), float("inf"), 1e-40])
def test_fp4_found_scale_without_a_maximum(cuda_device, rows, fill):
    """Zero, NaN, an infinity and data below 2688 times the least FP32 number, the same for a few rows and many."""
    x = torch.zeros(rows, 512)
    x[rows // 2, 40] = fill
    packed, bits, g, _ = _fp4_reference("nvfp4", x)
    op, _ = _fp4("nvfp4", x, cuda_device, values=False)
    # inf / inf is a NaN whose sign IEEE 754 leaves open, 0x7f or 0xff in E4M3; the kernel writes 0x7f.
    assert torch.equal(op.data, packed) and torch.equal(op.atoms, lowp.pack_scale_atoms(bits & 0x7F))
    assert float(op.tensor_scale_out) == float(torch.tensor(g, dtype=torch.float32))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_fp4_no_rows(cuda_device, fmt):
    op, v = _fp4(fmt, torch.empty(0, 64, dtype=torch.bfloat16), cuda_device)
    assert op.data.shape == (0, 32) and v.shape == (0, 64)


def test_division_is_exact_for_many_quotients(cuda_device):
    """The quotient by residual against torch's division: NVFP4 with tensor scale 1 and block maxima that
    make the block scale 1, so values are q(x / g) for many g and random x; compared through the codes."""
    g = torch.Generator().manual_seed(21)
    x = torch.rand(4096, 512, generator=g) * 6
    scale = torch.exp(3 * torch.randn(8, generator=g)).tolist()
    for s in scale:
        packed, bits, _, _ = _fp4_reference("nvfp4", x, s)
        op, _ = _fp4("nvfp4", x, cuda_device, s, values=False)
        assert torch.equal(op.atoms, lowp.pack_scale_atoms(bits)) and torch.equal(op.data, packed)


# ------------------------------------------------------------------ streams and graphs
def test_other_stream_and_graph(cuda_device):
    """Plans on a stream of their own, captured and replayed on new data."""
    stream = torch.cuda.Stream(device=cuda_device)
    x = _x(17, 320, torch.bfloat16).to(cuda_device)
    w = torch.ones(320, device=cuda_device)
    fp8 = lowp.Fp8GroupOperand.empty(17, 320, device=cuda_device)
    nv = lowp.Nvfp4Operand.empty(17, 320, device=cuda_device)
    stream.wait_stream(torch.cuda.current_stream(cuda_device))
    plans = [quantize.RmsNormFp8Plan(x, w, fp8, stream=stream), quantize.Fp4QuantPlan(x, nv, stream=stream)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for p in plans:
            p.run()
    for seed in (30, 31):
        new = _x(17, 320, torch.bfloat16, seed=seed, scale=1 + seed)
        x.copy_(new.to(cuda_device))
        graph.replay()
        torch.cuda.synchronize(cuda_device)
        _norm_check(new, None, w.cpu(), 1e-6, None, fp8.values.float().cpu(), fp8.scales.cpu())
        packed, bits, g, _ = _fp4_reference("nvfp4", new)
        assert torch.equal(nv.data.cpu(), packed) and torch.equal(nv.atoms.cpu(), lowp.pack_scale_atoms(bits))
        assert float(nv.tensor_scale_out) == float(torch.tensor(g, dtype=torch.float32))


def test_plan_made_while_the_default_stream_is_busy(cuda_device):
    """The counter of the maximum's launch is zero before a plan on another stream first runs, whatever the
    memory held and whatever is queued on the default stream (a busy wait of about 10 ms)."""
    big = _x(1184, 64, torch.bfloat16).to(cuda_device)
    plan = quantize.Fp4QuantPlan(big, lowp.Nvfp4Operand.empty(1184, 64, device=cuda_device))
    plan.run()
    plan.synchronize()
    plan.close()  # its maxima stay behind in the memory that the next plan gets
    stream = torch.cuda.Stream(device=cuda_device)
    x = _x(20, 64, torch.bfloat16, seed=3)
    xd, op = x.to(cuda_device), lowp.Nvfp4Operand.empty(20, 64, device=cuda_device)
    torch.cuda.synchronize(cuda_device)
    torch.cuda._sleep(20_000_000)
    plan = quantize.Fp4QuantPlan(xd, op, stream=stream)
    plan.run()
    plan.synchronize()
    packed, bits, g, _ = _fp4_reference("nvfp4", x)
    assert torch.equal(op.data.cpu(), packed) and torch.equal(op.atoms.cpu(), lowp.pack_scale_atoms(bits))
    assert float(op.tensor_scale_out) == float(torch.tensor(g, dtype=torch.float32))


def test_row_strides_past_32_bits(cuda_device):
    """Rows 2^31 elements apart."""
    ld, cols = 1 << 31, 288
    big = torch.empty(ld + cols, dtype=torch.bfloat16, device=cuda_device)
    x = big.as_strided((2, cols), (ld, 1))
    src = _x(2, cols, torch.bfloat16, seed=40)
    x.copy_(src.to(cuda_device))
    w = torch.ones(cols)
    out = lowp.Fp8GroupOperand.empty(2, cols, device=cuda_device)
    plan = quantize.RmsNormFp8Plan(x, w.to(cuda_device), out, residual=x, residual_out=x)  # h = 2 x, in place
    plan.run()
    plan.synchronize()
    _norm_check(src, src, w, 1e-6, x.cpu(), out.values.float().cpu(), out.scales.cpu())
    for fmt in ("mxfp4", "nvfp4"):
        x.copy_(src.to(cuda_device))
        packed, bits, _, deq = _fp4_reference(fmt, src)
        op = _operand(fmt, 2, cols, cuda_device, None)
        plan = quantize.Fp4QuantPlan(x, op, values=x)
        plan.run()
        plan.synchronize()
        assert torch.equal(op.data.cpu(), packed) and torch.equal(x.cpu(), deq.to(torch.bfloat16))


def test_tensors_past_32_bits(cuda_device):
    """More than 2^32 elements of x: the last rows against the first."""
    rows, cols = 524289, 8192
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device=cuda_device)
    x.view(-1)[: 128 * cols].copy_(_x(128, cols, torch.bfloat16, seed=41).to(cuda_device).view(-1))
    x[128:] = 0
    x[-1].copy_(x[77])
    x[rows // 2 + 1].copy_(x[3])
    op = lowp.Mxfp4Operand.empty(rows, cols, device=cuda_device)
    plan = quantize.Fp4QuantPlan(x, op)
    plan.run()
    plan.synchronize()
    bits = lowp.unpack_scale_atoms(op.atoms[-1:], 1, cols // 32)
    first = lowp.unpack_scale_atoms(op.atoms[:1], 128, cols // 32)
    assert torch.equal(op.data[-1], op.data[77]) and torch.equal(bits[0], first[77])
    assert torch.equal(op.data[rows // 2 + 1], op.data[3]) and not op.data[rows // 2 + 2].any()
    out = lowp.Fp8GroupOperand.empty(rows, cols, device=cuda_device)
    plan = quantize.RmsNormFp8Plan(x, torch.ones(cols, device=cuda_device), out)
    plan.run()
    plan.synchronize()
    assert torch.equal(out.data[-1], out.data[77]) and torch.equal(out.scales[-1], out.scales[77])
    assert torch.equal(out.data[rows // 2 + 1], out.data[3]) and not out.data[rows // 2 + 2].any()


def test_graphs_of_one_plan(cuda_device):
    """Two graphs captured from one plan, replayed in turn; then a closed plan refuses."""
    stream = torch.cuda.Stream(device=cuda_device)
    x = torch.empty(200, 512, dtype=torch.float16, device=cuda_device)
    op = lowp.Nvfp4Operand.empty(200, 512, device=cuda_device)
    plan = quantize.Fp4QuantPlan(x, op, stream=stream)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for n, graph in enumerate(graphs):
        with torch.cuda.graph(graph, stream=stream):
            plan.run(n + 1)
    for i, scale in enumerate((1.0, 5.0, 0.01, 300.0)):
        new = _x(200, 512, torch.float16, seed=50 + i) * scale
        x.copy_(new.to(cuda_device))
        torch.cuda.synchronize(cuda_device)
        with torch.cuda.stream(stream):
            graphs[i % 2].replay()
        stream.synchronize()
        packed, bits, g, _ = _fp4_reference("nvfp4", new)
        assert torch.equal(op.data.cpu(), packed) and torch.equal(op.atoms.cpu(), lowp.pack_scale_atoms(bits))
    del graphs
    plan.close()
    from gb300_microbench_b200 import _native as nat
    with pytest.raises(nat.NativeCallError):
        plan.run()
