"""CPU checks of the quantised linear layer: the MXFP4 and FP8 group formats in
torch against their definitions in 64 bits, the operands, and every refusal
that is decided before a GPU is touched."""
import ctypes

import numpy as np
import pytest
import torch

from gb300_microbench_b200 import _native as nat
from gb300_microbench_b200 import build as buildmod
from gb300_microbench_b200 import lowp, quantize
from oracle import lowp as olp


@pytest.fixture(scope="module")
def lib():
    buildmod.build()
    return nat.bench_lib()


def _mxfp4_oracle(x: np.ndarray):
    """Codes' values and scales by the definition, in 64 bits, one block at a time."""
    r, k = x.shape
    values, scales = np.zeros((r, k)), np.zeros((r, k // 32))
    grid = olp.E2M1_VALUES
    for i in range(r):
        for b in range(k // 32):
            v = x[i, 32 * b:32 * b + 32].astype(np.float64)
            top = np.abs(v).max()
            e = -127 if top == 0 else max(int(np.frexp(top)[1]) - 3, -127)
            scales[i, b] = 2.0 ** e
            for j, y in enumerate(np.minimum(np.abs(v) / 2.0 ** e, 6.0)):
                d = np.abs(grid - y)
                best = np.flatnonzero(d == d.min())
                q = best[0] if len(best) == 1 or best[0] % 2 == 0 else best[1]
                values[i, 32 * b + j] = np.copysign(grid[q], v[j]) * 2.0 ** e
    return values, scales


@pytest.mark.parametrize("magnitude", [1e-40, 1e-30, 1.0, 1e30, 3e38])
def test_mxfp4_matches_definition(magnitude):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 96, generator=g)
    x[0, :32] = 0
    x[1, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    x[1, 8:32] = 0
    x = (x / x.abs().max()) * magnitude
    values, scales = _mxfp4_oracle(x.numpy())
    packed, bits = lowp.mxfp4_quantize(x)
    np.testing.assert_array_equal(lowp.mxfp4_scale_values(bits).double().numpy(), scales)
    np.testing.assert_array_equal(lowp.mxfp4_dequantize(packed, bits).double().numpy(), values)


def test_mxfp4_non_finite_blocks_are_nan():
    x = torch.ones(3, 64)
    x[0, 5], x[1, 40], x[2, 0] = float("nan"), float("inf"), float("-inf")
    packed, bits = lowp.mxfp4_quantize(x)
    assert bits.tolist() == [[255, 125], [125, 255], [255, 125]]
    v = lowp.mxfp4_dequantize(packed, bits)
    assert torch.isnan(v).sum() == 3 * 32
    assert torch.equal(v[0, 32:], torch.ones(32))


def test_nvfp4_given_scale_is_used():
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(0))
    _, s1, g1 = lowp.nvfp4_quantize(x)
    _, s2, g2 = lowp.nvfp4_quantize(x, tensor_scale=g1)
    assert g2 == g1 and torch.equal(s1, s2)
    _, s3, g3 = lowp.nvfp4_quantize(x, tensor_scale=g1 / 1024)
    assert g3 == g1 / 1024 and int(s3.max()) == 0x7E  # saturated at 448


def test_fp8_group_format():
    x = torch.randn(3, 300, generator=torch.Generator().manual_seed(1))
    x[1, 128:256] = 0
    q, s = lowp.fp8_group_quantize(x)
    assert s.shape == (3, 3) and s[1, 1] == 1
    amax = torch.nn.functional.pad(x, (0, 84)).view(3, 3, 128).abs().amax(2).double() / 448
    np.testing.assert_allclose(s.double().numpy(), torch.where(amax > 0, amax, 1.0).numpy(), rtol=2.0 ** -24)
    got = lowp.fp8_group_dequantize(q, s).double()
    # Half a step of E4M3 (2^-4 relative, 2^-10 absolute below the normal numbers), the quotient
    # and the dequantised product each rounded once in FP32.
    spread = s.double().repeat_interleave(128, 1)[:, :300]
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, spread * 2.0 ** -10) * (1 + 2.0 ** -20)
    assert ((got - x.double()).abs() <= bound).all()


def test_fp8_groups_below_the_scales_range():
    """amax / 448 below half the least FP32 number (1.4e-45) is 0: such a group has scale 1 and codes 0. From there
    on the scale is a subnormal number and no code is NaN."""
    x = torch.zeros(3, 384)
    x[0, 0], x[0, 130], x[0, 300] = 1e-43, -3e-43, 2.0 ** -149
    x[1, 7], x[1, 129], x[1, 257] = 1e-42, -5e-41, 1.0
    q, s = lowp.fp8_group_quantize(x)
    v = q.view(torch.float8_e4m3fn).float()
    assert torch.equal(s[0], torch.ones(3)) and torch.equal(s[2], torch.ones(3))
    assert not v[0].any() and not v[2].any()
    assert (s[1] > 0).all() and torch.isfinite(v).all()
    assert (v[1] != 0).nonzero().flatten().tolist() == [7, 129, 257]
    # The scale is off by half of 2^-149 at most, or 448 times that once multiplied back; the code by half a step.
    got = lowp.fp8_group_dequantize(q, s).double()
    assert ((got - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + 448 * 2.0 ** -150 + 2.0 ** -150).all()


def test_fp8_blocks_below_the_scales_range():
    """The weights' 128 x 128 blocks likewise: scale 1 and codes 0 where amax / 448 is 0 in FP32."""
    x = torch.zeros(200, 256)
    x[5, 3], x[9, 4] = 1e-43, -3e-43
    x[130, 7], x[131, 200] = 1e-42, 2.0
    q, s = lowp.fp8_block_quantize(x)
    v = q.view(torch.float8_e4m3fn).float()
    assert torch.isfinite(v).all() and (s > 0).all()
    assert torch.equal(s[0], torch.ones(2)) and not v[:128].any()
    assert (v != 0).nonzero().tolist() == [[130, 7], [131, 200]]
    got = lowp.fp8_block_dequantize(q, s).double()
    assert ((got - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + 448 * 2.0 ** -150 + 2.0 ** -150).all()


@pytest.mark.parametrize("make", [lowp.Nvfp4Operand, lowp.Mxfp4Operand, lowp.Fp8GroupOperand, lowp.Fp8BlockOperand])
def test_operands_of_no_rows(make):
    op = make(torch.empty(0, 256))
    assert (op.rows, op.k) == (0, 256) and op.data.shape[0] == 0
    assert op.to("cpu").dequantize().shape == (0, 256)


@pytest.mark.parametrize("rows,width", [(1, 1), (130, 5), (128, 8), (257, 90)])
def test_scale_atoms_round_trip(rows, width):
    s = torch.randint(0, 256, (rows, width), dtype=torch.uint8, generator=torch.Generator().manual_seed(rows))
    atoms = lowp.pack_scale_atoms(s)
    assert atoms.shape == (-(-rows // 128), -(-width // 4), 512)
    assert torch.equal(lowp.unpack_scale_atoms(atoms, rows, width), s)


def test_operands_refuse_what_does_not_fit():
    u8 = torch.uint8
    with pytest.raises(ValueError):
        lowp.Mxfp4Operand.from_parts(torch.zeros(4, 32, dtype=u8), torch.zeros(4, 3, dtype=u8))
    with pytest.raises(ValueError):
        lowp.Mxfp4Operand.from_parts(torch.zeros(4, 24, dtype=u8), torch.zeros(4, 1, dtype=u8))
    with pytest.raises(ValueError):
        lowp.Mxfp4Operand.empty(4, 48, device="cpu")
    with pytest.raises(ValueError):
        lowp.Nvfp4Operand.empty(-1, 64, device="cpu")
    with pytest.raises(ValueError):
        lowp.Fp8GroupOperand.from_parts(torch.zeros(4, 128, dtype=u8), torch.ones(4, 2))
    with pytest.raises(ValueError):
        lowp.Fp8GroupOperand.from_parts(torch.zeros(4, 128), torch.ones(4, 1))
    op = lowp.Fp8GroupOperand.empty(5, 300, device="cpu")
    assert op.scales.shape == (5, 3) and op.scales.stride() == (1, 5) and op.values.dtype == torch.float8_e4m3fn


def test_values_follow_the_data():
    """``values`` is of the tensor that is ``data`` now, also where a new one begins at the old one's address."""
    op = lowp.Fp8GroupOperand.empty(5, 130, device="cpu")
    op.data.fill_(0x38)
    assert op.values.shape == (5, 130) and (op.values.float() == 1).all()
    first = op.data
    first.fill_(0x40)
    assert (op.values.float() == 2).all()
    op.data = first[:2]
    assert op.values.shape == (2, 130) and op.values.data_ptr() == first.data_ptr()
    op.data = torch.full((3, 130), 0x38, dtype=torch.uint8)
    assert op.values.shape == (3, 130) and (op.values.float() == 1).all()
    op.data = op.data.view(torch.float8_e4m3fn)
    assert op.values.shape == (3, 130) and (op.values.float() == 1).all()
    op.rows, op.scales = 3, torch.ones(2, 3).t()
    assert torch.equal(op.to("cpu").values.view(torch.uint8), op.data.view(torch.uint8))


def test_plans_refuse_before_any_launch():
    """Shapes, dtypes and strides are refused in Python, CPU tensors among them."""
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    fp8 = lowp.Fp8GroupOperand.empty(4, 64, device="cpu")
    w = torch.ones(64, dtype=torch.bfloat16)
    cases = [
        lambda: quantize.RmsNormFp8Plan(x, w, fp8),                                        # not on a GPU
        lambda: quantize.RmsNormFp8Plan(x[:, :32], w, fp8),
        lambda: quantize.RmsNormFp8Plan(x.double(), w, fp8),
        lambda: quantize.RmsNormFp8Plan(x, w.half(), fp8),
        lambda: quantize.RmsNormFp8Plan(x, w[:32], fp8),
        lambda: quantize.RmsNormFp8Plan(x, w, fp8, residual=x.float()),
        lambda: quantize.RmsNormFp8Plan(x, w, fp8, eps=-1.0),
        lambda: quantize.RmsNormFp8Plan(x, w, fp8, eps=float("nan")),
        lambda: quantize.RmsNormFp8Plan(x.t().contiguous().t(), w, fp8),
        lambda: quantize.RmsNormFp8Plan(x[:1].expand(4, 64), w, fp8),                       # rows overlap
        lambda: quantize.RmsNormFp8Plan(x, w, lowp.Mxfp4Operand.empty(4, 64, device="cpu")),
        lambda: quantize.Fp4QuantPlan(x, lowp.Mxfp4Operand.empty(4, 64, device="cpu")),     # not on a GPU
        lambda: quantize.Fp4QuantPlan(x, fp8),
        lambda: quantize.Fp4QuantPlan(x, lowp.Mxfp4Operand.empty(5, 64, device="cpu")),
        lambda: quantize.Fp4QuantPlan(x, lowp.Nvfp4Operand(torch.ones(4, 64))),
        lambda: quantize.Fp4QuantPlan(x, lowp.Nvfp4Operand.empty(4, 64, device="cpu", tensor_scale=0.0)),
        lambda: quantize.Fp4QuantPlan(x, lowp.Mxfp4Operand.empty(4, 64, device="cpu"), values=x.float()),
    ]
    a4, b4 = lowp.Mxfp4Operand.empty(4, 64, device="cpu"), lowp.Mxfp4Operand.empty(8, 64, device="cpu")
    d = torch.zeros(4, 8, dtype=torch.bfloat16)
    cases += [
        lambda: lowp.LowpLinearPlan(a4, b4, d),                                             # not on a GPU
        lambda: lowp.LowpLinearPlan(a4, b4, d[:, :7]),
        lambda: lowp.LowpLinearPlan(a4, b4, d.double()),
        lambda: lowp.LowpLinearPlan(a4, b4, torch.zeros(8, 4, dtype=torch.bfloat16).t()),
        lambda: lowp.LowpLinearPlan(a4, lowp.Nvfp4Operand(torch.ones(8, 64)), d),
        lambda: lowp.LowpLinearPlan(a4, lowp.Mxfp4Operand.empty(8, 96, device="cpu"), d),
        lambda: lowp.LowpLinearPlan(x, b4, d),
        lambda: lowp.LowpLinearPlan(lowp.Nvfp4Operand(torch.ones(4, 16)), lowp.Nvfp4Operand(torch.ones(8, 16)), d),
        lambda: lowp.LowpLinearPlan(fp8, b4, d),
    ]
    for i, case in enumerate(cases):
        with pytest.raises(ValueError):
            case()
            pytest.fail(f"case {i} was accepted")


def test_plans_refuse_buffers_of_other_types():
    """Large enough in bytes, but not the bytes that the kernels read."""
    x, d = torch.zeros(4, 128, dtype=torch.bfloat16), torch.zeros(4, 256, dtype=torch.bfloat16)
    a8, b8 = lowp.Fp8GroupOperand.empty(4, 128, device="cpu"), lowp.Fp8BlockOperand(torch.ones(256, 128))
    a4, b4 = lowp.Mxfp4Operand.empty(4, 128, device="cpu"), lowp.Mxfp4Operand(torch.ones(256, 128))
    floats = lowp.Fp8BlockOperand.from_parts(torch.ones(256, 128), torch.ones(2, 1))
    doubles = lowp.Fp8BlockOperand(torch.ones(256, 128))
    doubles.scales = doubles.scales.double()
    words = lowp.Mxfp4Operand(torch.ones(256, 128))
    words.atoms = words.atoms.int()
    wide8, wide4 = lowp.Fp8GroupOperand.empty(4, 128, device="cpu"), lowp.Mxfp4Operand.empty(4, 128, device="cpu")
    wide8.data, wide4.data = wide8.data.int(), wide4.data.int()
    for make, match in ((lambda: lowp.LowpLinearPlan(a8, floats, d), "w data"),
                        (lambda: lowp.LowpLinearPlan(a8, doubles, d), "w scales"),
                        (lambda: lowp.LowpLinearPlan(a4, words, d), "w atoms"),
                        (lambda: lowp.LowpLinearPlan(wide4, b4, d), "x data"),
                        (lambda: quantize.RmsNormFp8Plan(x, torch.ones(128), wide8), "out.data"),
                        (lambda: quantize.Fp4QuantPlan(x, wide4), "out.data"),
                        (lambda: lowp.LowpLinearPlan(a8, b8, d), "CUDA"),
                        (lambda: lowp.LowpLinearPlan(a4, b4, d), "CUDA")):
        with pytest.raises(ValueError, match=match):
            make()


def test_native_refusals(lib):
    """The C entries refuse bad arguments before they look for a device."""
    plan = ctypes.c_void_p()
    p = 1 << 20  # any aligned address: never read

    def linear(kind=nat.BB_LOWP_MXFP4, m=4, n=8, k=64, a=p, b=p, sfa=p, sfa_ld=4, sfb=p, d=p, dt=nat.BB_DTYPE_BF16,
               ldd=8, dev=None):
        return lib.bb_linear_plan_create(kind, m, n, k, a, b, sfa, sfa_ld, sfb, 1.0, dev, 1.0, None, d, dt, ldd, None,
                                         ctypes.byref(plan), None)

    for bad in (dict(kind=nat.BB_LOWP_FP8_BLOCK128), dict(kind=9), dict(m=-1), dict(n=0), dict(k=0), dict(k=48),
                dict(kind=nat.BB_LOWP_FP8_GROUP128, k=24), dict(kind=nat.BB_LOWP_FP8_GROUP128, sfa_ld=3), dict(a=None),
                dict(b=None), dict(sfa=None), dict(sfb=None), dict(d=None), dict(dt=7), dict(ldd=7), dict(a=p + 8),
                dict(b=p + 4), dict(sfa=p + 4), dict(d=p + 1), dict(dev=p + 2), dict(m=1 << 25), dict(n=1 << 25),
                dict(m=1 << 24, n=1 << 24, ldd=1 << 24)):
        assert linear(**bad) == nat.BB_ERR_ARGUMENT, bad
        assert lib.bb_last_error(), bad
        assert not plan.value
    assert lib.bb_linear_execute_n(None, 1) == nat.BB_ERR_ARGUMENT
    assert lib.bb_linear_synchronize(None) == nat.BB_ERR_ARGUMENT
    assert lib.bb_linear_launches(None) == -1 and lib.bb_linear_destroy(None) == nat.BB_OK

    def fp4(fmt=nat.BB_LOWP_NVFP4, rows=4, cols=64, x=p, dt=nat.BB_DTYPE_BF16, x_ld=64, data=p, sc=p, ts=1.0, out=None,
            v=None, v_ld=0):
        return lib.bb_fp4_quant_plan_create(fmt, rows, cols, x, dt, x_ld, data, sc, ts, out, v, v_ld, None,
                                            ctypes.byref(plan))

    for bad in (dict(fmt=nat.BB_LOWP_FP8_BLOCK128), dict(rows=-1), dict(cols=0), dict(cols=48), dict(x=None),
                dict(data=None), dict(sc=None), dict(dt=9), dict(x_ld=32), dict(ts=0.0), dict(ts=float("inf")),
                dict(ts=float("nan")), dict(ts=-1.0), dict(v=p, v_ld=32), dict(x=p + 1), dict(data=p + 8),
                dict(sc=p + 4), dict(out=p + 2), dict(rows=1 << 30, cols=1 << 24, x_ld=1 << 24)):
        assert fp4(**bad) == nat.BB_ERR_ARGUMENT, bad
        assert not plan.value

    def norm(rows=4, cols=64, x=p, dt=nat.BB_DTYPE_F16, x_ld=64, r=None, r_ld=0, ro=None, ro_ld=0, w=p,
             wdt=nat.BB_DTYPE_F32, eps=1e-6, q=p, q_ld=64, s=p, s_ld=4):
        return lib.bb_rmsnorm_fp8_plan_create(rows, cols, x, dt, x_ld, r, r_ld, ro, ro_ld, w, wdt, eps, q, q_ld, s, s_ld,
                                              None, ctypes.byref(plan))

    for bad in (dict(rows=-1), dict(cols=0), dict(cols=65537, x_ld=65537, q_ld=65537), dict(x=None), dict(w=None),
                dict(q=None), dict(s=None), dict(dt=0), dict(wdt=nat.BB_DTYPE_BF16), dict(eps=-1.0),
                dict(eps=float("nan")), dict(x_ld=63), dict(r=p, r_ld=63), dict(ro=p, ro_ld=8), dict(q_ld=32),
                dict(s_ld=3), dict(x=p + 1), dict(w=p + 2), dict(s=p + 2), dict(r=p + 1, r_ld=64)):
        assert norm(**bad) == nat.BB_ERR_ARGUMENT, bad
        assert not plan.value
    assert lib.bb_quant_execute_n(None, 1) == nat.BB_ERR_ARGUMENT
    assert lib.bb_quant_launches(None) == -1 and lib.bb_quant_destroy(None) == nat.BB_OK


def test_linear_scale_bytes(lib):
    f = lib.bb_linear_scale_bytes
    assert f(nat.BB_LOWP_NVFP4, 0, 300, 96) == 3 * 2 * 512
    assert f(nat.BB_LOWP_MXFP4, 1, 129, 160) == 2 * 2 * 512
    assert f(nat.BB_LOWP_FP8_GROUP128, 0, 5, 272) == 5 * 3 * 4
    assert f(nat.BB_LOWP_FP8_GROUP128, 1, 300, 272) == 3 * 3 * 4
    assert f(nat.BB_LOWP_MXFP4, 0, 4, 48) == -1 and f(nat.BB_LOWP_FP8_GROUP128, 0, 4, 24) == -1
    assert f(nat.BB_LOWP_FP8_BLOCK128, 0, 4, 128) == -1
