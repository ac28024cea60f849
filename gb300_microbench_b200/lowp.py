"""Low-precision operand formats of the block-scaled GEMMs (8192^3 FP8 128 x 128-block and NVFP4).

NVFP4: E2M1 values (two per byte, element 2i in the low nibble), one
UE4M3 scale per 16 consecutive K elements, and one FP32 scale per tensor:

    x ~= e2m1 * e4m3_block_scale * tensor_scale

with tensor_scale = amax(|x|) / (448 * 6) and block scale = amax(block) / 6 /
tensor_scale rounded to E4M3, values rounded to nearest (ties to even) on
the E2M1 grid {0, 0.5, 1, 1.5, 2, 3, 4, 6}.

MXFP4: E2M1 values with one E8M0 scale per 32 consecutive K elements,
scale = 2^(floor(log2 amax(block)) - 2), no tensor scale; a block that holds
a NaN or an infinity has the scale NaN.

FP8 block-scaled: E4M3 values with one FP32 scale per 128 x 128 block,
scale = amax(block) / 448. FP8 group-scaled (activations): one FP32 scale
per row and 128 consecutive K elements.

The kernels read the NVFP4 block scales in "scale atoms": for each group of
128 rows and each 64 K elements (4 scales per row), 512 bytes in which the
scale j of row r sits at byte (r % 32) * 16 + (r // 32) * 4 + j. One atom is
what one ``tcgen05.cp.32x128b.warpx4`` moves into TMEM for one K = 64 MMA.
MXFP4 block scales use the same atoms, each covering 128 K elements.

:class:`LowpGemmPlan` is the GEMM of two operands of aligned extents;
:class:`LowpLinearPlan` is a linear layer's product, for any number of rows
(one token upwards) and any output width. :mod:`.quantize` has the
quantisers as kernels; the functions here are their definitions in torch.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as nat

E2M1_GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3_MAX = 448.0
E2M1_MAX = 6.0


def _e2m1_codes(y: torch.Tensor) -> torch.Tensor:
    """Round |y| <= 6 to the E2M1 grid (nearest, ties to the even code) and
    return 4-bit codes (sign in bit 3)."""
    a = y.abs().clamp(max=E2M1_MAX)
    grid = E2M1_GRID.to(y.device)
    # Midpoints between grid points; ties go to the even code.
    mids = (grid[1:] + grid[:-1]) / 2
    idx = torch.bucketize(a, mids, right=False)  # a == mid -> lower index
    tie = (idx < 7) & (a == mids[idx.clamp(max=6)])
    idx = torch.where(tie & (idx % 2 == 1), idx + 1, idx)
    sign = (y < 0) & (idx > 0)
    return (idx | (sign.to(idx.dtype) << 3)).to(torch.uint8)


def e2m1_decode(codes: torch.Tensor) -> torch.Tensor:
    grid = E2M1_GRID.to(codes.device)
    mag = grid[(codes & 7).long()]
    return torch.where((codes & 8) != 0, -mag, mag)


def nvfp4_quantize(x: torch.Tensor, tensor_scale: float | None = None) -> tuple[torch.Tensor, torch.Tensor, float]:
    """x (R, K) float32, K % 16 == 0 -> (packed (R, K/2) uint8,
    block scales (R, K/16) uint8 E4M3 bits, tensor scale float). The tensor
    scale is found from x unless one is given (a calibrated one)."""
    if x.dim() != 2 or x.shape[1] % 16:
        raise ValueError("x must be (R, K) with K a multiple of 16")
    x = x.float()
    r, k = x.shape
    if tensor_scale is None:
        amax = float(x.abs().max()) if x.numel() else 0.0
        gscale = amax / (E4M3_MAX * E2M1_MAX) if amax > 0 else 1.0
        if torch.tensor(gscale, dtype=torch.float32) == 0:  # below FP32: everything rounds to zero
            gscale = 1.0
    else:
        gscale = float(tensor_scale)
    blocks = x.view(r, k // 16, 16)
    bs = (blocks.abs().amax(dim=2) / E2M1_MAX / gscale).clamp(max=E4M3_MAX)
    bs8 = bs.to(torch.float8_e4m3fn)
    bsf = bs8.float()
    denom = (bsf * gscale).unsqueeze(2)
    y = torch.where(denom > 0, blocks / torch.where(denom > 0, denom, torch.ones_like(denom)),
                    torch.zeros_like(blocks))
    codes = _e2m1_codes(y).view(r, k)
    packed = (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous()
    return packed, bs8.view(torch.uint8).contiguous(), gscale


def nvfp4_dequantize(packed: torch.Tensor, scales: torch.Tensor, gscale: float) -> torch.Tensor:
    r, kh = packed.shape
    codes = torch.empty(r, kh * 2, dtype=torch.uint8, device=packed.device)
    codes[:, 0::2] = packed & 0xF
    codes[:, 1::2] = packed >> 4
    vals = e2m1_decode(codes)
    s = scales.view(torch.float8_e4m3fn).float().repeat_interleave(16, dim=1)
    return vals * s * gscale


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x (R, K) float32, K % 32 == 0 -> (packed (R, K/2) uint8, block scales
    (R, K/32) uint8 E8M0 bits)."""
    if x.dim() != 2 or x.shape[1] % 32:
        raise ValueError("x must be (R, K) with K a multiple of 32")
    x = x.float()
    r, k = x.shape
    blocks = x.view(r, k // 32, 32)
    amax = blocks.abs().amax(dim=2)
    # floor(log2 amax) - 2 + 127: amax's biased exponent less 2, not below 0.
    e = (amax.view(torch.int32) >> 23) & 0xFF
    bits = torch.where(e == 255, 255, (e - 2).clamp(min=0)).to(torch.uint8)
    y = blocks * mxfp4_scale_values(254 - bits.clamp(max=253)).unsqueeze(2)  # 1 / scale, exactly
    y = torch.where((bits == 255).unsqueeze(2), torch.zeros_like(y), y)
    codes = _e2m1_codes(y).view(r, k)
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).contiguous(), bits


def mxfp4_scale_values(bits: torch.Tensor) -> torch.Tensor:
    """E8M0 bytes -> FP32: 2^(byte - 127), NaN for 255."""
    b = bits.to(torch.int32)
    f = torch.where(b == 0, 1 << 22, b << 23)  # 2^-127 lies below the normal numbers
    return torch.where(b == 255, 0x7FC00000, f).to(torch.int32).view(torch.float32)


def mxfp4_dequantize(packed: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    r, kh = packed.shape
    codes = torch.stack((packed & 0xF, packed >> 4), dim=2).view(r, kh * 2)
    return e2m1_decode(codes) * mxfp4_scale_values(scales).repeat_interleave(32, dim=1)


def pack_scale_atoms(scales: torch.Tensor) -> torch.Tensor:
    """(R, K/16) scale bytes -> (ceil(R/128), ceil(K/64), 512) atoms (rows and
    K padded with zero scales)."""
    r, ks = scales.shape
    rb = -(-r // 128)
    kg = -(-ks // 4)
    padded = torch.zeros(rb * 128, kg * 4, dtype=torch.uint8, device=scales.device)
    padded[:r, :ks] = scales
    # [rb][r32 = row // 32 within block][r % 32][kg][j]
    t = padded.view(rb, 4, 32, kg, 4)
    # atom byte = (r % 32) * 16 + (r // 32) * 4 + j  ->  order [rb][kg][r%32][r//32][j]
    return t.permute(0, 3, 2, 1, 4).contiguous().view(rb, kg, 512)


def unpack_scale_atoms(atoms: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    """The inverse of :func:`pack_scale_atoms`: (rows, width) scale bytes."""
    rb, kg, _ = atoms.shape
    t = atoms.view(rb, kg, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rb * 128, kg * 4)
    return t[:rows, :width].contiguous()


def _extents(rows: int, k: int, step: int) -> tuple[int, int]:
    rows, k = int(rows), int(k)
    if rows < 0 or k <= 0 or k % step:
        raise ValueError(f"rows must not be negative and K positive{f' and a multiple of {step}' if step > 1 else ''}: "
                         f"got {rows} x {k}")
    return rows, k


def fp8_block_quantize(x: torch.Tensor, block: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """x (R, K) -> (E4M3 bits (R, K) uint8, FP32 scales (ceil(R/128), ceil(K/128)))
    with scale = amax(block) / 448, 1 where that is 0 in FP32 or NaN."""
    x = x.float()
    r, k = x.shape
    rb, kb = -(-r // block), -(-k // block)
    pad = torch.zeros(rb * block, kb * block, device=x.device)
    pad[:r, :k] = x
    blocks = pad.view(rb, block, kb, block)
    amax = blocks.abs().amax(dim=(1, 3))
    scale = amax / E4M3_MAX
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = (blocks / scale[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(rb * block, kb * block)[:r, :k].contiguous().view(torch.uint8), scale.contiguous()


def fp8_block_dequantize(q: torch.Tensor, scale: torch.Tensor, block: int = 128) -> torch.Tensor:
    v = q.view(torch.float8_e4m3fn).float()
    s = scale.repeat_interleave(block, 0).repeat_interleave(block, 1)[: v.shape[0], : v.shape[1]]
    return v * s


def fp8_group_quantize(x: torch.Tensor, group: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """x (R, K) -> (E4M3 bits (R, K) uint8, FP32 scales (R, ceil(K/128)))
    with scale = amax(group) / 448, 1 where that is 0 in FP32."""
    x = x.float()
    r, k = x.shape
    kb = -(-k // group)
    blocks = torch.nn.functional.pad(x, (0, kb * group - k)).view(r, kb, group)
    amax = blocks.abs().amax(dim=2)
    scale = amax / torch.full_like(amax, E4M3_MAX)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    q = (blocks / scale[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(r, kb * group)[:, :k].contiguous().view(torch.uint8), scale


def fp8_group_dequantize(q: torch.Tensor, scale: torch.Tensor, group: int = 128) -> torch.Tensor:
    v = q.view(torch.float8_e4m3fn).float()
    return v * scale.repeat_interleave(group, 1)[:, : v.shape[1]]


# ------------------------------------------------------------------ operands
class Nvfp4Operand:
    """A quantised NVFP4 operand: packed E2M1 (R, K/2) bytes, scale atoms,
    per-tensor FP32 scale.

    One made by :meth:`empty` is filled by :class:`.quantize.Fp4QuantPlan`;
    it keeps its scales as atoms only (``scales`` is None), and where its
    tensor scale is found from the data that is the device tensor
    ``tensor_scale_out`` (1,) and ``tensor_scale`` is None."""

    tensor_scale_out: torch.Tensor | None = None

    def __init__(self, x: torch.Tensor):
        self.rows, self.k = x.shape
        packed, scales, self.tensor_scale = nvfp4_quantize(x)
        self.data = packed
        self.scales = scales
        self.atoms = pack_scale_atoms(scales)

    @classmethod
    def from_parts(cls, data: torch.Tensor, scales: torch.Tensor, tensor_scale: float) -> "Nvfp4Operand":
        """An operand from already-encoded parts: packed E2M1 (R, K/2) bytes
        and E4M3 scale bytes (R, K/16)."""
        op = cls.__new__(cls)
        op.rows, op.k = data.shape[0], data.shape[1] * 2
        op.data, op.scales, op.tensor_scale = data.contiguous(), scales.contiguous(), float(tensor_scale)
        op.atoms = pack_scale_atoms(op.scales)
        return op

    @classmethod
    def empty(cls, rows: int, k: int, device: str | torch.device = "cuda",
              tensor_scale: float | None = None) -> "Nvfp4Operand":
        """Buffers for a quantiser to fill, K a multiple of 32; ``tensor_scale``
        None: to be found from the data."""
        op = cls.__new__(cls)
        op.rows, op.k = _extents(rows, k, 32)
        op.data = torch.empty(rows, k // 2, dtype=torch.uint8, device=device)
        op.scales = None
        op.atoms = torch.empty(-(-rows // 128), -(-k // 64), 512, dtype=torch.uint8, device=device)
        op.tensor_scale = None if tensor_scale is None else float(tensor_scale)
        if tensor_scale is None:
            op.tensor_scale_out = torch.ones(1, dtype=torch.float32, device=device)
        return op

    def to(self, device) -> "Nvfp4Operand":
        if self.scales is None:
            op = Nvfp4Operand.__new__(Nvfp4Operand)
            op.rows, op.k, op.scales, op.tensor_scale = self.rows, self.k, None, self.tensor_scale
            op.data, op.atoms = self.data.to(device), self.atoms.to(device)
            if self.tensor_scale_out is not None:
                op.tensor_scale_out = self.tensor_scale_out.to(device)
            return op
        op = Nvfp4Operand.from_parts(self.data.to(device), self.scales.to(device), self.tensor_scale)
        return op

    def dequantize(self) -> torch.Tensor:
        scales = unpack_scale_atoms(self.atoms, self.rows, self.k // 16) if self.scales is None else self.scales
        gscale = self.tensor_scale_out if self.tensor_scale is None else self.tensor_scale
        return nvfp4_dequantize(self.data, scales, gscale)


class Mxfp4Operand:
    """A quantised MXFP4 operand: packed E2M1 (R, K/2) bytes and E8M0 scales
    (R, K/32) as scale atoms. One made by :meth:`empty` is filled by
    :class:`.quantize.Fp4QuantPlan`."""

    def __init__(self, x: torch.Tensor):
        self.rows, self.k = x.shape
        self.data, scales = mxfp4_quantize(x)
        self.atoms = pack_scale_atoms(scales)

    @classmethod
    def from_parts(cls, data: torch.Tensor, scales: torch.Tensor) -> "Mxfp4Operand":
        """An operand from already-encoded parts: packed E2M1 (R, K/2) bytes
        and E8M0 scale bytes (R, K/32)."""
        if data.dim() != 2 or data.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise ValueError("data and scales must be uint8, data (R, K/2)")
        op = cls.__new__(cls)
        op.rows, op.k = data.shape[0], data.shape[1] * 2
        if tuple(scales.shape) != (op.rows, op.k // 32) or op.k % 32:
            raise ValueError(f"scales {tuple(scales.shape)} do not fit data {tuple(data.shape)}: K must be a multiple "
                             "of 32 with one scale per 32")
        op.data, op.atoms = data.contiguous(), pack_scale_atoms(scales)
        return op

    @classmethod
    def empty(cls, rows: int, k: int, device: str | torch.device = "cuda") -> "Mxfp4Operand":
        """Buffers for a quantiser to fill, K a multiple of 32."""
        op = cls.__new__(cls)
        op.rows, op.k = _extents(rows, k, 32)
        op.data = torch.empty(rows, k // 2, dtype=torch.uint8, device=device)
        op.atoms = torch.empty(-(-rows // 128), -(-k // 128), 512, dtype=torch.uint8, device=device)
        return op

    def to(self, device) -> "Mxfp4Operand":
        op = Mxfp4Operand.__new__(Mxfp4Operand)
        op.rows, op.k, op.data, op.atoms = self.rows, self.k, self.data.to(device), self.atoms.to(device)
        return op

    def dequantize(self) -> torch.Tensor:
        return mxfp4_dequantize(self.data, unpack_scale_atoms(self.atoms, self.rows, self.k // 32))


class Fp8GroupOperand:
    """Activations in FP8: E4M3 (R, K) bytes and one FP32 scale per row and 128
    columns. ``scales`` is (R, ceil(K/128)) with the scales of one column
    group side by side in memory (strides (1, R)), as the product reads them.
    One made by :meth:`empty` is filled by :class:`.quantize.RmsNormFp8Plan`."""

    def __init__(self, x: torch.Tensor):
        self.rows, self.k = x.shape
        self.data, scales = fp8_group_quantize(x)
        self.scales = scales.t().contiguous().t()

    @classmethod
    def from_parts(cls, data: torch.Tensor, scales: torch.Tensor) -> "Fp8GroupOperand":
        """From E4M3 values (uint8 or float8_e4m3fn (R, K)) and FP32 scales (R, ceil(K/128))."""
        if data.dim() != 2 or data.dtype not in (torch.uint8, torch.float8_e4m3fn):
            raise ValueError("data must be (R, K) uint8 or float8_e4m3fn")
        op = cls.__new__(cls)
        op.rows, op.k = data.shape
        if tuple(scales.shape) != (op.rows, -(-op.k // 128)) or scales.dtype != torch.float32:
            raise ValueError(f"scales {tuple(scales.shape)} {scales.dtype}: expected float32 "
                             f"{(op.rows, -(-op.k // 128))}")
        op.data = data.contiguous().view(torch.uint8)
        op.scales = scales.t().contiguous().t()  # no copy where it is laid out so already
        return op

    @classmethod
    def empty(cls, rows: int, k: int, device: str | torch.device = "cuda") -> "Fp8GroupOperand":
        """Buffers for a quantiser to fill. (The product needs K a multiple of 16.)"""
        op = cls.__new__(cls)
        op.rows, op.k = _extents(rows, k, 1)
        op.data = torch.empty(rows, k, dtype=torch.uint8, device=device)
        op.scales = torch.empty(-(-k // 128), rows, dtype=torch.float32, device=device).t()
        return op

    @property
    def data(self) -> torch.Tensor:
        return self._data

    @data.setter
    def data(self, data: torch.Tensor) -> None:
        self._data, self._values = data, None

    @property
    def values(self) -> torch.Tensor:
        """The E4M3 values, (R, K) float8_e4m3fn (a view of ``data``)."""
        if self._values is None:  # one view per assigned ``data``: making one takes a microsecond
            self._values = self._data.view(torch.float8_e4m3fn)
        return self._values

    def to(self, device) -> "Fp8GroupOperand":
        return Fp8GroupOperand.from_parts(self.data.to(device), self.scales.to(device))

    def dequantize(self) -> torch.Tensor:
        return fp8_group_dequantize(self.data, self.scales)


class Fp8BlockOperand:
    """A quantised FP8 operand: E4M3 (R, K) bytes and FP32 128 x 128 block scales."""

    def __init__(self, x: torch.Tensor):
        self.rows, self.k = x.shape
        self.data, self.scales = fp8_block_quantize(x)

    @classmethod
    def from_parts(cls, data: torch.Tensor, scales: torch.Tensor) -> "Fp8BlockOperand":
        op = cls.__new__(cls)
        op.rows, op.k = data.shape
        op.data, op.scales = data.contiguous(), scales.contiguous().float()
        return op

    def to(self, device) -> "Fp8BlockOperand":
        return Fp8BlockOperand.from_parts(self.data.to(device), self.scales.to(device))

    def dequantize(self) -> torch.Tensor:
        return fp8_block_dequantize(self.data, self.scales)


def config4_inputs(m: int, n: int, k: int, seed: int = 0, device: str | torch.device = "cuda"):
    """The FP32 inputs of the block-scaled GEMMs: A (M, K) and B (N, K) ~ N(0, 1)
    from torch.Generator(seed) (the generator config 0 uses)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    a = torch.randn(m, k, generator=g)
    b = torch.randn(n, k, generator=g)
    return a.to(device), b.to(device)


# ------------------------------------------------------------------ GEMM plan
KINDS = {"nvfp4": nat.BB_LOWP_NVFP4, "fp8_block128": nat.BB_LOWP_FP8_BLOCK128}


_GEMM_OPERANDS = {"nvfp4": Nvfp4Operand, "fp8_block128": Fp8BlockOperand, "fp8_tensor_scaled": Fp8BlockOperand}


def _check_operands(kind: str, a, b) -> None:
    """Operands of the kind's own class: the classes share attribute names
    whose layouts differ (an Fp8GroupOperand's scales are per row)."""
    want = _GEMM_OPERANDS[kind]
    for name, op in (("A", a), ("B", b)):
        if not isinstance(op, want):
            raise ValueError(f"{name} is {type(op).__name__}, {kind} takes {want.__name__}")
        if kind == "nvfp4" and op.tensor_scale is None:
            raise ValueError(f"{name}'s tensor scale is found on the GPU, where only LowpLinearPlan reads it")


def _check_buffers(kind: str, a, b, d: torch.Tensor, sfa: torch.Tensor, sfb: torch.Tensor, stream) -> None:
    """Every buffer on D's device, contiguous, and at least as large as the
    native side reads: its tensor maps and scale loads are sized from M, N
    and K, not from the buffers."""
    if b.k != a.k or tuple(d.shape) != (a.rows, b.rows):
        raise ValueError("shape mismatch between A, B and D")
    for t in (a.data, b.data, sfa, sfb):
        if not t.is_cuda or not t.is_contiguous():
            raise ValueError("operands must be contiguous CUDA tensors")
        if t.device != d.device:
            raise ValueError(f"operands on {t.device}, D on {d.device}: all must be on one device")
    if stream.device != d.device:
        raise ValueError(f"stream on {stream.device}, tensors on {d.device}")
    row_bytes = a.k // 2 if kind == "nvfp4" else a.k
    for name, op in (("A", a), ("B", b)):
        if op.data.numel() * op.data.element_size() < op.rows * row_bytes:
            raise ValueError(f"{name} data holds fewer than {op.rows} x {row_bytes} bytes")
    scale_kind = nat.BB_LOWP_NVFP4 if kind == "nvfp4" else nat.BB_LOWP_FP8_BLOCK128
    for name, rows, t in (("A", a.rows, sfa), ("B", b.rows, sfb)):
        need = int(nat.bench_lib().bb_lowp_scale_bytes(scale_kind, rows, a.k))
        have = t.numel() * t.element_size()
        if need > 0 and have < need:
            raise ValueError(f"{name} scales hold {have} bytes, the kernel reads {need}")


class LowpGemmPlan:
    """D (M, N) BF16 = dequant(A) @ dequant(B)^T through the sm_100a
    block-scaled kernel (bb_lowp_plan_create of include/b200bench.h). A and B
    are :class:`Nvfp4Operand` for "nvfp4" (with a tensor scale known on the
    host) and :class:`Fp8BlockOperand` for "fp8_block128"."""

    def __init__(self, kind: str, a, b, d: torch.Tensor, stream: torch.cuda.Stream | None = None):
        if kind not in KINDS:
            raise ValueError(f"unknown kind {kind!r}; expected one of {sorted(KINDS)}")
        _check_operands(kind, a, b)
        if not d.is_cuda or d.dtype != torch.bfloat16 or not d.is_contiguous():
            raise ValueError("D must be a contiguous CUDA bfloat16 tensor")
        self.kind = kind
        self.m, self.n, self.k = a.rows, b.rows, a.k
        if b.k != a.k or tuple(d.shape) != (self.m, self.n):
            raise ValueError("shape mismatch between A, B and D")
        if kind == "nvfp4":
            sfa, sfb, gscale = a.atoms, b.atoms, a.tensor_scale * b.tensor_scale
        else:
            sfa, sfb, gscale = a.scales, b.scales, 1.0
        self.stream = stream if stream is not None else torch.cuda.current_stream(d.device)
        self._lib = nat.bench_lib()
        _check_buffers(kind, a, b, d, sfa, sfb, self.stream)
        self.a, self.b, self.d, self._keep = a, b, d, (sfa, sfb)
        handle = ctypes.c_void_p()
        info = nat.LowpInfo()
        with torch.cuda.device(d.device):
            nat.check("bb_lowp_plan_create", self._lib.bb_lowp_plan_create(
                KINDS[kind], self.m, self.n, self.k, a.data.data_ptr(), b.data.data_ptr(), sfa.data_ptr(),
                sfb.data_ptr(), float(gscale), d.data_ptr(), self.stream.cuda_stream, ctypes.byref(handle),
                ctypes.byref(info)))
        self._handle = handle
        self.info = info.as_dict()

    @property
    def flops(self) -> int:
        return 2 * self.m * self.n * self.k

    def run(self, iterations: int = 1) -> None:
        nat.check("bb_lowp_execute_n", self._lib.bb_lowp_execute_n(self._handle, int(iterations)))

    def synchronize(self) -> None:
        nat.check("bb_lowp_synchronize", self._lib.bb_lowp_synchronize(self._handle))

    @property
    def launches(self) -> int:
        return int(self._lib.bb_lowp_launches(self._handle))

    def close(self) -> None:
        if getattr(self, "_handle", None):
            self._lib.bb_lowp_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class CublasLtLowpPlan:
    """cuBLASLt's block-scaled GEMM on the same operands (the comparator, a
    library call; bb_cmp_lowp_plan_create of include/b200cmp.h).

    ``fp8_scales_kmajor`` chooses how the FP32 128 x 128 block scales are
    handed over: True passes them as stored ([row block][K block]), False
    passes the transpose ([K block][row block])."""

    CMP_KINDS = {**KINDS, "fp8_tensor_scaled": 3}

    def __init__(self, kind: str, a, b, d: torch.Tensor, autotune: bool = False,
                 stream: torch.cuda.Stream | None = None, fp8_scales_kmajor: bool = False):
        """kind "fp8_tensor_scaled" runs cuBLASLt's plain FP8 GEMM on the
        same E4M3 bytes without block scales: a throughput reference for the
        FP8 block-scaled kernel, not the same function."""
        if kind not in self.CMP_KINDS:
            raise ValueError(f"unknown kind {kind!r}")
        _check_operands(kind, a, b)
        self._lib = nat.cmp_lib()
        self.stream = stream if stream is not None else torch.cuda.current_stream(d.device)
        m, n, k = a.rows, b.rows, a.k
        if kind == "nvfp4":
            sfa, sfb, gscale = a.atoms, b.atoms, a.tensor_scale * b.tensor_scale
        else:
            sfa, sfb, gscale = a.scales, b.scales, 1.0
            if kind != "fp8_tensor_scaled" and not fp8_scales_kmajor:
                sfa, sfb = sfa.t().contiguous(), sfb.t().contiguous()
        if not d.is_cuda or d.dtype != torch.bfloat16 or not d.is_contiguous():
            raise ValueError("D must be a contiguous CUDA bfloat16 tensor")
        _check_buffers(kind, a, b, d, sfa, sfb, self.stream)
        self._keep = (a, b, sfa, sfb, d)
        handle = ctypes.c_void_p()
        info = nat.CmpInfo()
        rc = self._lib.bb_cmp_lowp_plan_create(self.CMP_KINDS[kind], m, n, k, a.data.data_ptr(), b.data.data_ptr(),
                                               sfa.data_ptr(), sfb.data_ptr(), float(gscale), d.data_ptr(),
                                               1 if autotune else 0, self.stream.cuda_stream, ctypes.byref(handle),
                                               ctypes.byref(info))
        if rc != 0:
            raise nat.NativeCallError("bb_cmp_lowp_plan_create", rc, self._lib.bb_cmp_last_error().decode())
        self._handle = handle
        self.info = info.as_dict()

    def run(self, iterations: int = 1) -> None:
        rc = self._lib.bb_cmp_execute_n(self._handle, int(iterations))
        if rc != 0:
            raise nat.NativeCallError("bb_cmp_execute_n", rc, self._lib.bb_cmp_last_error().decode())

    def close(self) -> None:
        if getattr(self, "_handle", None):
            self._lib.bb_cmp_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ------------------------------------------------------------------ linear layer
_LINEAR_KINDS = {Nvfp4Operand: ("nvfp4", nat.BB_LOWP_NVFP4, Nvfp4Operand),
                 Mxfp4Operand: ("mxfp4", nat.BB_LOWP_MXFP4, Mxfp4Operand),
                 Fp8GroupOperand: ("fp8_group128", nat.BB_LOWP_FP8_GROUP128, Fp8BlockOperand)}
_D_DTYPES = {torch.bfloat16: nat.BB_DTYPE_BF16, torch.float16: nat.BB_DTYPE_F16, torch.float32: nat.BB_DTYPE_F32}


class LowpLinearPlan:
    """D (M, N) = dequant(x) @ dequant(w)^T: the product of a linear layer with
    quantised weights and activations, for any number of rows from one token
    upwards and any N (bb_linear_plan_create of include/b200bench.h).

    The kind follows from the operands: :class:`Nvfp4Operand` or
    :class:`Mxfp4Operand` for both (K a multiple of 32), or
    :class:`Fp8GroupOperand` activations with :class:`Fp8BlockOperand`
    weights (K a multiple of 16). D is bfloat16, float16 or float32 with
    unit column stride and row stride >= N; its bytes outside (M, N) are not
    touched. Tensor scales found on the GPU (``tensor_scale_out``) are read there
    at every run. The plan keeps its operands; x and w may be refilled between
    runs by work on the plan's stream. Runs can be captured into a CUDA graph,
    which then needs the plan to stay alive."""

    def __init__(self, x, w, d: torch.Tensor, stream: torch.cuda.Stream | None = None):
        if type(x) not in _LINEAR_KINDS:
            raise ValueError(f"x is {type(x).__name__}; expected one of "
                             f"{sorted(c.__name__ for c in _LINEAR_KINDS)}")
        self.kind, kind, w_type = _LINEAR_KINDS[type(x)]
        if type(w) is not w_type:
            raise ValueError(f"{type(x).__name__} activations take {w_type.__name__} weights, got {type(w).__name__}")
        if d.dtype not in _D_DTYPES:
            raise ValueError("D must be bfloat16, float16 or float32")
        self.m, self.n, self.k = x.rows, w.rows, x.k
        if w.k != x.k or tuple(d.shape) != (self.m, self.n):
            raise ValueError(f"shape mismatch: x ({x.rows}, {x.k}), w ({w.rows}, {w.k}), D {tuple(d.shape)}")
        if (self.n > 1 and d.stride(1) != 1) or (self.m > 1 and d.stride(0) < self.n):
            raise ValueError("D must have unit column stride and a row stride of at least N")
        step = 16 if self.kind == "fp8_group128" else 32
        if self.k % step:
            raise ValueError(f"K = {self.k} must be a multiple of {step} for {self.kind}")
        fp8 = self.kind == "fp8_group128"
        sx, sw = (x.scales, w.scales) if fp8 else (x.atoms, w.atoms)
        scale_devs = [None if fp8 else getattr(op, "tensor_scale_out", None) for op in (x, w)]
        for name, t in (("x data", x.data), ("w data", w.data)) + (() if fp8 else (("x atoms", sx), ("w atoms", sw))):
            if t.element_size() != 1:
                raise ValueError(f"{name} is {t.dtype}, expected one byte an element")
        if fp8 and sw.dtype != torch.float32:
            raise ValueError(f"w scales are {sw.dtype}, expected torch.float32")
        tensors = [x.data, w.data, sx, sw, d] + [t for t in scale_devs if t is not None]
        if not all(t.is_cuda for t in tensors):
            raise ValueError("operands and D must be CUDA tensors")
        if len({t.device for t in tensors}) != 1:
            raise ValueError(f"operands and D on {sorted({str(t.device) for t in tensors})}: all must be on one device")
        row_bytes = self.k if fp8 else self.k // 2
        for name, op in (("x", x), ("w", w)):
            if not op.data.is_contiguous() or op.data.numel() * op.data.element_size() < op.rows * row_bytes:
                raise ValueError(f"{name} data must be contiguous and hold {op.rows} x {row_bytes} bytes")
        self._lib = nat.bench_lib()
        self._execute = self._lib.bb_linear_execute_n
        sx_ld = self.m
        if fp8:
            if tuple(sx.shape) != (self.m, -(-self.k // 128)) or (self.m > 1 and sx.stride(0) != 1) or (
                    sx.shape[1] > 1 and sx.stride(1) < self.m) or sx.dtype != torch.float32:
                raise ValueError("x scales must be float32 (M, ceil(K/128)) with strides (1, >= M)")
            sx_ld = sx.stride(1) if sx.shape[1] > 1 else max(self.m, 1)
        for name, t, weights, rows in (("x", sx, 0, self.m), ("w", sw, 1, self.n)):
            need = int(self._lib.bb_linear_scale_bytes(kind, weights, rows, self.k))
            if not (fp8 and not weights) and (not t.is_contiguous() or t.numel() * t.element_size() < need):
                raise ValueError(f"{name} scales must be contiguous and hold {need} bytes")
        self.stream = stream if stream is not None else torch.cuda.current_stream(d.device)
        if self.stream.device != d.device:
            raise ValueError(f"stream on {self.stream.device}, tensors on {d.device}")
        scales = [1.0 if fp8 or getattr(op, "tensor_scale", None) is None else op.tensor_scale for op in (x, w)]
        self.x, self.w, self.d, self._keep = x, w, d, tensors
        handle = ctypes.c_void_p()
        info = nat.LowpInfo()
        with torch.cuda.device(d.device):
            nat.check("bb_linear_plan_create", self._lib.bb_linear_plan_create(
                kind, self.m, self.n, self.k, x.data.data_ptr(), w.data.data_ptr(), sx.data_ptr(), sx_ld,
                sw.data_ptr(), scales[0], None if scale_devs[0] is None else scale_devs[0].data_ptr(), scales[1],
                None if scale_devs[1] is None else scale_devs[1].data_ptr(), d.data_ptr(), _D_DTYPES[d.dtype],
                d.stride(0) if self.m > 1 else self.n, self.stream.cuda_stream, ctypes.byref(handle),
                ctypes.byref(info)))
        self._handle = handle
        self.info = info.as_linear_dict()

    @property
    def flops(self) -> int:
        return 2 * self.m * self.n * self.k

    def run(self, iterations: int = 1) -> None:
        """`iterations` back-to-back launches on the plan's stream (async). A
        device-side wait that times out ends its launch without an error here;
        :meth:`synchronize` reports it, and until then later launches of the
        plan give up early and leave D undefined."""
        status = self._execute(self._handle, int(iterations))
        if status:
            nat.check("bb_linear_execute_n", status)

    def synchronize(self) -> None:
        """Waits for the stream; raises on a device-side wait timeout (the plan
        is then to be closed)."""
        nat.check("bb_linear_synchronize", self._lib.bb_linear_synchronize(self._handle))

    @property
    def launches(self) -> int:
        return int(self._lib.bb_linear_launches(self._handle))

    def close(self) -> None:
        if getattr(self, "_handle", None):
            self._lib.bb_linear_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
