"""Quantisers as kernels: RMS norm with the residual's addition and FP8 output,
and the 4-bit microscaled formats. They fill the operands that
:class:`.lowp.LowpLinearPlan` multiplies.

Like the GEMM plans, a plan is built once for fixed tensors and run many
times on its stream; the tensors stay the caller's, and x may hold new data at
every run. Runs can be captured into a CUDA graph, which then needs the plan
(and its tensors) to stay alive; a plan's runs belong to one stream at a time.
``lowp.nvfp4_quantize``, ``lowp.mxfp4_quantize`` and
``lowp.fp8_group_quantize`` are the same formats in torch; the 4-bit
kernels equal them bit for bit (on the CPU, where torch divides exactly).
Plans are made outside a capture (making one may allocate), and run on their own
stream whatever the current one is.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as nat
from .lowp import Fp8GroupOperand, Mxfp4Operand, Nvfp4Operand

_DTYPES = {torch.bfloat16: nat.BB_DTYPE_BF16, torch.float16: nat.BB_DTYPE_F16, torch.float32: nat.BB_DTYPE_F32}


def _matrix(name: str, t: torch.Tensor, shape: tuple[int, int], like: torch.Tensor | None = None) -> int:
    """Checks one (rows, cols) tensor; returns its row stride."""
    if t.dim() != 2 or tuple(t.shape) != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {shape}")
    if t.dtype not in _DTYPES or (like is not None and t.dtype != like.dtype):
        raise ValueError(f"{name} is {t.dtype}, expected {like.dtype if like is not None else sorted(map(str, _DTYPES))}")
    rows, cols = shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        raise ValueError(f"{name} must have unit column stride and a row stride of at least its width")
    return t.stride(0) if rows > 1 else cols


def _one_device(tensors: list[torch.Tensor], stream: torch.cuda.Stream | None) -> torch.cuda.Stream:
    if not all(t.is_cuda for t in tensors):
        raise ValueError("all tensors must be CUDA tensors")
    devices = {t.device for t in tensors}
    if len(devices) != 1:
        raise ValueError(f"tensors on {sorted(map(str, devices))}: all must be on one device")
    device = tensors[0].device
    stream = stream if stream is not None else torch.cuda.current_stream(device)
    if stream.device != device:
        raise ValueError(f"stream on {stream.device}, tensors on {device}")
    return stream


class _QuantPlan:
    _handle: ctypes.c_void_p | None = None

    def run(self, iterations: int = 1) -> None:
        """`iterations` back-to-back runs on the plan's stream (async)."""
        status = self._execute(self._handle, int(iterations))
        if status:
            nat.check("bb_quant_execute_n", status)

    def synchronize(self) -> None:
        nat.check("bb_quant_synchronize", self._lib.bb_quant_synchronize(self._handle))

    @property
    def launches(self) -> int:
        return int(self._lib.bb_quant_launches(self._handle))

    def close(self) -> None:
        if self._handle:
            self._lib.bb_quant_destroy(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RmsNormFp8Plan(_QuantPlan):
    """FP8 activations of the next linear layer from the residual stream:

        h = x + residual                   (rounded to x's dtype; h = x without a residual)
        y = h * rsqrt(mean(h^2) + eps) * weight
        s = max|y| / 448                   per row and 128 columns, 1 where that is 0 in FP32
        out = e4m3(y / s), out.scales = s

    ``x``, ``residual`` and ``residual_out`` are (rows, cols) bfloat16, float16
    or float32 of one dtype, with unit column stride; ``residual_out`` receives
    h (it may be ``residual`` or ``x``; by default the sum is not stored).
    ``weight`` is (cols,), of x's dtype or float32. cols is at most 65536;
    rows may be 0. Finite rows are right up to the ends of x's range, where
    squares leave FP32's (y itself must lie inside). A row that holds a NaN is NaN, scales and codes. In one
    that holds an infinity the formula gives NaN for its 128 columns and, as
    1 / rms is 0, codes 0 with scale 1 for the others: a product's row of either
    is NaN. With eps = 0 a row of zeros is NaN (0 / 0)."""

    def __init__(self, x: torch.Tensor, weight: torch.Tensor, out: Fp8GroupOperand, residual: torch.Tensor | None = None,
                 residual_out: torch.Tensor | None = None, eps: float = 1e-6,
                 stream: torch.cuda.Stream | None = None):
        if not isinstance(out, Fp8GroupOperand):
            raise ValueError(f"out is {type(out).__name__}, expected Fp8GroupOperand")
        shape = (out.rows, out.k)
        x_ld = _matrix("x", x, shape)
        lds = [_matrix(name, t, shape, x) if t is not None else 0
               for name, t in (("residual", residual), ("residual_out", residual_out))]
        if weight.dim() != 1 or weight.shape[0] != out.k or not weight.is_contiguous():
            raise ValueError(f"weight is {tuple(weight.shape)}, expected contiguous ({out.k},)")
        if weight.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"weight is {weight.dtype}, expected {x.dtype} or torch.float32")
        if not eps >= 0:
            raise ValueError("eps must not be negative")
        if not out.data.is_contiguous() or out.data.numel() < out.rows * out.k or out.data.element_size() != 1:
            raise ValueError("out.data must be contiguous (rows, cols) of one byte an element")
        s = out.scales
        if tuple(s.shape) != (out.rows, -(-out.k // 128)) or (out.rows > 1 and s.stride(0) != 1) or (
                s.shape[1] > 1 and s.stride(1) < out.rows) or s.dtype != torch.float32:
            raise ValueError("out.scales must be float32 (rows, ceil(cols/128)) with strides (1, >= rows)")
        tensors = [t for t in (x, residual, residual_out, weight, out.data, out.scales) if t is not None]
        self.stream = _one_device(tensors, stream)
        self.x, self.out, self.residual_out, self._keep = x, out, residual_out, tensors
        self._lib = nat.bench_lib()
        self._execute = self._lib.bb_quant_execute_n
        handle = ctypes.c_void_p()
        with torch.cuda.device(x.device):
            nat.check("bb_rmsnorm_fp8_plan_create", self._lib.bb_rmsnorm_fp8_plan_create(
                out.rows, out.k, x.data_ptr(), _DTYPES[x.dtype], x_ld,
                None if residual is None else residual.data_ptr(), lds[0],
                None if residual_out is None else residual_out.data_ptr(), lds[1], weight.data_ptr(),
                _DTYPES[weight.dtype], float(eps), out.data.data_ptr(), out.k, s.data_ptr(),
                s.stride(1) if s.shape[1] > 1 else max(out.rows, 1), self.stream.cuda_stream, ctypes.byref(handle)))
        self._handle = handle


class Fp4QuantPlan(_QuantPlan):
    """x (rows, K) bfloat16, float16 or float32 into ``out``, an
    :class:`.lowp.Nvfp4Operand` or :class:`.lowp.Mxfp4Operand` made by its
    ``empty``: codes, and scales as the atoms the product reads. An NVFP4
    operand without a tensor scale has it found from x at every run (one more
    reading of x, and one more launch unless x is a few rows and ``values`` is
    not given) and left in ``out.tensor_scale_out``.

    ``values``, if given, is (rows, K) of x's dtype and receives what the codes
    stand for (x as the product sees it: the forward value of
    quantisation-aware training, or the quantisation error's other side). It
    may be x itself."""

    def __init__(self, x: torch.Tensor, out: Nvfp4Operand | Mxfp4Operand, values: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None):
        if not isinstance(out, (Nvfp4Operand, Mxfp4Operand)):
            raise ValueError(f"out is {type(out).__name__}, expected Nvfp4Operand or Mxfp4Operand")
        nvfp4 = isinstance(out, Nvfp4Operand)
        shape = (out.rows, out.k)
        x_ld = _matrix("x", x, shape)
        v_ld = _matrix("values", values, shape, x) if values is not None else 0
        if out.k % 32:
            raise ValueError(f"K = {out.k} must be a multiple of 32")
        if nvfp4 and out.scales is not None:
            raise ValueError("out holds quantised data already: make one with Nvfp4Operand.empty")
        scale_out = out.tensor_scale_out if nvfp4 else None
        if nvfp4 and scale_out is None and not 0 < out.tensor_scale < float("inf"):
            raise ValueError(f"tensor scale {out.tensor_scale} must be positive and finite")
        per_atom = 64 if nvfp4 else 128
        atoms = -(-out.rows // 128) * -(-out.k // per_atom) * 512
        if not out.data.is_contiguous() or out.data.numel() < out.rows * out.k // 2 or not out.atoms.is_contiguous() \
                or out.atoms.numel() < atoms or out.data.element_size() != 1 or out.atoms.element_size() != 1:
            raise ValueError("out.data and out.atoms must be contiguous bytes and hold (rows, K/2) and all atoms")
        tensors = [t for t in (x, values, out.data, out.atoms, scale_out) if t is not None]
        self.stream = _one_device(tensors, stream)
        self.x, self.out, self.values, self._keep = x, out, values, tensors
        self._lib = nat.bench_lib()
        self._execute = self._lib.bb_quant_execute_n
        handle = ctypes.c_void_p()
        with torch.cuda.device(x.device):
            nat.check("bb_fp4_quant_plan_create", self._lib.bb_fp4_quant_plan_create(
                nat.BB_LOWP_NVFP4 if nvfp4 else nat.BB_LOWP_MXFP4, out.rows, out.k, x.data_ptr(), _DTYPES[x.dtype],
                x_ld, out.data.data_ptr(), out.atoms.data_ptr(),
                out.tensor_scale if nvfp4 and scale_out is None else 1.0,
                None if scale_out is None else scale_out.data_ptr(),
                None if values is None else values.data_ptr(), v_ld, self.stream.cuda_stream, ctypes.byref(handle)))
        self._handle = handle
