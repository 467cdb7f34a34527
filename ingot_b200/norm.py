"""The step between two sublayers: residual addition, weighted RMS norm, and int8 codes for W8A8 linears in one kernel
(iq_add_rmsnorm). The reference's norms are kernels of their own (Shaders/verify.metal:503-523)."""
from __future__ import annotations

from typing import Optional

import torch

from . import capi
from .linear import _DT, _no_cpu, _raw_stream

MAX_WIDTH = 32768
ROTATIONS = (0, 32, 256)


def _rows(name: str, t: torch.Tensor, rows: int, d: int):
    if t.dim() != 2 or t.shape[0] < rows or t.shape[1] != d or (d > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} is [at least {rows}, {d}] with neighbouring elements in a row, not {tuple(t.shape)} of strides {t.stride()}")


def _check(x, residual, weight, rows, eps, residual_out, out, codes, scales, rotate):
    """Shapes, types and devices, whatever device they are on."""
    if residual.dim() != 2:
        raise ValueError("residual is [rows, d]")
    d = residual.shape[1]
    if rows < 0 or not 1 <= d <= MAX_WIDTH or not eps >= 0:
        raise ValueError(f"rows = {rows}, d = {d} (1 to {MAX_WIDTH}), eps = {eps}")
    if x is None and residual_out is not None:
        raise ValueError("residual_out is the sum's place: without x there is none")
    if out is None and codes is None:
        raise ValueError("neither out nor codes is wanted")
    if (codes is None) != (scales is None):
        raise ValueError("codes come with scales")
    if rotate not in ROTATIONS or (rotate and (codes is None or d % rotate)):
        raise ValueError(f"the rotation is the codes', in blocks of 32 or 256 that divide d = {d}, not {rotate}")
    for name, t in (("x", x), ("residual", residual), ("residual_out", residual_out), ("out", out)):
        if t is not None:
            if t.dtype not in _DT:
                raise TypeError(f"{name} is float32, float16 or bfloat16, not {t.dtype}")
            _rows(name, t, rows, d)
    if residual_out is not None and residual_out.dtype != residual.dtype:
        raise TypeError("residual_out has residual's type")
    if weight is not None:
        if weight.dtype not in _DT:
            raise TypeError(f"weight is float32, float16 or bfloat16, not {weight.dtype}")
        if weight.numel() != d or not weight.is_contiguous():
            raise ValueError(f"weight is [{d}], contiguous")
    if codes is not None:
        if codes.dtype != torch.int8 or scales.dtype != torch.float32:
            raise TypeError("codes are int8, scales float32")
        _rows("codes", codes, rows, d)
        if scales.dim() != 1 or scales.numel() < rows or (rows > 1 and scales.stride(0) != 1):
            raise ValueError(f"scales is [at least {rows}], contiguous")
    for t in (x, weight, residual_out, out, codes, scales):
        if t is not None and t.device != residual.device:
            raise ValueError("the tensors are on different devices")


def add_rmsnorm(x: Optional[torch.Tensor], residual: torch.Tensor, weight: Optional[torch.Tensor], rows: int, *, eps: float = 1e-6,
                weight_offset: float = 0.0, residual_out: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                codes: Optional[torch.Tensor] = None, scales: Optional[torch.Tensor] = None, rotate: int = 0,
                stream: Optional[torch.cuda.Stream] = None):
    """r = residual + x into residual_out (residual itself when absent), then RMSNorm(r) * (weight + weight_offset) into `out` and / or as
    int8 rows into `codes` and `scales`, rotated in blocks of `rotate` inputs (what `I8Linear.rotate` says). Tensors are
    [rows, d] with any row stride; x None: the norm of residual alone; weight None: weights of one.
    residual_out may be residual, out may be x (same stride and element size); nothing else may overlap."""
    try:
        dev = residual.get_device()
    except AttributeError:  # no tensor
        dev = -1
    st = None
    if dev >= 0:  # (a call of one row is bound by the host: the conditions are looked at in csrc/pycall.c, and what fails one is described by _check)
        ctx = capi.context(dev)
        st = capi.call().add_rmsnorm(ctx.address, stream.cuda_stream if stream is not None else _raw_stream(dev), dev, x, residual, weight, rows, eps, weight_offset,
                                     residual_out, out, codes, scales, rotate)
    if st is None:
        _check(x, residual, weight, rows, eps, residual_out, out, codes, scales, rotate)
        if residual.device.type != "cuda":
            _no_cpu()
        raise ValueError("add_rmsnorm does not take these tensors")
    if st:
        ctx.check(st)
