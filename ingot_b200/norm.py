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
    # (each condition once, in few steps: a call of one row is bound by the host. What fails one is described by _check)
    dev, ok = -1, (out is not None or codes is not None) and rotate in ROTATIONS and (x is not None or residual_out is None)
    xp = xt = ldx = rop = ldro = wp = wt = op = ot = ldo = cp = ldc = sp = 0
    try:
        (have, d), (ldr, step) = residual.shape, residual.stride()
        rt, dev = _DT.get(residual.dtype, -1), residual.get_device()
        ok = ok and 0 <= rows <= have and (step == 1 or d == 1) and 1 <= d <= MAX_WIDTH and rt >= 0 and eps >= 0
        if x is not None:
            (n, k), (ldx, step) = x.shape, x.stride()
            xp, xt = x.data_ptr(), _DT.get(x.dtype, -1)
            ok = ok and n >= rows and k == d and (step == 1 or d == 1) and xt >= 0 and x.get_device() == dev
            if residual_out is None:
                rop, ldro = residual.data_ptr(), ldr
            else:
                (n, k), (ldro, step) = residual_out.shape, residual_out.stride()
                rop = residual_out.data_ptr()
                ok = ok and n >= rows and k == d and (step == 1 or d == 1) and residual_out.get_device() == dev and residual_out.dtype == residual.dtype
        if weight is not None:
            wp, wt = weight.data_ptr(), _DT.get(weight.dtype, -1)
            ok = ok and wt >= 0 and weight.get_device() == dev and weight.numel() == d and weight.is_contiguous()
        if out is not None:
            (n, k), (ldo, step) = out.shape, out.stride()
            op, ot = out.data_ptr(), _DT.get(out.dtype, -1)
            ok = ok and n >= rows and k == d and (step == 1 or d == 1) and ot >= 0 and out.get_device() == dev
        if codes is not None:
            (n, k), (ldc, step), (m,), (one,) = codes.shape, codes.stride(), scales.shape, scales.stride()
            cp, sp = codes.data_ptr(), scales.data_ptr()
            ok = (ok and n >= rows and k == d and (step == 1 or d == 1) and codes.dtype == torch.int8 and scales.dtype == torch.float32 and m >= rows and (one == 1 or rows <= 1)
                  and codes.get_device() == dev and scales.get_device() == dev and (not rotate or d % rotate == 0))
        elif rotate or scales is not None:
            ok = False
    except (ValueError, AttributeError):  # another number of dimensions, no tensor
        ok = False
    if not ok or dev < 0:
        _check(x, residual, weight, rows, eps, residual_out, out, codes, scales, rotate)
        if residual.device.type != "cuda":
            _no_cpu()
        raise ValueError("add_rmsnorm does not take these tensors")
    if rows == 0:  # (tensors of no rows have no address)
        return
    ctx = capi.context(dev)
    if rows <= 1:  # (one row has no stride)
        ldx = ldr = ldro = ldo = ldc = d
    st = capi.call().add_rmsnorm(ctx.address, stream.cuda_stream if stream is not None else _raw_stream(dev), xp, xt, ldx, residual.data_ptr(), rt, ldr,
                                 rop, ldro, wp, wt, weight_offset, eps, rows, d, op, ot, ldo, cp, ldc, sp, rotate)
    if st:
        ctx.check(st)
