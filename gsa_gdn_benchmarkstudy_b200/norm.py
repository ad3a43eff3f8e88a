"""Root-mean-square norm with the residual's addition, in the inputs' type (with
gradients) or with an output in 8 bits.

    h = x + residual              (rounded to the inputs' type; x without a residual)
    y = h / sqrt(mean(h^2) + eps) * weight

Both functions run on the tensors' device and its current stream; there is no
CPU path.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DTYPES, _cuda, _dtype_code, _no_tangents, _on, _ptr, _raw_stream


def _unit(t: torch.Tensor) -> torch.Tensor:
    """Rows [R, D] with unit inner stride (a copy only where the layout needs one)."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(x, weight, residual) -> None:
    _no_tangents(x, weight, residual)
    if not x.is_cuda:
        _cuda(x, weight, residual)
    device = x.get_device()
    if weight.get_device() != device or (residual is not None
                                         and residual.get_device() != device):
        _cuda(x, weight, residual)
        raise ValueError("all tensors must be on one device")
    shape = x.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"x must have a last dim of at least 1, got {tuple(shape)}")
    width = shape[-1]
    if x.dtype not in _DTYPES or weight.dtype not in _DTYPES:
        _dtype_code(x), _dtype_code(weight)
    if width > 32768:
        raise ValueError(f"rows of at most 32768 values, got {width}")
    if weight.shape != (width,):
        raise ValueError(f"weight must be [{width}], got {tuple(weight.shape)}")
    if residual is not None and (residual.shape != shape or residual.dtype is not x.dtype):
        raise ValueError("residual must match x in shape and dtype")


def _forward(x, weight, residual, eps, want_rstd):
    """(y, h, rstd) of x and residual as rows."""
    rows, width = x.shape
    device = x.device
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty(
        (rows, width), dtype=x.dtype, device=device)
    h = rstd = h_ptr = r_ptr = rstd_ptr = None
    r_stride = 0
    if residual is not None:
        h = torch.empty_like(y)
        h_ptr, r_ptr, r_stride = h.data_ptr(), residual.data_ptr(), _row_stride(residual)
    if want_rstd:
        rstd = torch.empty(rows, dtype=torch.float32, device=device)
        rstd_ptr = rstd.data_ptr()
    with _on(device):
        rc = _lib.load().gsa_rms_norm(
            x.data_ptr(), _row_stride(x), r_ptr, r_stride, weight.data_ptr(),
            _DTYPES[weight.dtype], eps, _DTYPES[x.dtype], rows, width, y.data_ptr(), width, h_ptr,
            width, rstd_ptr, _raw_stream(device.index))
    if rc:
        _lib.check(rc, "gsa_rms_norm")
    return y, h, rstd


class _RmsNorm(torch.autograd.Function):
    """rms_norm of rows [R, D]."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = _forward(_unit(x), weight, None if residual is None else _unit(residual), eps,
                              True)
        ctx.set_materialize_grads(False)
        if h is None:
            ctx.save_for_backward(x, weight, rstd)
            return y
        ctx.save_for_backward(h, weight, rstd)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        _, want_w, want_r, _ = ctx.needs_input_grad
        if dy is None:  # only the sum h was used
            return dh, None, dh, None
        h, weight, rstd = ctx.saved_tensors
        h, dy = _unit(h), _unit(dy.to(h.dtype))
        rows, width = h.shape
        dh_ptr = dw = dw_ptr = ws = ws_ptr = None
        dh_stride = need = 0
        if dh is not None:
            dh = _unit(dh.to(h.dtype))
            dh_ptr, dh_stride = dh.data_ptr(), _row_stride(dh)
        lib, device = _lib.load(), h.device
        dx = torch.empty_like(h) if h.is_contiguous() else torch.empty(
            (rows, width), dtype=h.dtype, device=device)
        if want_w:
            dw = torch.empty_like(weight)
            need = lib.gsa_rms_norm_backward_workspace_size(rows, width)
            ws = rstd.new_empty(need // 4)  # floats
            dw_ptr, ws_ptr = dw.data_ptr(), ws.data_ptr()
        with _on(device):
            rc = lib.gsa_rms_norm_backward(
                dy.data_ptr(), _row_stride(dy), dh_ptr, dh_stride, h.data_ptr(), _row_stride(h),
                weight.data_ptr(), _DTYPES[weight.dtype], rstd.data_ptr(), _DTYPES[h.dtype], rows,
                width, dx.data_ptr(), width, dw_ptr, ws_ptr, need, _raw_stream(device.index))
        if rc:
            _lib.check(rc, "gsa_rms_norm_backward")
        return dx, dw, dx if want_r else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             residual: torch.Tensor | None = None):
    """RMS norm over the last dim (at most 32768 values), with an optional residual.

    x [..., D] (bf16 or fp32), weight [D] (bf16 or fp32).  Returns y in x's dtype, or
    (y, h) with ``residual`` (x's shape and dtype): h = x + residual rounded to
    that dtype, which is what the norm reads and the next residual is.
    Differentiable once, in reverse mode, in x, weight and the residual; the weight's gradient
    adds the rows up in a fixed order."""
    _check(x, weight, residual)
    weight = weight.contiguous()
    eps = float(eps)
    shape = x.shape
    flat = len(shape) == 2
    if not flat:
        x = x.reshape(-1, shape[-1])
        residual = residual.reshape(-1, shape[-1]) if residual is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (
            residual is not None and residual.requires_grad)):
        got = _RmsNorm.apply(x, weight, residual, eps)
        y, h = (got, None) if residual is None else got
    else:
        y, h, _ = _forward(_unit(x), weight, None if residual is None else _unit(residual), eps,
                           False)
    if not flat:
        y = y.view(shape)
        h = h.view(shape) if h is not None else None
    return y if h is None else (y, h)


def _rows_of(t: torch.Tensor, width: int, group_size) -> torch.Tensor:
    """t as rows [R, width] that the 8-bit kernel reads: group scales move 16 bytes at a time, so
    rows that are not on 16 bytes are copied for them."""
    t = _unit(t if t.dim() == 2 else t.reshape(-1, width))
    if group_size and (t.data_ptr() % 16 or _row_stride(t) * t.element_size() % 16):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
                 residual: torch.Tensor | None = None, group_size: int | None = None):
    """``rms_norm`` with its output in 8 bits (torch.float8_e4m3fn) and fp32 scales.

    y8 * scale stands for the norm's values: the scale is the largest magnitude
    of a row, or of each ``group_size`` = 128 values of it (D a multiple of 128),
    over 448, the type's largest number; the values are rounded once, from fp32.
    Returns (y8 [..., D], scale [..., 1] or [..., D / 128]) and, with a residual, h.
    No gradients."""
    _check(x, weight, residual)
    if group_size not in (None, 128):
        raise ValueError(f"group_size must be None or 128, got {group_size}")
    width = x.shape[-1]
    if group_size and width % 128:
        raise ValueError(f"group scales need a last dim that is a multiple of 128, got {width}")
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (
            residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm_fp8 has no gradients; use rms_norm")

    x2 = _rows_of(x, width, group_size)
    r2 = None if residual is None else _rows_of(residual, width, group_size)
    weight = weight.contiguous()
    if group_size and weight.data_ptr() % 16:
        weight = weight.clone()
    rows, groups = x2.shape[0], width // group_size if group_size else 1
    device, dtype = x.device, x.dtype
    y = (torch.empty_like(x2, dtype=torch.float8_e4m3fn) if x2.is_contiguous() else
         x2.new_empty((rows, width), dtype=torch.float8_e4m3fn))
    scale = x2.new_empty((rows, groups), dtype=torch.float32)
    h = h_ptr = r_ptr = None
    r_stride = 0
    if r2 is not None:
        h = torch.empty_like(x2) if x2.is_contiguous() else x2.new_empty((rows, width))
        h_ptr, r_ptr, r_stride = h.data_ptr(), r2.data_ptr(), _row_stride(r2)
    with _on(device):
        rc = _lib.load().gsa_rms_norm_fp8(
            x2.data_ptr(), _row_stride(x2), r_ptr, r_stride, weight.data_ptr(),
            _DTYPES[weight.dtype], float(eps), _DTYPES[dtype], rows, width, y.data_ptr(), width,
            scale.data_ptr(), group_size or 0, h_ptr, width, _raw_stream(device.index))
    if rc:
        _lib.check(rc, "gsa_rms_norm_fp8")
    shape = x.shape
    if len(shape) != 2:
        y, scale = y.view(shape), scale.view(shape[:-1] + (groups,))
        h = h.view(shape) if h is not None else None
    return (y, scale) if h is None else (y, scale, h)
