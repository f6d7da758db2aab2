"""Root-mean-square norm with the residual's addition (gs_rms_norm_forward / _backward) and its
8-bit output for the next product (gs_rms_norm_e4m3)."""

from __future__ import annotations

import torch

from custom_rasterizer_cuda import _lib

from ._tokens import DTYPES, on_device, require, stream, usable, wants_grad

MAX_WIDTH = 32768


def _check(x, weight, residual, eps):
    for t, name in ((x, "x"), (weight, "weight"), (residual, "residual")):
        if t is None:
            continue
        require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
        require(t.dtype == x.dtype and t.device == x.device,
                f"{name} must have x's type and device")
    require(x.dtype in DTYPES, "x must be float32, float16 or bfloat16")
    require(x.dim() >= 1 and 1 <= x.shape[-1] <= MAX_WIDTH,
            f"the last axis must have between 1 and {MAX_WIDTH} elements")
    require(weight.shape == x.shape[-1:], "weight must have one element for each of the last axis")
    require(residual is None or residual.shape == x.shape, "residual must have x's shape")
    require(eps >= 0.0, "eps must be non-negative")


def _rows(t):
    """A contiguous tensor with t's numbers, on a 16-byte boundary where that costs no copy."""
    return t if t.is_contiguous() else t.contiguous()


def _forward(x, weight, residual, eps, save):
    x, weight = _rows(x), _rows(weight)
    width = x.shape[-1]
    rows = x.numel() // width
    y = torch.empty_like(x)
    h = None
    if residual is not None:
        residual = _rows(residual)
        h = torch.empty_like(x)
    rstd = torch.empty(rows, device=x.device, dtype=torch.float32) if save else None
    if rows:
        with on_device(x.device):
            _lib.check(_lib.lib.gs_rms_norm_forward(
                DTYPES[x.dtype], rows, width, x.data_ptr(),
                None if residual is None else residual.data_ptr(), weight.data_ptr(), eps,
                y.data_ptr(), None if h is None else h.data_ptr(),
                None if rstd is None else rstd.data_ptr(), stream(x.device)))
    return x, weight, y, h, rstd


def _backward(dy, dh, h, weight, rstd):
    width = h.shape[-1]
    rows = h.numel() // width
    dy = _rows(dy)
    if dh is not None:
        dh = _rows(dh)
    dx = torch.empty_like(h)
    dw = torch.empty_like(weight)
    ws_bytes = _lib.lib.gs_rms_norm_backward_workspace_size(rows, width)
    ws = torch.empty(ws_bytes, device=h.device, dtype=torch.uint8)
    with on_device(h.device):
        _lib.check(_lib.lib.gs_rms_norm_backward(
            DTYPES[h.dtype], rows, width, dy.data_ptr(), None if dh is None else dh.data_ptr(),
            h.data_ptr(), weight.data_ptr(), rstd.data_ptr(), dx.data_ptr(), dw.data_ptr(),
            ws.data_ptr(), ws_bytes, stream(h.device)))
    return dx, dw


class RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        x, weight, y, _, rstd = _forward(x, weight, None, eps, True)
        ctx.save_for_backward(x, weight, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        h, weight, rstd = ctx.saved_tensors
        dx, dw = _backward(dy, None, h, weight, rstd)
        return dx, dw, None


class RMSNormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.set_materialize_grads(False)
        _, weight, y, h, rstd = _forward(x, weight, residual, eps, True)
        ctx.save_for_backward(h, weight, rstd)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:  # only the residual stream was used
            return dh, None, dh, None
        dx, dw = _backward(dy, dh, h, weight, rstd)
        return dx, dw, dx, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
             eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last axis, with h = x + residual where a
    residual is given: then (y, h) is returned, h being the new residual stream, else y alone.
    float32, float16 or bfloat16, all of one type."""
    _check(x, weight, residual, eps)
    if wants_grad(x, weight, residual):
        if residual is None:
            return RMSNorm.apply(x, weight, float(eps))
        return RMSNormResidual.apply(x, weight, residual, float(eps))
    _, _, y, h, _ = _forward(x, weight, residual, float(eps), False)
    return y if residual is None else (y, h)


def rms_norm_8bit(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                  eps: float = 1e-6, group: int = 0):
    """rms_norm whose y is written in 8 bits: (q, scales), or (q, scales, h) with a residual, with
    q (float8_e4m3fn, x's shape) times its scale near y and scales = max|y| / 448 of each row
    ([..., 1]) or, with `group` 128, of each 128 numbers ([..., width / 128]). For prediction:
    no gradient."""
    _check(x, weight, residual, eps)
    require(not wants_grad(x, weight, residual), "rms_norm_8bit has no gradient")
    width = x.shape[-1]
    require(group == 0 or (group == 128 and width % 128 == 0),
            "group must be 0 (one scale a row) or 128, dividing the width")
    x, weight = _rows(x), _rows(weight)
    if residual is not None:
        residual = _rows(residual)
    if group:
        per = 16 // x.element_size()
        x, weight = usable(x, per), usable(weight, per)
        residual = residual if residual is None else usable(residual, per)
    rows = x.numel() // width
    q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
    scales = torch.empty((*x.shape[:-1], width // group if group else 1), device=x.device,
                         dtype=torch.float32)
    h = None if residual is None else torch.empty_like(x)
    if rows:
        with on_device(x.device):
            _lib.check(_lib.lib.gs_rms_norm_e4m3(
                DTYPES[x.dtype], rows, width, group, x.data_ptr(),
                None if residual is None else residual.data_ptr(), weight.data_ptr(), float(eps),
                q.data_ptr(), scales.data_ptr(), None if h is None else h.data_ptr(),
                stream(x.device)))
    return (q, scales) if h is None else (q, scales, h)
