"""Rotary positions with several axes, as one autograd op over gs_rotary_axes.

`rotary_axes(x, positions, axis_dims)` turns pairs of each head's numbers by angles that grow with
the token's coordinates, one block of numbers for each axis: for images and video (view or time,
row, column). Image tokens sit at whole coordinates (int32), Gaussians at those of their projected
means (float32).
"""

from __future__ import annotations

import ctypes
import math

import torch

from custom_rasterizer_cuda import _lib

from ._tokens import DTYPES, check_tokens, on_device, require, stream, usable, view4, wants_grad


def _rotate(x, positions, n, dims, bases, interleaved, inverse):
    B, L, H, D = x.shape
    x = usable(x)
    y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
    if y.numel() == 0:
        return y
    xv, yv = view4(x), view4(y)
    pb = positions.stride(0) if positions.shape[0] > 1 else 0
    with on_device(x.device):
        _lib.check(_lib.lib.gs_rotary_axes(
            DTYPES[x.dtype], B, L, H, D, ctypes.addressof(xv), ctypes.addressof(yv),
            positions.data_ptr(),
            _lib.GS_INT32 if positions.dtype == torch.int32 else _lib.GS_FP32, pb,
            positions.stride(1), n, dims, bases, int(interleaved), int(inverse),
            stream(x.device)))
    return y


class RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, n, dims, bases, interleaved, inverse):
        ctx.save_for_backward(positions)
        ctx.args = (n, dims, bases, interleaved, not inverse)
        return _rotate(x, positions, n, dims, bases, interleaved, inverse)

    @staticmethod
    def backward(ctx, dy):
        (positions,) = ctx.saved_tensors
        return _rotate(dy, positions, *ctx.args), None, None, None, None, None, None


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, axis_dims, base=10000.0,
                interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """x[B, L, H, D] (float32, float16 or bfloat16) turned by positions[B or 1, L, axes] (int32 or
    float32). `axis_dims` gives the (even) number of a head's numbers that each axis owns, from
    the first on; what is left over is copied. Pair j of an axis with d numbers turns by
    position * base^(-2 j / d); pairs are (j, j + d / 2) of the axis's block, or neighbours when
    `interleaved`. `base` is one number or one for each axis. `inverse` turns back. No gradient
    reaches the positions."""
    check_tokens(x, "x", 4)
    check_tokens(positions, "positions", 3)
    require(x.dtype in DTYPES, "x must be float32, float16 or bfloat16")
    require(positions.dtype in (torch.int32, torch.float32), "positions must be int32 or float32")
    require(positions.device == x.device, "x and positions must be on the same device")
    n = len(axis_dims)
    require(1 <= n <= 4, "between 1 and 4 axes")
    require(positions.shape[0] in (1, x.shape[0]) and positions.shape[1] == x.shape[1]
            and positions.shape[2] == n, "positions must be [B or 1, L, number of axes]")
    D = x.shape[3]
    require(D % 2 == 0 and 2 <= D <= 256, "the head size must be even, between 2 and 256")
    require(all(d >= 2 and d % 2 == 0 for d in axis_dims) and sum(axis_dims) <= D,
            "axis_dims must be even, at least 2, and add up to at most the head size")
    bases = [float(b) for b in base] if isinstance(base, (tuple, list)) else [float(base)] * n
    require(len(bases) == n and all(b > 0 and math.isfinite(b) for b in bases),
            "base must be one positive number, or one for each axis")
    if positions.stride(2) != 1:
        positions = positions.contiguous()
    args = (positions.detach(), n, (ctypes.c_int * n)(*axis_dims), (ctypes.c_double * n)(*bases),
            bool(interleaved), bool(inverse))
    if wants_grad(x):
        return RotaryAxes.apply(x, *args)
    return _rotate(x, *args)
