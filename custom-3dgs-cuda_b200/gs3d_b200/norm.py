"""Root-mean-square norm with the residual's addition (gs_rms_norm_forward / _backward) and its
8-bit output for the next product (gs_rms_norm_e4m3)."""

from __future__ import annotations

import torch

from ._tokens import native


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
             eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last axis (at most 32,768 elements), with
    h = x + residual where a residual is given: then (y, h) is returned, h being the new residual
    stream, else y alone. float32, float16 or bfloat16, all of one type. First derivatives
    backwards only: a tangent (forward mode) is refused."""
    return native.rms_norm(x, weight, residual, eps)


def rms_norm_8bit(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                  eps: float = 1e-6, group: int = 0):
    """rms_norm whose y is written in 8 bits: (q, scales), or (q, scales, h) with a residual, with
    q (float8_e4m3fn, x's shape) times its scale near y and scales = max|y| / 448 of each row
    ([..., 1]) or, with `group` 128, of each 128 numbers ([..., width / 128]). For prediction:
    no gradient."""
    return native.rms_norm_8bit(x, weight, residual, eps, group)
