"""Rotary positions with several axes, as one autograd op over gs_rotary_axes.

`rotary_axes(x, positions, axis_dims)` turns pairs of each head's numbers by angles that grow with
the token's coordinates, one block of numbers for each axis: for images and video (view or time,
row, column). Image tokens sit at whole coordinates (int32), Gaussians at those of their projected
means (float32).
"""

from __future__ import annotations

import torch

from ._tokens import native


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, axis_dims, base=10000.0,
                interleaved: bool = False, inverse: bool = False) -> torch.Tensor:
    """x[B, L, H, D] (float32, float16 or bfloat16) turned by positions[B or 1, L, axes] (int32 or
    float32). `axis_dims` gives the (even) number of a head's numbers that each axis owns, from
    the first on; what is left over is copied. Pair j of an axis with d numbers turns by
    position * base^(-2 j / d); pairs are (j, j + d / 2) of the axis's block, or neighbours when
    `interleaved`. `base` is one number or one for each axis. `inverse` turns back. Differentiable in
    x, forward mode included; the positions count as constants in both modes."""
    bases = base if isinstance(base, (tuple, list)) else (base,) * len(axis_dims)
    return native.rotary_axes(x, positions, axis_dims, bases, interleaved, inverse)
