"""Cross attention of Gaussian (or other) query tokens to an encoder's states of another length,
as one autograd op over gs_cross_attention_forward / gs_cross_attention_backward."""

from __future__ import annotations

import torch

from ._tokens import native


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                    scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v for q[B, Lq, Hq, D] and k, v[B, Lk, Hkv, D] of float16 or bfloat16,
    D a multiple of 8 up to 128, Hq a multiple of Hkv (neighbouring query heads share a key head).
    `lengths` (int32 [B]): the keys of each batch item; later ones are not looked at. `mask` (bool,
    [B or 1, Hq or 1, Lq or 1, Lk]): False leaves a key out. A query that keeps no key gives zeros and
    takes no part in the gradients, whatever it holds.
    `scale` is 1 / sqrt(D) unless given. With `return_lse`, (out, lse[B, Hq, Lq] float32): log sum
    exp of the scaled scores, -inf for a query without keys; no gradient flows through it. First
    derivatives backwards only: a tangent (forward mode) is refused.

    Tensors whose last axis is contiguous are used in place, whatever the other strides, if address
    and strides are multiples of 16 bytes; others are copied first. What k and v hold at a key that no
    query of its batch item keeps, of none of the heads that share it, never reaches a result, NaN
    included. Where some of them keep a key and others do not, v must be finite there; gradients need
    a finite k at every key that is kept."""
    return native.cross_attention(q, k, v, lengths, mask, scale, return_lse)
