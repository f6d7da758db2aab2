"""Cross attention of Gaussian (or other) query tokens to an encoder's states of another length,
as one autograd op over gs_cross_attention_forward / gs_cross_attention_backward."""

from __future__ import annotations

import ctypes
import math

import torch

from custom_rasterizer_cuda import _lib

from ._tokens import (DTYPES, check_tokens, on_device, require, stream, usable, view4,
                      wants_grad)


def _args(q, k, v, lengths, mask, scale, out, lse):
    B, Lq, Hq, D = q.shape
    a = _lib.AttentionArgs(DTYPES[q.dtype], B, Lq, k.shape[1], Hq, k.shape[2], D, scale, view4(q),
                           view4(k), view4(v), view4(out),
                           None if lengths is None else lengths.data_ptr())
    if mask is not None and mask.numel():
        a.mask = mask.data_ptr()
        a.mask_batch_stride, a.mask_head_stride, a.mask_query_stride = (
            0 if n == 1 else s for n, s in zip(mask.shape[:3], mask.stride()[:3]))
    a.lse = None if lse is None else lse.data_ptr()
    return a


def _forward(q, k, v, lengths, mask, scale, want_lse):
    B, Lq, Hq, D = q.shape
    dev = q.device
    out = torch.empty((B, Lq, Hq, D), device=dev, dtype=q.dtype)
    lse = torch.empty((B, Hq, Lq), device=dev, dtype=torch.float32) if want_lse else None
    if out.numel() == 0:
        return out, lse
    a = _args(q, k, v, lengths, mask, scale, out, lse)
    with on_device(dev):
        ws_bytes = _lib.lib.gs_cross_attention_workspace_size(ctypes.addressof(a))
        ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8) if ws_bytes else None
        _lib.check(_lib.lib.gs_cross_attention_forward(
            ctypes.addressof(a), None if ws is None else ws.data_ptr(), ws_bytes, stream(dev)))
    return out, lse


class CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, mask, scale):
        out, lse = _forward(q, k, v, lengths, mask, scale, True)
        ctx.save_for_backward(q, k, v, lengths, mask, out, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    def backward(ctx, dout, _):
        q, k, v, lengths, mask, out, lse = ctx.saved_tensors
        dev = q.device
        dout = usable(dout, 8)
        dq, dk, dv = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k, v))
        a = _args(q, k, v, lengths, mask, ctx.scale, out, lse)
        views = [view4(t) for t in (dout, dq, dk, dv)]
        with on_device(dev):
            ws_bytes = _lib.lib.gs_cross_attention_backward_workspace_size(ctypes.addressof(a))
            ws = torch.empty(ws_bytes, device=dev, dtype=torch.uint8)
            _lib.check(_lib.lib.gs_cross_attention_backward(
                ctypes.addressof(a), *(ctypes.addressof(t) for t in views),
                ws.data_ptr() if ws_bytes else None, ws_bytes, stream(dev)))
        return dq, dk, dv, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    lengths: torch.Tensor | None = None, mask: torch.Tensor | None = None,
                    scale: float | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v for q[B, Lq, Hq, D] and k, v[B, Lk, Hkv, D] of float16 or bfloat16,
    D a multiple of 8 up to 128, Hq a multiple of Hkv (neighbouring query heads share a key head).
    `lengths` (int32 [B]): the keys of each batch item; later ones are not looked at. `mask` (bool,
    [B or 1, Hq or 1, Lq or 1, Lk]): False leaves a key out. A query that keeps no key gives zeros.
    `scale` is 1 / sqrt(D) unless given. With `return_lse`, (out, lse[B, Hq, Lq] float32): log sum
    exp of the scaled scores, -inf for a query without keys; no gradient flows through it.

    Tensors whose last axis is contiguous are used in place, whatever the other strides, if address
    and strides are multiples of 16 bytes; others are copied first. Under a mask that differs
    between queries v must be finite everywhere below the lengths."""
    check_tokens(q, "q", 4)
    check_tokens(k, "k", 4)
    check_tokens(v, "v", 4)
    require(q.dtype in (torch.float16, torch.bfloat16), "q must be float16 or bfloat16")
    require(k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v must have the same type")
    require(k.device == q.device and v.device == q.device, "q, k and v must be on one device")
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    require(k.shape == v.shape and k.shape[0] == B and k.shape[3] == D,
            "k and v must be [B, Lk, Hkv, D] with q's B and D")
    require(8 <= D <= 128 and D % 8 == 0, "the head size must be a multiple of 8 up to 128")
    require(Hq == 0 if Hkv == 0 else Hq % Hkv == 0, "the key heads must divide the query heads")
    if lengths is not None:
        require(lengths.is_cuda and lengths.device == q.device and lengths.dtype == torch.int32
                and lengths.shape == (B,), "lengths must be an int32 tensor [B] on q's device")
        lengths = lengths.contiguous()
    if mask is not None:
        require(isinstance(mask, torch.Tensor) and mask.device == q.device
                and mask.dtype == torch.bool and mask.dim() == 4,
                "mask must be a bool tensor of 4 dimensions on q's device")
        require(mask.shape[0] in (1, B) and mask.shape[1] in (1, Hq) and mask.shape[2] in (1, Lq)
                and mask.shape[3] == Lk, "mask must be [B or 1, Hq or 1, Lq or 1, Lk]")
        if Lk > 1 and mask.stride(3) != 1:
            mask = mask.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    require(math.isfinite(scale), "scale must be finite")
    q, k, v = usable(q, 8), usable(k, 8), usable(v, 8)
    if wants_grad(q, k, v):
        out, lse = CrossAttention.apply(q, k, v, lengths, mask, scale)
    else:
        out, lse = _forward(q, k, v, lengths, mask, scale, return_lse)
    return (out, lse) if return_lse else out
