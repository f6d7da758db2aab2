"""What the token operators' Python boundaries share: element types, views and streams."""

from __future__ import annotations

import torch

from custom_rasterizer_cuda import _lib

DTYPES = {torch.float32: _lib.GS_FP32, torch.float16: _lib.GS_FP16, torch.bfloat16: _lib.GS_BF16}


def require(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def check_tokens(t: torch.Tensor, name: str, dims: int) -> None:
    require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    require(t.dim() == dims, f"{name} must have {dims} dimensions")


def usable(t: torch.Tensor, elements: int = 1) -> torch.Tensor:
    """t, or a contiguous copy of it where its last axis is not contiguous, or where its address
    or strides are not multiples of `elements` elements (those of axes of length 1 do not count), or,
    where `elements` is above 1, an axis other than the first repeats itself (a stride of 0)."""
    if t.numel() == 0:
        return t
    if t.data_ptr() % (elements * t.element_size()):
        return t.clone(memory_format=torch.contiguous_format)
    *outer, last = zip(t.shape, t.stride())
    if (last[1] != 1 and last[0] > 1) or any(n > 1 and s % elements for n, s in outer):
        return t.contiguous()
    if elements > 1 and any(n > 1 and s == 0 for n, s in outer[1:]):
        return t.contiguous()
    return t


def view4(t: torch.Tensor) -> _lib.TokenView:
    """The [batch, token, head, D] view of t; the stride of an axis of length 1 counts as 0."""
    s = [0 if n <= 1 else st for n, st in zip(t.shape, t.stride())]
    return _lib.TokenView(t.data_ptr() if t.numel() else None, s[0], s[1], s[2])


class on_device:
    """torch.cuda.device(dev), without its cost where dev is current already."""

    def __init__(self, dev: torch.device):
        self.guard = None
        if dev.index is not None and dev.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(dev)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def stream(dev: torch.device) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
