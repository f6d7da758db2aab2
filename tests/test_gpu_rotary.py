"""Rotary positions with several axes against a 64-bit plain form.

Tolerances: the angle is reduced exactly and sin / cos are good to 2^-22 or so, and each output is
two products and a sum in 32 bits, so a number is within 2^-21 (|u| + |v|) of the exact rotation
plus one rounding of its type."""

from __future__ import annotations

import pytest
import torch

from token_refs import ROUND, STEP, assert_within, rotary64

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.float16, torch.bfloat16)


def check(x, pos, dims, base, interleaved, inverse=False):
    from gs3d_b200.rotary import rotary_axes

    y = rotary_axes(x, pos, dims, base=base, interleaved=interleaved, inverse=inverse)
    bases = base if isinstance(base, tuple) else (base,) * len(dims)
    ref, mag = rotary64(x, pos, dims, bases, interleaved, inverse)
    assert y.dtype == x.dtype and y.is_contiguous()
    bound = 2.0 ** -21 * mag + ROUND[x.dtype] * ref.abs() * 1.01 + STEP[x.dtype]
    rest = sum(dims)
    bound[..., rest:] = 0.0  # copied
    assert_within(y, ref, bound, "rotary")
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("B,L,H,D,dims,whole", [
    (1, 1, 1, 2, (2,), True), (4, 1, 16, 64, (16, 24, 24), False),
    (2, 37, 5, 64, (16, 24, 24), True), (1, 300, 12, 96, (24, 36, 36), False),
    (3, 19, 7, 80, (6, 10, 14, 2), False), (2, 5, 3, 128, (32, 48, 48), True),
    (1, 9, 33, 256, (256,), False), (1, 4, 2, 250, (2, 4), True)])
def test_matches_64_bit_rotation(cuda_device, dtype, interleaved, B, L, H, D, dims, whole):
    g = torch.Generator(cuda_device).manual_seed(B * 1000 + L)
    x = torch.randn(B, L, H, D, generator=g, device=cuda_device).to(dtype)
    pos = torch.rand(B, L, len(dims), generator=g, device=cuda_device) * 500 - 100
    pos = pos.to(torch.int32) if whole else pos
    check(x, pos, dims, 100.0, interleaved)
    check(x, pos, dims, tuple(10.0 ** (a + 2) for a in range(len(dims))), interleaved, True)


def test_large_coordinates_keep_their_accuracy(cuda_device):
    x = torch.randn(1, 64, 2, 64, device=cuda_device)
    pos = torch.arange(64, device=cuda_device, dtype=torch.int32).view(1, 64, 1) + (1 << 24) - 64
    check(x, pos, (64,), 10000.0, False)


def test_strides_shared_positions_and_offsets(cuda_device):
    g = torch.Generator(cuda_device).manual_seed(1)
    big = torch.randn(2, 6, 21, 3, 64, generator=g, device=cuda_device).bfloat16()
    pos = torch.rand(1, 21, 2, generator=g, device=cuda_device) * 50
    check(big[:, :, :, 1].transpose(1, 2), pos, (32, 32), 100.0, False)  # [2, 21, 6, 64] strided
    check(big[:, :, :, 1].permute(0, 2, 1, 3)[..., 1:63], pos, (20, 32), 100.0, True)  # odd start
    wide = torch.rand(2, 21, 5, generator=g, device=cuda_device)
    check(big[:, :, :, 0].transpose(1, 2), wide[..., 1:3], (32, 32), 100.0, False)
    check(big[:, :, :, 0].transpose(1, 2), wide[..., ::4], (32, 32), 100.0, False)
    check(big[:1, :1, :, 0].transpose(1, 2).expand(2, 21, 6, 64), pos, (32, 32), 100.0, False)


def test_empty(cuda_device):
    from gs3d_b200.rotary import rotary_axes

    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        x = torch.zeros(shape, device=cuda_device)
        pos = torch.zeros(shape[0], shape[1], 1, device=cuda_device)
        assert rotary_axes(x, pos, (8,)).shape == shape


@pytest.mark.parametrize("interleaved", (False, True))
def test_gradient_is_the_inverse_and_matches_differences(cuda_device, interleaved):
    from gs3d_b200.rotary import rotary_axes

    g = torch.Generator(cuda_device).manual_seed(5)
    x = torch.randn(2, 11, 3, 24, generator=g, device=cuda_device, requires_grad=True)
    pos = torch.rand(2, 11, 3, generator=g, device=cuda_device) * 90
    dy = torch.randn(2, 11, 3, 24, generator=g, device=cuda_device)
    dims = (4, 8, 8)
    y = rotary_axes(x, pos, dims, base=100.0, interleaved=interleaved)
    (dx,) = torch.autograd.grad(y, (x,), dy)
    ref, mag = rotary64(dy, pos, dims, (100.0,) * 3, interleaved, inverse=True)
    assert_within(dx, ref, 2.0 ** -21 * mag + 2.0 ** -24 * ref.abs(), "gradient")
    # the map is linear: a difference along d is exact up to rounding
    d = torch.randn(2, 11, 3, 24, generator=g, device=cuda_device)
    plus, _ = rotary64(x.detach().double() + d, pos, dims, (100.0,) * 3, interleaved)
    minus, _ = rotary64(x.detach().double() - d, pos, dims, (100.0,) * 3, interleaved)
    want = float(((plus - minus) / 2 * dy.double()).sum())
    scale = float((dy.abs() * d.abs()).sum())
    assert abs(float((dx.double() * d.double()).sum()) - want) < 2.0 ** -20 * scale


def test_runs_on_the_current_stream(cuda_device):
    from gs3d_b200.rotary import rotary_axes

    x = torch.randn(1, 4000, 8, 64, device=cuda_device)
    pos = torch.rand(1, 4000, 1, device=cuda_device)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a = x * 2.0
        y = rotary_axes(a, pos, (64,))
    s.synchronize()
    ref, mag = rotary64(x * 2.0, pos, (64,), (10000.0,))
    assert_within(y, ref, 2.0 ** -20 * mag, "other stream")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", (False, True))
@pytest.mark.parametrize("B,L,H,D,dims", [
    (1, 20000, 17, 64, (16, 24, 24)), (1, 9000, 33, 80, (8, 16, 40, 16)),
    (2, 3000, 16, 256, (64, 128)), (1, 160000, 16, 8, (8,)), (1, 20000, 17, 64, (20, 44))])
def test_many_tokens(cuda_device, dtype, interleaved, B, L, H, D, dims):
    """Work enough for 16 heads a thread; heads outside of tokens; NaN and infinities in what no
    axis owns."""
    g = torch.Generator(cuda_device).manual_seed(L + D)
    x = torch.randn(B, H, L, D, generator=g, device=cuda_device).to(dtype).transpose(1, 2)
    pos = torch.randint(-300, 300, (B, L, len(dims)), generator=g, device=cuda_device)
    check(x, pos.to(torch.int32), dims, 100.0, interleaved)
    y = check(x.contiguous(), pos.float() + 0.5, dims, 100.0, interleaved, True)
    if sum(dims) < D:
        bad = x.clone()
        bad[..., sum(dims)::2], bad[..., sum(dims) + 1::2] = float("nan"), float("inf")
        from gs3d_b200.rotary import rotary_axes

        out = rotary_axes(bad, pos.float() + 0.5, dims, base=100.0, interleaved=interleaved,
                          inverse=True)
        assert torch.equal(out[..., :sum(dims)], y[..., :sum(dims)])
        assert torch.equal(out[..., sum(dims):].isnan(), bad[..., sum(dims):].isnan())
