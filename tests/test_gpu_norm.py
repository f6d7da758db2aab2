"""Root-mean-square norm with the residual's addition, its gradient and its 8-bit output against
64-bit plain forms.

Tolerances: the sum of squares is a chain of at most 32 additions a thread and a tree above it, all
of one sign, so rstd is within 2^-19 of the exact one (half of 45 roundings of 2^-24 and the
reciprocal root's own), and the two products add two roundings; a result is rounded once to its
type. A sum over rows of n products has n roundings of 2^-24 against the sum of magnitudes."""

from __future__ import annotations

import pytest
import torch

from token_refs import ROUND, STEP, assert_within, norm64, norm_backward64

pytestmark = pytest.mark.gpu
TYPES = (torch.float32, torch.float16, torch.bfloat16)
REL = 2.0 ** -18


def draw(rows, width, dtype, dev, residual, seed=0):
    g = torch.Generator(dev).manual_seed(seed + rows * 7 + width)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x, r = n(rows, width).to(dtype), (3 * n(rows, width)).to(dtype) if residual else None
    return x, (1 + 0.2 * n(width)).to(dtype), r, n(rows, width).to(dtype), n(rows, width).to(dtype)


SIZES = [(1, 1), (1, 7), (3, 768), (130, 1000), (5, 1023), (2, 1024), (4, 1025), (3, 4096),
         (2, 5000), (3, 6001), (2, 32768), (1, 32767), (2500, 96)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("rows,width", SIZES)
def test_forward_and_gradient(cuda_device, dtype, residual, rows, width):
    from gs3d_b200.norm import rms_norm

    x, w, r, dy, dh = draw(rows, width, dtype, cuda_device, residual)
    y64, h64, _ = norm64(x, w, r, 1e-6)
    plain = rms_norm(x, w, residual=r)
    y, h = plain if residual else (plain, x)
    rnd = ROUND[dtype]
    assert_within(y, y64, (REL + rnd) * y64.abs() * 1.01 + STEP[dtype], "y")
    assert_within(h, h64, (2.0 ** -23 + rnd) * h64.abs() + STEP[dtype], "h")
    ins = [t.clone().requires_grad_() for t in ((x, w, r) if residual else (x, w))]
    out = rms_norm(*ins[:2], residual=ins[2] if residual else None)
    if residual:
        assert torch.equal(out[0], y) and torch.equal(out[1], h)
        dx, dw, dr = torch.autograd.grad(out, ins, (dy, dh))
        assert torch.equal(dx, dr)
    else:
        dx, dw = torch.autograd.grad(out, ins, dy)
    dx64, dw64 = norm_backward64(dy, dh if residual else None, h, w, 1e-6)
    _, _, rstd = norm64(h, w, None, 1e-6)
    u = h.double() * rstd
    g = (dy.double() * w.double()).abs()
    # rstd comes from the unrounded h: a relative error of the mean of h's roundings
    rel = REL + (2 * rnd if residual else 0.0)
    part = rstd * (g + 3 * u.abs() * (g * u.abs()).mean(-1, keepdim=True))
    base = rel * part + rnd * dx64.abs() * 1.01 + STEP[dtype]
    if residual:
        base = base + 2.0 ** -23 * dh.double().abs()
    assert_within(dx, dx64, base, "dx")
    mag = (dy.double() * u).abs().sum(0)
    assert_within(dw, dw64, (rel + rows * 2.0 ** -24) * mag + rnd * dw64.abs() * 1.01 +
                  STEP[dtype], "dw")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("group", (0, 128))
@pytest.mark.parametrize("residual", (False, True))
@pytest.mark.parametrize("rows,width", [(1, 128), (33, 768), (7, 1000), (5, 1024), (2, 1100),
                                        (3, 4096), (2, 32768), (300, 256)])
def test_8bit(cuda_device, dtype, group, residual, rows, width):
    from gs3d_b200.norm import rms_norm_8bit

    if group and width % group:
        pytest.skip("the group has to divide the width")
    x, w, r, _, _ = draw(rows, width, dtype, cuda_device, residual, 3)
    y64, h64, _ = norm64(x, w, r, 1e-6)
    out = rms_norm_8bit(x, w, residual=r, group=group)
    q, s = out[0], out[1]
    n = group or width
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert s.shape == (rows, width // n)
    s64 = y64.view(rows, -1, n).abs().amax(-1) / 448.0
    assert_within(s, s64, 2 * REL * s64, "scales")
    sv = s64.repeat_interleave(n, -1)
    back = q.double() * s.double().repeat_interleave(n, -1)
    # e4m3: 4 bits of precision, the smallest step 2^-9; ties may go either way
    assert_within(back, y64, y64.abs() * (2.0 ** -4 + 4 * REL) + sv * 2.0 ** -10 * 1.01, "q s")
    assert float(q.float().abs().amax()) == 448.0
    if residual:
        assert_within(out[2], h64, (2.0 ** -23 + ROUND[dtype]) * h64.abs() + STEP[dtype], "h")


def test_zero_rows_and_nan(cuda_device):
    from gs3d_b200.norm import rms_norm, rms_norm_8bit

    x = torch.zeros(4, 256, device=cuda_device)
    x[1] = torch.randn(256, device=cuda_device)
    x[2, 5] = float("nan")
    x[3, 130] = float("inf")
    w = torch.ones(256, device=cuda_device)
    y = rms_norm(x, w)
    assert not y[0].any() and torch.isfinite(y[1]).all() and y[2].isnan().all()
    q, s = rms_norm_8bit(x, w, group=128)
    assert not q[0].float().any() and not s[0].any()
    assert torch.isfinite(q[1].float()).all()
    assert s[2].isnan().all() and q[2].float().isnan().all()
    y = rms_norm(x, w, eps=0.0)
    assert y[0].isnan().all()  # 0 / 0, as the formula has it


def test_shapes_strides_and_empty(cuda_device):
    from gs3d_b200.norm import rms_norm, rms_norm_8bit

    big = torch.randn(3, 5, 2, 260, device=cuda_device)
    w = torch.randn(256, device=cuda_device)
    for x in (big[:, :, 1, :256], big[..., 1:257], big.permute(1, 0, 2, 3)[..., :256],
              big[0, 0, 0, 3:259]):
        y64, _, _ = norm64(x, w, None, 1e-6)
        assert_within(rms_norm(x, w), y64, REL * y64.abs(), "strided")
        q, s = rms_norm_8bit(x, w, group=128)
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], 2)
    # a contiguous tensor that does not start on a 16-byte boundary
    x = torch.randn(1025, device=cuda_device)[1:].view(4, 256)
    y64, _, _ = norm64(x, w, None, 1e-6)
    assert_within(rms_norm(x, w), y64, REL * y64.abs(), "misaligned")
    q, s = rms_norm_8bit(x, w, group=128)
    assert_within(q.double() * s.double().repeat_interleave(128, -1), y64,
                  y64.abs() * (2.0 ** -4 + 4 * REL) + s.double().amax() * 2.0 ** -10, "misaligned")
    e = torch.zeros(0, 256, device=cuda_device, requires_grad=True)
    we = w.clone().requires_grad_()
    ye = rms_norm(e, we)
    de, dwe = torch.autograd.grad(ye, (e, we), torch.zeros_like(ye))
    assert de.shape == (0, 256) and not dwe.any()


def test_gradient_matches_differences_and_repeats(cuda_device):
    from gs3d_b200.norm import rms_norm

    x, w, r, dy, dh = draw(37, 200, torch.float32, cuda_device, True, 9)
    ins = [t.clone().requires_grad_() for t in (x, w, r)]

    def loss64(a, b, c):
        y, h, _ = norm64(a, b, c, 1e-6)
        return float((y * dy.double()).sum() + (h * dh.double()).sum())

    grads = torch.autograd.grad(rms_norm(ins[0], ins[1], residual=ins[2]), ins, (dy, dh))
    again = torch.autograd.grad(rms_norm(ins[0], ins[1], residual=ins[2]), ins, (dy, dh))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    step = 1e-5
    for i, got in enumerate(grads):
        d = torch.randn_like(ins[i]).double()
        at = [t.double() for t in (x, w, r)]
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + step * d, at[i] - step * d
        want = (loss64(*plus) - loss64(*minus)) / (2 * step)
        scale = float((got.double() * d).abs().sum())
        # the difference's own error is step^2; the kernel's 2^-18 of each term
        assert abs(float((got.double() * d).sum()) - want) < (2.0 ** -17 + 1e-7) * scale


def test_only_one_output_used(cuda_device):
    from gs3d_b200.norm import rms_norm

    x, w, r, dy, _ = draw(6, 64, torch.float32, cuda_device, True)
    ins = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = rms_norm(ins[0], ins[1], residual=ins[2])
    (dx,) = torch.autograd.grad(h, (ins[0],), dy, retain_graph=True)
    assert torch.equal(dx, dy)
    dx, dr = torch.autograd.grad(y, (ins[0], ins[2]), dy)
    ref, _ = norm_backward64(dy, None, h.detach(), w, 1e-6)
    torch.testing.assert_close(dx.double(), ref, rtol=1e-4, atol=1e-5)
    assert torch.equal(dx, dr)


@pytest.mark.parametrize("group", (0, 128))
def test_8bit_rows_of_tiny_numbers(cuda_device, group):
    """max|y| / 448 below the smallest normal number, whose reciprocal would be infinite."""
    from gs3d_b200.norm import rms_norm_8bit

    x = torch.randn(3, 256, device=cuda_device)
    x[:, ::3] = 0.0
    w = torch.full((256,), 2.0 ** -124, device=cuda_device)
    q, s = rms_norm_8bit(x, w, group=group)
    assert bool((s >= 2.0 ** -126).all())
    assert not q.float().isnan().any() and not q.float()[:, ::3].any()
    y = (x.double() * torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-6)) * w.double()
    got = (q.double().view(3, -1, 256 if group == 0 else 128) * s.double().unsqueeze(-1)).view(3, 256)
    # 4 bits of precision: half a step of 2^-3 relative, or of 2^-9 of the scale near zero
    assert bool(((got - y).abs() <= y.abs() * (2.0 ** -4 + 2.0 ** -18)
                 + 2.0 ** -10 * s.double().amax(-1, keepdim=True)).all())


def test_no_second_derivative(cuda_device):
    from gs3d_b200.norm import rms_norm

    x = torch.randn(4, 64, device=cuda_device, requires_grad=True)
    w = torch.ones(64, device=cuda_device, requires_grad=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(rms_norm(x, w).sum(), x, create_graph=True)
