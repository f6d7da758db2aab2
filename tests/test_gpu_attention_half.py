"""Cross attention in half precision where its type's few exponents tell: gradients of small
upstream gradients, and weights far below the largest."""

from __future__ import annotations

import pytest
import torch

from token_refs import attention64

pytestmark = pytest.mark.gpu


def draw(dev, B, Lq, Lk, Hq, Hkv, D, seed):
    g = torch.Generator(dev).manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return ((1.5 * n(B, Lq, Hq, D)).half(), n(B, Lk, Hkv, D).half(), n(B, Lk, Hkv, D).half(),
            n(B, Lq, Hq, D))


def gradients(q, k, v, dout, **kw):
    from gs3d_b200.attention import cross_attention

    ins = [t.clone().requires_grad_() for t in (q, k, v)]
    return torch.autograd.grad(cross_attention(*ins, **kw), ins, dout)


def assert_close_in_norm(got, ref, what):
    """Per batch item and head, the norm of the error against the norm of the result: what one rounding
    of the exact result to half costs (measured on it, since small results are subnormal), and
    1.2 x 2^-11 for the products' operands. An operand's rounding is at most 2^-11 of it, 2^-11 /
    sqrt(3) in the mean square; those of P (or dS) and, through delta, of the output add up in the mean
    square too, since their signs are independent."""
    err = (got.double() - ref).square().sum((1, 3)).sqrt()
    size = ref.square().sum((1, 3)).sqrt()
    once = (ref.half().double() - ref).square().sum((1, 3)).sqrt()
    assert bool(torch.isfinite(got.float()).all()), what
    over = err - once - 1.2 * 2.0 ** -11 * size
    assert bool((over <= 0).all()), (what, (err / size).tolist(), (once / size).tolist())


SIZES = [(1, 999, 3600, 4, 2, 64), (2, 300, 2000, 4, 4, 128), (1, 2000, 260, 6, 3, 80),
         (2, 37, 5000, 8, 2, 64)]


@pytest.mark.parametrize("deviation", (1.0, 1e-2, 1e-3, 1e-4))
@pytest.mark.parametrize("size", SIZES)
def test_gradients_of_small_upstream_gradients(cuda_device, size, deviation):
    """dS is about P dO, which lies among half's subnormals long before dO or the results do."""
    q, k, v, g = draw(cuda_device, *size, seed=21)
    g = (g * deviation).half()
    ref = attention64(q, k, v, dout=g)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, g)):
        assert_close_in_norm(got, ref[name][0], name)


def test_items_and_heads_of_different_magnitudes(cuda_device):
    """Each item's and key head's gradients keep their own precision, with lengths and a mask that hide
    NaN, infinities and the type's lowest number."""
    B, Lq, Lk, Hq, Hkv, D = 3, 150, 1500, 4, 2, 64
    q, k, v, g = draw(cuda_device, B, Lq, Lk, Hq, Hkv, D, seed=22)
    size = torch.tensor([[1.0, 1e-3], [1e-4, 30.0], [1e-3, 1e-2]], device=cuda_device)
    g = (g.view(B, Lq, Hkv, 2, D) * size[:, None, :, None, None]).view(B, Lq, Hq, D).half()
    lengths = torch.tensor([1500, 1100, 700], dtype=torch.int32, device=cuda_device)
    mask = torch.rand(B, 1, 1, Lk, device=cuda_device,
                      generator=torch.Generator(cuda_device).manual_seed(3)) < 0.7
    ref = attention64(q, k, v, lengths, mask, dout=g)
    hidden = ~mask[:, 0, 0] | (torch.arange(Lk, device=cuda_device) >= lengths[:, None])
    for bad in (float("nan"), float("inf"), torch.finfo(torch.float16).min):
        k2, v2 = k.clone(), v.clone()
        k2[hidden], v2[hidden] = bad, bad
        for name, got in zip(("dq", "dk", "dv"),
                             gradients(q, k2, v2, g, lengths=lengths, mask=mask)):
            assert_close_in_norm(got, ref[name][0], (name, bad))


def test_upstream_gradients_of_any_size_stay_finite(cuda_device):
    q, k, v, g = draw(cuda_device, 1, 140, 300, 2, 1, 64, seed=23)
    for size in (0.0, 6e-8, 100.0, 3000.0):
        ref = attention64(q, k, v, dout=(g * size).half())
        for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, (g * size).half())):
            if size > 1.0:
                assert_close_in_norm(got, ref[name][0], (name, size))
            assert bool(torch.isfinite(got).all())
    # one row much larger than the others, and values that no gradient reaches
    g = g.half()
    g[0, 5] = 2000.0
    ref = attention64(q, k, v, dout=g)
    for name, got in zip(("dq", "dk", "dv"), gradients(q, k, v, g)):
        assert_close_in_norm(got, ref[name][0], name)


@pytest.mark.parametrize("Lq,Hq,Hkv,D", [(1, 2, 2, 64), (1, 4, 1, 128), (12, 1, 1, 64), (40, 4, 2, 64),
                                         (130, 2, 2, 64), (300, 1, 1, 128)])
@pytest.mark.parametrize("at", (0, 30000, 60000))
def test_many_keys_of_little_weight(cuda_device, Lq, Hq, Hkv, D, at):
    """One key has nearly all the weight, 60,000 others 2^-25.3 of it each: together 1.5e-3 of the sum,
    and all of the result, since the values are 0 at the one and 1 at the others. The weights are
    rounded to half at 2^7 times their size or more (the largest is 2^8, and half ends at 2^16), where
    half's steps are 2^-24: an error of at most 2^-32 each."""
    from gs3d_b200.attention import cross_attention

    Lk, dev = 60001, cuda_device
    q = torch.zeros(1, Lq, Hq, D, device=dev).half()
    k, v = (torch.zeros(1, Lk, Hkv, D, device=dev).half() for _ in range(2))
    q[..., 0], k[..., 0], v[:] = 1.0, -17.54, 1.0
    k[:, at], v[:, at] = 0.0, 0.0
    out, lse = cross_attention(q, k, v, scale=1.0, return_lse=True)
    w = 60000 * torch.exp(k[0, (at + 1) % Lk, 0, 0].double())
    ref = float(w / (1.0 + w))
    worst = float((out.double() - ref).abs().max())
    assert worst <= 60000 * 2.0 ** -32 + 2.0 ** -10 * ref, (worst, ref)
    assert float((lse.double() - torch.log1p(w)).abs().max()) <= 2.0 ** -18


def test_many_keys_of_little_weight_in_one_piece(cuda_device):
    """The same where one CTA takes all keys of a key head: many items that share their keys."""
    from gs3d_b200.attention import cross_attention

    B, Lk, D, dev = 500, 20000, 64, cuda_device
    q = torch.zeros(B, 1, 1, D, device=dev).half()
    k, v = (torch.zeros(1, Lk, 1, D, device=dev).half() for _ in range(2))
    q[..., 0], k[..., 0], v[:] = 1.0, -17.54, 1.0
    k[:, 0], v[:, 0] = 0.0, 0.0
    out = cross_attention(q, k.expand(B, Lk, 1, D), v.expand(B, Lk, 1, D), scale=1.0)
    w = (Lk - 1) * torch.exp(k[0, 1, 0, 0].double())
    ref = float(w / (1.0 + w))
    worst = float((out.double() - ref).abs().max())
    assert worst <= Lk * 2.0 ** -32 + 2.0 ** -10 * ref, (worst, ref)
