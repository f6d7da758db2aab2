"""Derivatives of the token operators that do not come from backward: a tangent (forward mode) is
either carried or refused, never dropped, and what cannot see the operators (a trace, vmap) is
told so."""

from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fw

from token_refs import ROUND, assert_within, rotary64


def calls(device, wrap):
    """One call of each operator without a forward-mode form, for each input that could carry a
    tangent, with `wrap` around that input."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm, rms_norm_8bit

    x, r = torch.randn(3, 64, device=device), torch.randn(3, 64, device=device)
    w = torch.ones(64, device=device)
    q, k, v = (torch.randn(1, n, 2, 64, device=device).half() for n in (5, 7, 7))
    for name, f, ins in (("rms_norm", rms_norm, (x, w)), ("rms_norm", rms_norm, (x, w, r)),
                         ("rms_norm_8bit", rms_norm_8bit, (x, w, r)),
                         ("cross_attention", cross_attention, (q, k, v))):
        for i in range(len(ins)):
            def call(f=f, ins=ins, i=i):
                return f(*ins[:i], wrap(ins[i]), *ins[i + 1:])
            yield name, call


def refuses_tangents(device):
    for grad in (True, False):
        with fw.dual_level(), torch.set_grad_enabled(grad):
            for name, call in calls(device, lambda t: fw.make_dual(t, torch.ones_like(t))):
                with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                    call()


def test_tangents_are_refused_before_anything_else():
    refuses_tangents("cpu")


def test_a_trace_is_refused():
    from gs3d_b200.norm import rms_norm, rms_norm_8bit
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.rotary import rotary_axes

    x, w, p = torch.zeros(1, 2, 1, 64), torch.zeros(64), torch.zeros(1, 2, 1)
    for name, f, ins in (("rms_norm", rms_norm, (x, w)), ("rms_norm_8bit", rms_norm_8bit, (x, w)),
                         ("cross_attention", cross_attention, (x, x, x)),
                         ("rotary_axes", lambda a, b: rotary_axes(a, b, (64,)), (x, p))):
        with pytest.raises(RuntimeError, match=f"{name} cannot be traced"):
            torch.jit.trace(f, ins, check_trace=False)


@pytest.mark.gpu
def test_tangents_are_refused(cuda_device):
    refuses_tangents(cuda_device)
    # without a tangent, or where they are switched off, the calls go through
    for _, call in calls(cuda_device, lambda t: t):
        call()
    with fw.dual_level():
        for _, call in calls(cuda_device, lambda t: t):
            call()
    with torch.inference_mode():
        for _, call in calls(cuda_device, lambda t: t):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16, torch.bfloat16))
@pytest.mark.parametrize("interleaved,inverse", ((False, False), (True, False), (False, True)))
def test_rotary_turns_the_tangent(cuda_device, dtype, interleaved, inverse):
    """The map is linear: its tangent is the rotation of the tangent, whether or not x also wants a
    gradient, and that rotation differentiates in turn."""
    from gs3d_b200.rotary import rotary_axes

    x = torch.randn(2, 13, 3, 40, device=cuda_device).to(dtype)
    t = torch.randn(2, 13, 3, 40, device=cuda_device).to(dtype)
    pos = torch.rand(2, 13, 2, device=cuda_device) * 60
    kw = dict(base=100.0, interleaved=interleaved, inverse=inverse)
    plain = rotary_axes(x, pos, (16, 20), **kw)
    ref, mag = rotary64(t, pos, (16, 20), (100.0, 100.0), interleaved, inverse)
    for grad in (False, True):
        xi, ti = x.clone().requires_grad_(grad), t.clone().requires_grad_(grad)
        with fw.dual_level():
            y, dy = fw.unpack_dual(rotary_axes(fw.make_dual(xi, ti), pos, (16, 20), **kw))
            assert torch.equal(y, plain) and dy is not None
            # the bound of the rotation itself (tests/test_gpu_rotary.py)
            assert_within(dy.detach(), ref, 2.0 ** -21 * mag + ROUND[dtype] * 1.01 * ref.abs()
                          + 2.0 ** -133, "tangent")
            if grad:
                g = torch.randn_like(y)
                (dx,) = torch.autograd.grad(y, xi, g, retain_graph=True)
                (dt,) = torch.autograd.grad(dy, ti, g)
                back = rotary_axes(g, pos, (16, 20), **{**kw, "inverse": not inverse})
                assert torch.equal(dx, back) and torch.equal(dt, back)


@pytest.mark.gpu
def test_tangents_of_upstream_gradients(cuda_device):
    """Forward over backward: a tangent may first appear in the upstream gradient."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm
    from gs3d_b200.rotary import rotary_axes

    x = torch.randn(1, 5, 2, 64, device=cuda_device).half().requires_grad_()
    w = torch.ones(64, device=cuda_device).half()
    pos = torch.rand(1, 5, 1, device=cuda_device) * 60
    g, t = torch.randn_like(x).detach(), torch.randn_like(x).detach()
    with fw.dual_level():
        for name, y in (("rms_norm", rms_norm(x, w)), ("rms_norm", rms_norm(x, w, residual=x)[0]),
                        ("cross_attention", cross_attention(x, x, x))):
            with pytest.raises(RuntimeError, match=f"{name}'s gradient has no forward-mode"):
                torch.autograd.grad(y, x, fw.make_dual(g, t))
        y = rotary_axes(x, pos, (64,))
        dx, dt = fw.unpack_dual(torch.autograd.grad(y, x, fw.make_dual(g, t))[0])
        assert torch.equal(dx, rotary_axes(g, pos, (64,), inverse=True))
        assert torch.equal(dt, rotary_axes(t, pos, (64,), inverse=True))


@pytest.mark.gpu
def test_functional_transforms_are_refused(cuda_device):
    """vmap and torch.func.jvp hand over tensors without memory of their own: an error, no answer."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm
    from gs3d_b200.rotary import rotary_axes

    x, w = torch.randn(4, 3, 64, device=cuda_device), torch.ones(64, device=cuda_device)
    q = torch.randn(4, 1, 3, 2, 64, device=cuda_device).half()
    p = torch.zeros(1, 3, 1, device=cuda_device)
    for f, ins in ((lambda a: rms_norm(a, w), x), (lambda a: cross_attention(a, a, a), q),
                   (lambda a: rotary_axes(a, p, (64,)), q)):
        with pytest.raises(RuntimeError):
            torch.vmap(f)(ins)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (ins[0],), (torch.ones_like(ins[0]),))
