"""The Gaussian decoder on the token operators: it trains through the rasterizer, its operators
agree with plain torch forms of them, and prediction agrees with the training path."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_view_tokens_and_positions(cuda_device):
    from gs3d_b200 import decoder, scenes

    images = torch.arange(2 * 20 * 33 * 3, device=cuda_device, dtype=torch.float32)
    images = images.view(2, 20, 33, 3)
    x, at = decoder.view_tokens(images)
    assert x.shape == (1, 2 * 2 * 3, 768) and at.shape == (1, 12, 3) and at.dtype == torch.int32
    assert at[0, 5].tolist() == [0, 1, 2] and at[0, 6].tolist() == [1, 0, 0]
    tile = x[0, 5].view(16, 16, 3)  # rows 16..19, column 32
    assert torch.equal(tile[:4, :1], images[0, 16:20, 32:33]) and not tile[4:].any()
    v = scenes.pinhole((0.0, 0.0, 4.0), 128, 64, 100.0)
    mu = torch.tensor([[0.0, 0.0, 0.0], [0.0, 0.0, 9.0]], device=cuda_device)
    p = decoder.gaussian_positions(mu, v)[0]
    # both at the image's centre: one looked at, one behind the camera
    torch.testing.assert_close(p, torch.tensor([[0.0, 2.0, 4.0]] * 2, device=cuda_device))


def test_training_lowers_the_loss_and_prediction_agrees(cuda_device):
    import custom_rasterizer_cuda as crc
    from gs3d_b200 import decoder

    model, losses, (start, positions, images, _) = decoder.train(steps=40, device=cuda_device)
    assert losses[-1] < 0.9 * losses[0]
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all())
               for p in model.parameters())
    with torch.no_grad():
        states = model.encode(images)
        full = model(start, positions, states)
        prepared = model.prepare_8bit()
        answer = model.predict(start, positions, states, prepared)
        moved = (full - start).norm()
        # 8-bit rows and weights: 2^-4 relative each, averaged over 256 numbers of a product
        assert float((answer - full).norm()) < 0.1 * float(moved)
        # one query at a time takes the kernel for single queries
        one = model.predict(start[7:8], positions[:, 7:8], states, prepared)
        assert float((one - answer[7:8]).norm()) < 0.05 * float((answer[7:8] - start[7:8]).norm())
    assert crc.device_error_bits() == 0


def test_operators_inside_agree_with_plain_forms(cuda_device, monkeypatch):
    """The same decoder with torch forms in float32 in the operators' place: outputs and gradients
    within what bfloat16 tokens lose."""
    from gs3d_b200 import decoder

    def plain_rotary(x, at, dims, base):
        B, L, H, D = x.shape
        out = []
        start = 0
        for a, d in enumerate(dims):
            f = base ** (-2.0 * torch.arange(d // 2, device=x.device) / d)
            ang = (at[..., a].float()[..., None] * f)[:, :, None]
            u, v = x[..., start:start + d // 2].float(), x[..., start + d // 2:start + d].float()
            out += [u * ang.cos() - v * ang.sin(), u * ang.sin() + v * ang.cos()]
            start += d
        return torch.cat(out + [x[..., start:].float()], -1).to(x.dtype)

    def plain_norm(x, w, residual=None, eps=1e-6):
        h = x.float() + (0 if residual is None else residual.float())
        y = (h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * w.float()).to(x.dtype)
        return y if residual is None else (y, h.to(x.dtype))

    def plain_attention(q, k, v):
        rep = q.shape[2] // k.shape[2]
        qf, kf, vf = (t.float().transpose(1, 2) for t in (q, k, v))
        kf, vf = kf.repeat_interleave(rep, 1), vf.repeat_interleave(rep, 1)
        p = torch.softmax(qf @ kf.transpose(2, 3) * q.shape[3] ** -0.5, -1)
        return (p @ vf).transpose(1, 2).to(q.dtype)

    model, _, (start, positions, images, _) = decoder.train(steps=3, device=cuda_device)
    g = torch.randn_like(start)

    def run():
        model.zero_grad(set_to_none=True)
        out = model(start, positions, model.encode(images))
        (out * g).sum().backward()
        return out.detach() - start, [p.grad.clone() for p in model.parameters()]

    out, grads = run()
    monkeypatch.setattr(decoder, "rotary_axes", plain_rotary)
    monkeypatch.setattr(decoder, "rms_norm", plain_norm)
    monkeypatch.setattr(decoder, "cross_attention", plain_attention)
    ref, ref_grads = run()
    # a dozen roundings of 2^-9 or so on the way, partly correlated between the two
    assert float((out - ref).norm()) < 0.03 * float(ref.norm())
    for got, want in zip(grads, ref_grads):
        assert float((got - want).norm()) < 0.06 * float(want.norm()) + 1e-6
