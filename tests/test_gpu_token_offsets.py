"""Token operators on tensors whose elements lie more than 2^31 (and 2^32) elements or bytes apart, as
in a long cache of keys and values."""

from __future__ import annotations

import pytest
import torch

from token_refs import ROUND, assert_within, attention64, norm64, rotary64

pytestmark = pytest.mark.gpu
FAR = (1 << 32) + 64  # elements


@pytest.fixture
def far(cuda_device):
    """Makes [2, ...] tensors of half whose items lie FAR elements apart in one block of 8.6 GB."""
    block = torch.empty(FAR + (1 << 24), dtype=torch.float16, device=cuda_device)

    def place(t, offset=0):
        assert offset + t[0].numel() <= 1 << 24
        out = block.as_strided(t.shape, (FAR, *t[0].contiguous().stride()), offset)
        out.copy_(t)
        return out

    yield place
    del block
    torch.cuda.empty_cache()


@pytest.mark.parametrize("Lq,Lk,Hq,Hkv,D", [(1, 700, 4, 2, 64), (150, 300, 4, 2, 128)])
def test_attention_over_items_far_apart(cuda_device, far, Lq, Lk, Hq, Hkv, D):
    from gs3d_b200.attention import cross_attention

    g = torch.Generator(cuda_device).manual_seed(81)
    n = lambda *s: torch.randn(*s, generator=g, device=cuda_device).half()  # noqa: E731
    q, k, v, dout = n(2, Lq, Hq, D), n(2, Lk, Hkv, D), n(2, Lk, Hkv, D), n(2, Lq, Hq, D)
    ref = attention64(q, k, v, dout=dout)
    *ins, dout = [far(t, i << 22) for i, t in enumerate((q, k, v, dout))]
    ins = [t.detach().requires_grad_() for t in ins]
    out = cross_attention(*ins)
    assert_within(out.detach(), *ref["out"], "out")
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, ins, dout)):
        assert_within(got, *ref[name], name)


def test_a_key_head_of_many_tokens(cuda_device):
    """One item's keys, 2^31 bytes and more from the first to the last, in both forms."""
    from gs3d_b200.attention import cross_attention

    Lk, H, D = 140_000, 64, 128  # 2.3 GB each
    g = torch.Generator(cuda_device).manual_seed(82)
    k, v = (torch.randn(1, Lk, H, D, generator=g, device=cuda_device, dtype=torch.float16)
            for _ in range(2))
    for Lq in (1, 40):
        q = torch.randn(1, Lq, H, D, generator=g, device=cuda_device, dtype=torch.float16)
        out = cross_attention(q, k, v)
        for h in (0, H - 1):
            one = slice(h, h + 1)
            ref = attention64(q[:, :, one], k[:, :, one], v[:, :, one])
            assert_within(out[:, :, one], *ref["out"], f"head {h}")
    del k, v
    torch.cuda.empty_cache()


def test_rotary_and_norm_far_into_a_tensor(cuda_device, far):
    from gs3d_b200.norm import rms_norm
    from gs3d_b200.rotary import rotary_axes

    g = torch.Generator(cuda_device).manual_seed(83)
    x = torch.randn(2, 50, 3, 64, generator=g, device=cuda_device).half()
    pos = torch.rand(2, 50, 1, generator=g, device=cuda_device) * 40
    y = rotary_axes(far(x), pos, (64,), base=100.0)
    ref, mag = rotary64(x, pos, (64,), (100.0,))
    assert_within(y, ref, 2.0 ** -21 * mag + ROUND[x.dtype] * 1.01 * ref.abs() + 2.0 ** -25, "rotary")
    # 2,200,000 rows of 1,024: the last ones start past 2^31 elements
    rows = 2_200_000
    x = torch.randn(rows, 1024, generator=g, device=cuda_device, dtype=torch.float16)
    w = torch.ones(1024, device=cuda_device).half()
    got = rms_norm(x, w)
    for part in (slice(0, 100), slice(rows - 100, rows)):
        y64, _, _ = norm64(x[part], w, None, 1e-6)
        assert_within(got[part], y64, (2.0 ** -18 + ROUND[x.dtype]) * 1.01 * y64.abs() + 2.0 ** -25,
                      "norm")
    del x, got
    torch.cuda.empty_cache()
