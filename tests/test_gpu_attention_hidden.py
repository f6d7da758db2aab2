"""What lies at keys that no query keeps, and at queries that keep no key, never reaches a result of
cross attention: NaN, infinities and the type's lowest number there, under every kind of mask."""

from __future__ import annotations

import pytest
import torch

from token_refs import assert_within, attention64

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)
SIZES = [(2, 1, 300, 8, 2, 64), (2, 3, 1030, 4, 4, 128), (1, 2, 6000, 8, 2, 128), (2, 5, 900, 6, 2, 64),
         (2, 150, 261, 4, 2, 64), (1, 260, 391, 4, 2, 128), (2, 70, 1500, 4, 1, 80),
         (1, 2100, 333, 2, 2, 64), (2, 12, 1000, 16, 2, 96)]


def draw(dev, dtype, B, Lq, Lk, Hq, Hkv, D, seed):
    g = torch.Generator(dev).manual_seed(seed + 31 * Lq + 7 * Lk + D)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return ((1.5 * n(B, Lq, Hq, D)).to(dtype), n(B, Lk, Hkv, D).to(dtype), n(B, Lk, Hkv, D).to(dtype),
            n(B, Lq, Hq, D).to(dtype))


def draw_mask(dev, kind, B, Lq, Lk, Hq, seed):
    g = torch.Generator(dev).manual_seed(seed)
    u = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    shape = {"key": (B, 1, 1, Lk), "query": (B, 1, Lq, Lk), "shared": (1, 1, Lq, Lk),
             "head": (B, Hq, 1, Lk), "full": (B, Hq, Lq, Lk)}[kind]
    return u(*shape) < 0.6


def check(q, k, v, g, mask, lengths, dirty):
    """Results on the dirty inputs against the 64-bit form on the clean ones."""
    from gs3d_b200.attention import cross_attention

    ref = attention64(q, k, v, lengths, mask, dout=g)
    ins = [t.clone().requires_grad_() for t in dirty[:3]]
    out, lse = cross_attention(*ins, lengths=lengths, mask=mask, return_lse=True)
    assert_within(out.detach(), *ref["out"], "out")
    assert torch.equal(lse == -torch.inf, ref["lse"] == -torch.inf)
    for name, got in zip(("dq", "dk", "dv"), torch.autograd.grad(out, ins, dirty[3])):
        assert_within(got, *ref[name], name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ("key", "query", "shared", "head", "full"))
@pytest.mark.parametrize("size", SIZES)
def test_keys_that_no_query_keeps(cuda_device, dtype, kind, size):
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=41)
    mask = draw_mask(cuda_device, kind, B, Lq, Lk, Hq, 42)
    mask[..., :Lk // 3] &= torch.rand(Lk // 3, device=cuda_device) < 0.5  # some for nobody
    mask[..., Lk - 40:Lk - 3] = False
    # per item and key head: does any query of any head that shares it keep the key
    any_row = mask.expand(B, Hq, Lq, Lk).view(B, Hkv, Hq // Hkv, Lq, Lk).any(3).any(2)
    lengths = torch.tensor([Lk - 7 * b for b in range(B)], dtype=torch.int32, device=cuda_device)
    hidden = ~any_row | (torch.arange(Lk, device=cuda_device) >= lengths[:, None, None])
    hidden = hidden.transpose(1, 2)  # [B, Lk, Hkv]
    k2, v2 = k.clone(), v.clone()
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(dtype).min)):
        at = hidden & (torch.arange(Lk, device=cuda_device) % 4 == i)[None, :, None]
        k2[at], v2[at] = bad, bad
    assert not torch.isfinite(k2.float()).all()
    check(q, k, v, g, mask, lengths, (q, k2, v2, g))


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_head_leaves_out_what_another_keeps(cuda_device, dtype):
    for size in ((1, 3, 500, 4, 2, 64), (2, 140, 300, 4, 2, 64), (1, 20, 700, 4, 2, 128)):
        B, Lq, Lk, Hq, Hkv, D = size
        q, k, v, g = draw(cuda_device, dtype, *size, seed=43)
        mask = draw_mask(cuda_device, "head", B, Lq, Lk, Hq, 44)
        mask[:, :2, :, 100:200] = False  # both heads of the first key head
        k2, v2 = k.clone(), v.clone()
        k2[:, 100:200, 0], v2[:, 100:200, 0] = float("nan"), float("inf")
        check(q, k, v, g, mask, None, (q, k2, v2, g))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ("query", "shared", "full"))
@pytest.mark.parametrize("size", SIZES)
def test_queries_that_keep_no_key(cuda_device, dtype, kind, size):
    """They have no gradient and give none, whatever they and their upstream gradients hold."""
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=45)
    mask = draw_mask(cuda_device, kind, B, Lq, Lk, Hq, 46)
    mask[:, :, ::3] = False
    if kind == "full":
        mask[:, Hq - 1, -1] = False
    dead = ~mask.expand(B, Hq, Lq, Lk).any(3).transpose(1, 2)  # [B, Lq, Hq]
    assert dead.any()
    q, g = q.masked_fill(dead[..., None], 0.0), g.masked_fill(dead[..., None], 0.0)
    q2, g2 = q.clone(), g.clone()
    for i, bad in enumerate((float("nan"), float("inf"), torch.finfo(dtype).min)):
        at = dead & (torch.arange(Lq, device=cuda_device) // 3 % 3 == i)[None, :, None]
        q2[at], g2[at] = bad, bad
    check(q, k, v, g, mask, None, (q2, k, v, g2))


def test_no_queries_under_a_mask(cuda_device):
    """At the C entry point, where a mask of queries without queries may be given: dk and dv are 0."""
    import ctypes

    from custom_rasterizer_cuda import _lib

    k, v, dk, dv = (torch.randn(1, 5, 1, 64, device=cuda_device).half() for _ in range(4))
    mask = torch.ones(5, dtype=torch.bool, device=cuda_device)
    view = lambda t: _lib.TokenView(t.data_ptr() if t is not None else None, 320, 64, 64)  # noqa: E731
    a = _lib.AttentionArgs(_lib.GS_FP16, 1, 0, 5, 1, 1, 64, 0.125, view(None), view(k), view(v),
                           view(None), None, mask.data_ptr(), 0, 0, 5, None)
    none, vk, vv = view(None), view(dk), view(dv)
    p = [ctypes.addressof(x) for x in (a, none, none, vk, vv)]
    size = _lib.lib.gs_cross_attention_backward_workspace_size(p[0])
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=cuda_device)
    stream = torch.cuda.current_stream().cuda_stream
    status = _lib.lib.gs_cross_attention_backward(*p, ws.data_ptr(), size, stream)
    assert status == _lib.GS_OK, _lib.lib.gs_last_error()
    torch.cuda.synchronize()
    assert not dk.any() and not dv.any()
