"""What the token operators (rotary positions, norms, cross attention) refuse, before any CUDA
call: status codes at the C entry points, RuntimeErrors in Python."""

from __future__ import annotations

import ctypes

import pytest
import torch

A = 4096  # a well-aligned address that is never looked at


def rotary(L, dtype=0, B=1, n=2, D=8, dims=(4, 4), bases=(10.0, 10.0), ptype=0, views=True):
    from custom_rasterizer_cuda import _lib

    v = ctypes.addressof(_lib.TokenView(A, 8, 8, 8)) if views else None
    return L.gs_rotary_axes(dtype, B, 1, 1, D, v, v, A, ptype, 0, 2, n,
                            (ctypes.c_int * 4)(*dims), (ctypes.c_double * 4)(*bases), 0, 0, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), b"dtype"), (dict(ptype=2), b"positions"), (dict(B=-1), b"sizes"),
    (dict(D=7), b"head size"), (dict(D=258), b"head size"), (dict(n=5), b"axes"),
    (dict(n=0), b"axes"), (dict(dims=(3, 5)), b"even"), (dict(dims=(4, 6)), b"more numbers"),
    (dict(bases=(0.0, 1.0)), b"bases"), (dict(views=False), b"null")])
def test_rotary_refusals(kw, msg):
    from custom_rasterizer_cuda import _lib

    assert rotary(_lib.lib, **kw) == _lib.GS_ERR_INVALID_ARG
    assert msg in _lib.lib.gs_last_error()


def test_rotary_of_nothing_is_a_noop():
    from custom_rasterizer_cuda import _lib

    assert rotary(_lib.lib, B=0) == _lib.GS_OK


def test_norm_refusals():
    from custom_rasterizer_cuda import _lib

    L, bad = _lib.lib, _lib.GS_ERR_INVALID_ARG
    assert L.gs_rms_norm_forward(9, 1, 8, A, None, A, 1e-6, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, -1, 8, A, None, A, 1e-6, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, 1, 0, A, None, A, 1e-6, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, 1, 32769, A, None, A, 1e-6, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, 1, 8, A, None, A, -1.0, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, 1, 8, None, None, A, 1e-6, A, None, None, None) == bad
    assert L.gs_rms_norm_forward(0, 1, 8, A, None, A, 1e-6, A, A, None, None) == bad
    assert b"residual" in L.gs_last_error()
    assert L.gs_rms_norm_forward(0, 0, 8, None, None, None, 1e-6, None, None, None, None) == 0
    assert L.gs_rms_norm_e4m3(0, 1, 256, 64, A, None, A, 1e-6, A, A, None, None) == bad
    assert L.gs_rms_norm_e4m3(0, 1, 200, 128, A, None, A, 1e-6, A, A, None, None) == bad
    assert L.gs_rms_norm_e4m3(0, 1, 256, 128, A + 4, None, A, 1e-6, A, A, None, None) == bad
    assert b"16-byte" in L.gs_last_error()
    need = L.gs_rms_norm_backward_workspace_size(100, 64)
    assert need >= 64 * 4
    assert L.gs_rms_norm_backward_workspace_size(-1, 64) == 0
    assert L.gs_rms_norm_backward(0, 100, 64, A, None, A, A, A, A, A, A, need - 1, None) == bad
    assert b"workspace" in L.gs_last_error()
    assert L.gs_rms_norm_backward(0, 100, 64, A, None, A, A, None, A, A, A, need, None) == bad


def attention_args(**kw):
    from custom_rasterizer_cuda import _lib

    v = lambda: _lib.TokenView(A, 1024, 64, 64)  # noqa: E731
    a = _lib.AttentionArgs(2, 1, 4, 4, 1, 1, 64, 0.125, v(), v(), v(), v())
    for name, val in kw.items():
        setattr(a, name, val)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=0), b"dtype"), (dict(B=-1), b"sizes"), (dict(D=4), b"head size"),
    (dict(D=136), b"head size"), (dict(D=66), b"head size"), (dict(Hkv=2), b"key heads"),
    (dict(Hkv=0), b"key heads"), (dict(scale=float("inf")), b"scale"),
    (dict(B=1 << 20, Lq=1 << 20), b"rows"), (dict(B=1 << 20, Lk=1 << 20), b"rows")])
def test_attention_refusals(kw, msg):
    from custom_rasterizer_cuda import _lib

    L, a = _lib.lib, attention_args(**kw)
    p = ctypes.addressof(a)
    assert L.gs_cross_attention_forward(p, A, 1 << 40, None) == _lib.GS_ERR_INVALID_ARG
    assert msg in L.gs_last_error()
    v = ctypes.addressof(a.out)
    assert L.gs_cross_attention_backward(p, v, v, v, v, A, 1 << 40, None) == \
        _lib.GS_ERR_INVALID_ARG
    assert msg in L.gs_last_error()


@pytest.mark.parametrize("name", ("q", "k", "v", "out"))
def test_attention_refuses_views_it_cannot_read(name):
    from custom_rasterizer_cuda import _lib

    for view, msg in ((_lib.TokenView(None, 64, 64, 64), b"null"),
                      (_lib.TokenView(A + 2, 64, 64, 64), b"16-byte"),
                      (_lib.TokenView(A, 64, 65, 64), b"16-byte")):
        a = attention_args(**{name: view})
        assert _lib.lib.gs_cross_attention_forward(ctypes.addressof(a), A, 1 << 40, None) == \
            _lib.GS_ERR_INVALID_ARG
        assert msg in _lib.lib.gs_last_error()


def test_attention_backward_needs_lse_and_workspace():
    from custom_rasterizer_cuda import _lib

    L = _lib.lib
    a = attention_args()
    v = ctypes.addressof(a.out)
    assert L.gs_cross_attention_backward(ctypes.addressof(a), v, v, v, v, A, 1 << 40, None) == \
        _lib.GS_ERR_INVALID_ARG
    assert b"lse" in L.gs_last_error()
    a = attention_args(lse=A)
    need = L.gs_cross_attention_backward_workspace_size(ctypes.addressof(a))
    assert need > 0
    assert L.gs_cross_attention_backward(ctypes.addressof(a), v, v, v, v, A, need - 1, None) == \
        _lib.GS_ERR_INVALID_ARG
    assert b"workspace" in L.gs_last_error()
    assert L.gs_cross_attention_forward(None, None, 0, None) == _lib.GS_ERR_INVALID_ARG
    # nothing to do
    assert L.gs_cross_attention_forward(ctypes.addressof(attention_args(B=0)), None, 0, None) == 0


def test_python_refuses_cpu_tensors():
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm, rms_norm_8bit
    from gs3d_b200.rotary import rotary_axes

    x = torch.zeros(1, 2, 1, 64)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        rotary_axes(x, torch.zeros(1, 2, 1), (64,))
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        rms_norm(x, torch.zeros(64))
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        rms_norm_8bit(x, torch.zeros(64))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        cross_attention(x, x, x)


@pytest.mark.gpu
def test_python_refusals(cuda_device):
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm, rms_norm_8bit
    from gs3d_b200.rotary import rotary_axes

    d = cuda_device
    x = torch.zeros(2, 3, 4, 64, device=d)
    pos = torch.zeros(2, 3, 2, device=d)
    for args, kw, msg in [
            ((x.double(), pos, (32, 32)), {}, "float32"), ((x[0], pos, (32, 32)), {}, "dimensions"),
            ((x, pos.double(), (32, 32)), {}, "int32 or float32"), ((x, pos, (32,)), {}, "positions"),
            ((x, pos[:, :2], (32, 32)), {}, "positions"), ((x, pos, (32, 34)), {}, "axis_dims"),
            ((x, pos, (31, 33)), {}, "axis_dims"), ((x, pos, (32, 32)), dict(base=-1.0), "base"),
            ((x[..., :63], pos, (2, 2)), {}, "even"), ((x, pos, (32, 32)), dict(base=(1.0,)), "base")]:
        with pytest.raises(RuntimeError, match=msg):
            rotary_axes(*args, **kw)
    w = torch.ones(64, device=d)
    for args, kw, msg in [
            ((x, w.half()), {}, "type"), ((x, w[:3]), {}, "weight"), ((x.int(), w.int()), {}, "x must"),
            ((x, w), dict(residual=x[:1]), "residual"), ((x, w), dict(eps=-1.0), "eps")]:
        with pytest.raises(RuntimeError, match=msg):
            rms_norm(*args, **kw)
    with pytest.raises(RuntimeError, match="group"):
        rms_norm_8bit(x, w, group=64)
    with pytest.raises(RuntimeError, match="gradient"):
        rms_norm_8bit(x.clone().requires_grad_(), w)
    q = x.bfloat16()
    mask = torch.ones(2, 1, 1, 3, dtype=torch.bool, device=d)
    for args, kw, msg in [
            ((x, x, x), {}, "float16 or bfloat16"), ((q, q, q.half()), {}, "same type"),
            ((q, q[:, :, :3], q[:, :, :3]), {}, "divide"), ((q, q, q[:, :2]), {}, "k and v"),
            ((q[..., :60], q[..., :60], q[..., :60]), {}, "multiple of 8"),
            ((q, q, q), dict(lengths=torch.zeros(2, device=d)), "lengths"),
            ((q, q, q), dict(lengths=torch.zeros(3, device=d, dtype=torch.int32)), "lengths"),
            ((q, q, q), dict(mask=mask.float()), "mask"), ((q, q, q), dict(mask=mask[..., :2]), "mask"),
            ((q, q, q), dict(mask=mask[0]), "mask"), ((q, q, q), dict(scale=float("nan")), "scale"),
            ((q, q, q), dict(lengths=torch.zeros(2, dtype=torch.int32)), "lengths")]:
        with pytest.raises(RuntimeError, match=msg):
            cross_attention(*args, **kw)


@pytest.mark.parametrize("kw", [dict(Lk=(1 << 31) - 1, D=8), dict(Lk=(1 << 31) - 1000, D=8),
                                dict(Lq=(1 << 31) - 1, D=8), dict(B=1 << 30, Hq=1 << 30, Lq=1 << 30),
                                dict(B=1 << 30, Hkv=1 << 30, Hq=1 << 30, Lq=0, Lk=16)])
def test_attention_refuses_rows_whose_tiles_would_pass_32_bits(kw):
    """A tile that reaches past the last row has to have indexes too; the product of three sizes may pass
    64 bits."""
    from custom_rasterizer_cuda import _lib

    L, a = _lib.lib, attention_args(lse=A, **kw)
    p, v = ctypes.addressof(a), ctypes.addressof(a.out)
    assert L.gs_cross_attention_forward(p, A, 1 << 62, None) == _lib.GS_ERR_INVALID_ARG
    assert b"rows" in L.gs_last_error()
    assert L.gs_cross_attention_backward(p, v, v, v, v, A, 1 << 62, None) == _lib.GS_ERR_INVALID_ARG
    assert b"rows" in L.gs_last_error()
    assert L.gs_cross_attention_workspace_size(p) == 0
    assert L.gs_cross_attention_backward_workspace_size(p) == 0


def test_attention_workspace_sizes_count_in_64_bits():
    from custom_rasterizer_cuda import _lib

    # 2^21 queries' statistics of two floats, and their parts; nothing but those without keys
    a = attention_args(B=1 << 10, Hq=1 << 6, Hkv=1, Lq=1 << 14, Lk=0, D=8)
    assert _lib.lib.gs_cross_attention_backward_workspace_size(ctypes.addressof(a)) >= 8 << 30


def test_attention_refuses_a_workspace_it_cannot_read_16_bytes_at_a_time():
    from custom_rasterizer_cuda import _lib

    L, bad = _lib.lib, _lib.GS_ERR_INVALID_ARG
    # one with a mask, one whose keys are split; the backward always needs one
    for kw in (dict(Lq=100, mask=A, mask_query_stride=4), dict(Lk=1 << 20, Lq=40)):
        a = attention_args(lse=A, **kw)
        p, v = ctypes.addressof(a), ctypes.addressof(a.out)
        assert L.gs_cross_attention_workspace_size(p) > 0
        for off in (4, 8):
            assert L.gs_cross_attention_forward(p, A + off, 1 << 40, None) == bad
            assert b"workspace" in L.gs_last_error()
            assert L.gs_cross_attention_backward(p, v, v, v, v, A + off, 1 << 40, None) == bad
            assert b"workspace" in L.gs_last_error()
        assert L.gs_cross_attention_forward(p, None, 1 << 40, None) == bad
        assert L.gs_cross_attention_backward(p, v, v, v, v, None, 1 << 40, None) == bad
