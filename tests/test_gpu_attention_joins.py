"""The ways in which cross attention joins the parts of split keys: in a cluster's shared memory, or
by a second kernel, from the single-query form and from the tiled one, with parts that keep nothing
and with NaN and infinities at keys that are kept."""

from __future__ import annotations

import math
import threading

import pytest
import torch

from test_gpu_attention import TYPES, check, draw, masks
from token_refs import attention64

pytestmark = pytest.mark.gpu

# B, Lq, Lk, Hq, Hkv, D
SINGLE = [
    (1, 1, 9000, 4, 2, 64), (2, 1, 5000, 8, 2, 128), (1, 2, 7001, 4, 2, 80),  # more than 8 splits
    (1, 3, 12345, 4, 4, 40),
    (1, 12, 6000, 2, 2, 64), (1, 5, 9001, 6, 2, 64),                          # two groups of 8 rows
    (1, 12, 1100, 2, 2, 64), (2, 3, 2000, 16, 4, 32), (3, 16, 700, 4, 4, 64),
    (4, 1, 2600, 8, 8, 128), (5, 1, 900, 9, 9, 64)]                           # 2 to 8 splits
TILED = [(1, 17, 9000, 2, 2, 64), (1, 300, 4000, 1, 1, 128), (2, 200, 3000, 2, 1, 80),
         (1, 130, 6000, 8, 8, 64), (2, 999, 1500, 8, 2, 64), (1, 9, 8000, 8, 2, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SINGLE + TILED)
def test_split_keys(cuda_device, dtype, size):
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=51)
    check(q, k, v, g)
    # lengths that leave the later parts without keys, and none at all
    for n in ((Lk, Lk // 2, 3), (1, 0, Lk), (0, Lk // 5, 129)):
        t = torch.tensor([n[b % 3] for b in range(B)], dtype=torch.int32, device=cuda_device)
        check(q, k, v, lengths=t)
    for kind in ("key", "query", "head", "full"):
        mask = masks(cuda_device, B, Hq, Lq, Lk, kind)
        check(q, k, v, mask=mask)
        mask[..., Lk // 4:] = False  # nothing kept in the later parts
        check(q, k, v, mask=mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(1, 1, 300, 2, 2, 64), (1, 1, 2500, 2, 2, 64), (1, 1, 9000, 2, 2, 64),
                                  (1, 12, 6000, 2, 2, 64), (1, 2, 5000, 4, 2, 128),
                                  (1, 140, 300, 2, 2, 64), (1, 140, 2500, 2, 2, 128),
                                  (1, 140, 9000, 2, 2, 64), (2, 300, 3000, 4, 4, 64),
                                  (1, 20, 3000, 8, 1, 64)])
def test_nan_and_infinities_that_are_kept(cuda_device, dtype, size):
    """A query that keeps a key of NaN, or one whose score is infinite, has NaN for an answer; NaN in
    a value stays in its own number, and infinity arrives as infinity. Other queries, items and heads
    do not see any of it, wherever along the keys it lies."""
    from gs3d_b200.attention import cross_attention

    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, _ = draw(cuda_device, dtype, *size, seed=52, gain=0.5)
    group = Hq // Hkv
    q[:, Lq // 2, :, 3] = -1.0
    q[:, :Lq // 2, :, 3] = 1.0
    q[:, Lq // 2 + 1:, :, 3] = 1.0
    clean = cross_attention(q, k, v)
    for at in (0, Lk // 2, Lk - 1):
        k2 = k.clone()
        k2[0, at, 0] = float("nan")
        out, lse = cross_attention(q, k2, v, return_lse=True)
        assert out[0, :, :group].isnan().all() and lse[0, :group].isnan().all()
        assert torch.equal(out[0, :, group:], clean[0, :, group:])
        assert torch.equal(out[1:], clean[1:])
        # +inf for the queries with a positive number there, -inf (weight 0) for the one without
        k2 = k.clone()
        k2[0, at, 0, 3] = float("inf")
        out, lse = cross_attention(q, k2, v, return_lse=True)
        rows = torch.arange(Lq, device=cuda_device) != Lq // 2
        assert out[0, rows, :group].isnan().all() and lse[0, :group, rows].isnan().all()
        keep = torch.ones(1, 1, 1, Lk, dtype=torch.bool, device=cuda_device)
        keep[..., at] = False
        ref = attention64(q, k, v, mask=keep)["out"]
        got, want, bound = (t[0, Lq // 2, :group].double() for t in (out, *ref))
        assert bool(((got - want).abs() <= bound).all())
        assert torch.equal(out[0, :, group:], clean[0, :, group:])
        v2 = v.clone()
        v2[0, at, 0, 7], v2[0, at, 0, 2] = float("nan"), float("inf")
        out, lse = cross_attention(q, k, v2, return_lse=True)
        assert out[0, :, :group, 7].isnan().all() and torch.isfinite(lse).all()
        assert bool((out[0, :, :group, 2] == math.inf).all())
        others = [d for d in range(D) if d not in (2, 7)]
        assert torch.equal(out[..., others], clean[..., others])


def test_calls_from_several_threads_and_streams(cuda_device):
    """Each thread on its own stream, each with its own inputs, sizes and masks: the results are those
    of calls one after another."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm

    cases = []
    for i, size in enumerate([(1, 1, 9000, 4, 2, 64), (2, 150, 700, 4, 2, 64), (1, 300, 500, 4, 4, 128),
                              (2, 3, 1200, 8, 2, 128)]):
        q, k, v, g = draw(cuda_device, torch.bfloat16, *size, seed=60 + i)
        mask = masks(cuda_device, size[0], size[3], size[1], size[2], "query") if i % 2 else None
        cases.append((q, k, v, g, mask, torch.ones(size[5], device=cuda_device).bfloat16()))

    def step(q, k, v, g, mask, w):
        ins = [t.detach().requires_grad_() for t in (q, k, v, w)]
        y, h = rms_norm(ins[0], ins[3], residual=q)
        out = cross_attention(y, ins[1], ins[2], mask=mask)
        return (out.detach(), h.detach(), *torch.autograd.grad(out, ins, g))

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * len(cases), []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got[i] = step(*cases[i])
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def training_step(sizes, dev):
    """Norm, attention and their gradients, of sizes whose backward splits keys, queries, both or
    neither, with masks and lengths."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm
    from gs3d_b200.rotary import rotary_axes

    state = []
    for i, size in enumerate(sizes):
        B, Lq, Lk, Hq, Hkv, D = size
        q, k, v, g = draw(dev, torch.bfloat16, *size, seed=70 + i)
        mask = masks(dev, B, Hq, Lq, Lk, (None, "query", "key", "head")[i % 4])
        n = torch.full((B,), Lk - i, dtype=torch.int32, device=dev)
        pos = torch.rand(B, Lq, 1, device=dev) * 30
        state.append(([t.requires_grad_() for t in (q, k, v)], g, mask, n, pos,
                      torch.ones(D, device=dev).bfloat16().requires_grad_()))

    def step(wait):
        res = []
        for ins, g, mask, n, pos, w in state:
            x = rotary_axes(ins[0], pos, (w.shape[0],))
            wait()
            y, h = rms_norm(x, w, residual=ins[0])
            wait()
            out = cross_attention(y, ins[1], ins[2], lengths=n, mask=mask)
            wait()
            res += [out.detach(), *torch.autograd.grad((out, h), (*ins, w), (g, g))]
            wait()
        return res

    return state, step


# the backward's splits of the queries (for dk and dv) and of the keys (for dq): both, only dk and dv,
# only dq, neither
TRAINING = [(1, 300, 700, 2, 2, 64), (1, 6000, 130, 4, 2, 64), (1, 130, 9000, 4, 4, 64),
            (2, 700, 1500, 16, 8, 64), (1, 300, 700, 2, 1, 128), (1, 5000, 130, 4, 2, 128),
            (1, 130, 9000, 4, 2, 128), (2, 900, 1300, 16, 8, 128)]


def test_training_steps_back_to_back(cuda_device):
    """Kernels that start before the one in front has ended, dq's among them: the same bits as when
    the host waits after every call."""
    _, step = training_step(TRAINING, cuda_device)
    apart = step(torch.cuda.synchronize)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(step(lambda: None), apart))


def test_training_steps_in_a_graph(cuda_device):
    state, step = training_step(TRAINING, cuda_device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(lambda: None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(lambda: None)
    for seed in (1, 2):
        torch.manual_seed(seed)
        with torch.no_grad():
            for ins, g, _, n, _, _ in state:
                for t in (*ins, g):
                    t.copy_(torch.randn_like(t))
                n.sub_(20)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(lambda: None)))
