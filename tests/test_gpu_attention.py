"""Cross attention against a 64-bit plain form, forward and backward, with elementwise bounds
(tests/token_refs.py: P and dS rounded once to the inputs' type, the rest in 32 bits)."""

from __future__ import annotations

import math

import pytest
import torch

from token_refs import assert_within, attention64

pytestmark = pytest.mark.gpu
TYPES = (torch.bfloat16, torch.float16)


def draw(dev, dtype, B, Lq, Lk, Hq, Hkv, D, seed=0, gain=1.5):
    g = torch.Generator(dev).manual_seed(seed + 31 * Lq + 7 * Lk + D)
    n = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return ((gain * n(B, Lq, Hq, D)).to(dtype), n(B, Lk, Hkv, D).to(dtype),
            n(B, Lk, Hkv, D).to(dtype), n(B, Lq, Hq, D).to(dtype))


def masks(dev, B, Hq, Lq, Lk, kind, seed=0):
    g = torch.Generator(dev).manual_seed(seed + 11)
    u = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    if kind == "key":
        return u(B, 1, 1, Lk) < 0.7
    if kind == "query":  # some rows keep nothing
        return (u(B, 1, Lq, Lk) < 0.5) & (u(B, 1, Lq, 1) < 0.9)
    if kind == "head":
        return u(1, Hq, 1, Lk) < 0.6
    if kind == "full":
        return u(B, Hq, Lq, Lk) < 0.5
    return None


def check(q, k, v, dout=None, lengths=None, mask=None, scale=None):
    from gs3d_b200.attention import cross_attention

    ref = attention64(q, k, v, lengths, mask, scale, dout)
    out, lse = cross_attention(q, k, v, lengths=lengths, mask=mask, scale=scale, return_lse=True)
    assert_within(out, *ref["out"], "out")
    dead = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, dead)
    assert_within(torch.where(dead, 0.0, lse), torch.where(dead, 0.0, ref["lse"]),
                  torch.where(dead, 0.0, ref["lse_bound"]), "lse")
    assert not bool((out.transpose(1, 2)[dead] != 0).any())
    again = cross_attention(q, k, v, lengths=lengths, mask=mask, scale=scale)
    assert torch.equal(out, again)
    if dout is None:
        return
    ins = [t.detach().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*ins, lengths=lengths, mask=mask, scale=scale)
    assert torch.equal(o, out)
    grads = torch.autograd.grad(o, ins, dout, retain_graph=True)
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert_within(got, *ref[name], name)
    twice = torch.autograd.grad(o, ins, dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, twice)), "not the same bits again"


SIZES = [  # B, Lq, Lk, Hq, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 77, 4, 4, 64), (1, 1, 513, 8, 2, 128), (1, 2, 200, 12, 3, 80),
    (2, 3, 65, 4, 1, 64), (1, 17, 64, 2, 2, 32), (1, 128, 128, 2, 1, 64), (2, 129, 127, 3, 3, 64),
    (1, 257, 300, 4, 2, 128), (1, 300, 1, 2, 2, 64), (2, 100, 33, 2, 1, 72), (1, 64, 1000, 2, 2, 40),
    (1, 383, 641, 6, 2, 96), (1, 700, 129, 1, 1, 120)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_matches_64_bit(cuda_device, dtype, size):
    q, k, v, g = draw(cuda_device, dtype, *size)
    check(q, k, v, g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ("key", "query", "head", "full"))
@pytest.mark.parametrize("size", [(2, 1, 300, 8, 2, 64), (2, 3, 1030, 4, 4, 128),
                                  (2, 150, 261, 4, 2, 64), (1, 260, 391, 2, 2, 128),
                                  (2, 65, 7, 2, 1, 80)])
def test_masks(cuda_device, dtype, kind, size):
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=2)
    check(q, k, v, g, mask=masks(cuda_device, B, Hq, Lq, Lk, kind))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq,D", [(1, 64), (4, 128), (140, 64), (270, 128)])
def test_lengths_and_what_lies_past_them(cuda_device, dtype, Lq, D):
    """Lengths of zero, one, a tile's end and its neighbours, more than Lk and negative ones;
    infinities and NaN in keys and values past them."""
    lengths = [0, 1, 63, 64, 65, 128, 200, 256, 300, 301, 1000, -5]
    B, Lk = len(lengths), 300
    q, k, v, g = draw(cuda_device, dtype, B, Lq, Lk, 4, 2, D, seed=4)
    for b, n in enumerate(lengths):
        k[b, max(n, 0):] = float("nan") if b % 2 else float("inf")
        v[b, max(n, 0):] = float("inf") if b % 2 else float("nan")
    t = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    check(q, k, v, g, lengths=t)
    check(q, k, v, g, lengths=t, mask=masks(cuda_device, B, 4, Lq, Lk, "query"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq", (1, 200))
def test_a_key_mask_hides_infinities_and_nan(cuda_device, dtype, Lq):
    q, k, v, g = draw(cuda_device, dtype, 2, Lq, 333, 4, 2, 64, seed=5)
    mask = masks(cuda_device, 2, 4, Lq, 333, "key")
    mask[1, ..., :200] = False
    hidden = ~mask[:, 0, 0]
    for i, bad in enumerate((float("nan"), float("inf"), -float("inf"),
                             torch.finfo(dtype).min)):
        at = hidden.clone()
        at[:, torch.arange(333, device=cuda_device) % 4 != i] = False
        k[at], v[at] = bad, bad
    check(q, k, v, g, mask=mask)


@pytest.mark.parametrize("Lq", (1, 2, 130))
def test_masked_tiles_first_and_last(cuda_device, Lq):
    """The first kept key comes late, or the kept keys end early, for some rows."""
    q, k, v, g = draw(cuda_device, torch.bfloat16, 1, Lq, 700, 2, 2, 64, seed=6)
    mask = torch.zeros(1, 2, Lq, 700, dtype=torch.bool, device=cuda_device)
    mask[:, 0, :, 650:] = True
    mask[:, 1, :, :3] = True
    mask[:, 1, -1] = False
    check(q, k, v, g, mask=mask)


def test_large_scores_and_growing_maxima(cuda_device):
    """Scores of a few hundred, growing along the keys, so that the running maximum moves often."""
    for Lq in (1, 130):
        q, k, v, g = draw(cuda_device, torch.bfloat16, 1, Lq, 600, 2, 2, 64, seed=7, gain=1.0)
        ramp = torch.linspace(0.0, 8.0, 600, device=cuda_device).view(1, 600, 1, 1)
        k = (k * ramp).bfloat16()
        q = (q * 8.0).bfloat16()
        check(q, k, v, g)
        check(q, k.flip(1), v, g, scale=-0.05)


def test_strides_and_orders(cuda_device):
    from gs3d_b200.attention import cross_attention

    q, k, v, g = draw(cuda_device, torch.bfloat16, 2, 150, 90, 4, 2, 64, seed=8)
    dev = cuda_device

    def moved(t, order):  # the same numbers with the axes in another order in memory
        inv = [order.index(i) for i in range(4)]
        return t.permute(order).contiguous().permute(inv)

    for order in ((0, 2, 1, 3), (1, 0, 2, 3), (2, 1, 0, 3), (0, 1, 3, 2)):
        check(moved(q, order), moved(k, order), moved(v, order), moved(g, order))
    packed = torch.randn(2, 90, 2, 2, 64, device=dev).bfloat16()
    check(q, packed[:, :, 0], packed[:, :, 1], g)  # keys and values in one tensor
    odd = torch.randn(2, 90, 2, 65, device=dev).bfloat16()
    check(q, odd[..., 1:], odd[..., :64], g)       # neither aligned
    check(q, k[:1].expand(2, 90, 2, 64), v[:1].expand(2, 90, 2, 64), g)  # one encoder for all
    check(q[:, :1].expand(2, 150, 4, 64), k, v, g[:, :, :1].expand(2, 150, 4, 64))
    # the gradient of a broadcast input is the sum over its readers
    one = k[:1].detach().clone().requires_grad_()
    o = cross_attention(q, one.expand(2, 90, 2, 64), v)
    (d1,) = torch.autograd.grad(o, (one,), g)
    ref = attention64(q, one.detach().expand(2, 90, 2, 64), v, dout=g)["dk"]
    assert_within(d1, ref[0].sum(0, keepdim=True),
                  ref[1].sum(0, keepdim=True) + 2.0 ** -7 * ref[0].abs().sum(0, keepdim=True), "dk")


def test_gradient_of_a_scalar_loss(cuda_device):
    """sum().backward() hands the backward a gradient with strides of zero."""
    from gs3d_b200.attention import cross_attention

    q, k, v, _ = draw(cuda_device, torch.bfloat16, 1, 140, 70, 2, 2, 64, seed=9)
    ins = [t.requires_grad_() for t in (q, k, v)]
    cross_attention(*ins).sum().backward()
    ref = attention64(q.detach(), k.detach(), v.detach(), dout=torch.ones_like(q))
    for t, name in zip(ins, ("dq", "dk", "dv")):
        assert_within(t.grad, *ref[name], name)


def test_empty(cuda_device):
    from gs3d_b200.attention import cross_attention

    for B, Lq, Lk, H in ((0, 4, 4, 2), (2, 0, 4, 2), (2, 4, 0, 2), (1, 1, 0, 2), (2, 4, 4, 0)):
        q = torch.randn(B, Lq, H, 64, device=cuda_device).half().requires_grad_()
        k = torch.randn(B, Lk, H, 64, device=cuda_device).half().requires_grad_()
        v = torch.randn(B, Lk, H, 64, device=cuda_device).half().requires_grad_()
        o, lse = cross_attention(q, k, v, return_lse=True)
        assert o.shape == (B, Lq, H, 64) and not o.any()
        assert bool((lse == -math.inf).all()) or Lk
        grads = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert all(d.shape == t.shape and not d.any() for d, t in zip(grads, (q, k, v)))


def test_gradient_matches_differences(cuda_device):
    from gs3d_b200.attention import cross_attention

    q, k, v, g = draw(cuda_device, torch.bfloat16, 2, 70, 90, 4, 2, 64, seed=10)
    mask = masks(cuda_device, 2, 4, 70, 90, "query")
    ins = [t.clone().requires_grad_() for t in (q, k, v)]
    o = cross_attention(*ins, mask=mask)
    grads = torch.autograd.grad(o, ins, g)
    ref = attention64(q, k, v, None, mask, dout=g)
    step = 1e-4
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn_like(ins[i]).double()
        at = [t.double() for t in (q, k, v)]
        loss = []
        for sign in (1, -1):
            m = list(at)
            m[i] = at[i] + sign * step * d
            loss.append(float((_out64(*m, mask) * g.double()).sum()))
        want = (loss[0] - loss[1]) / (2 * step)
        got = float((grads[i].double() * d).sum())
        # every element may be off by its bound; the difference itself by step^2 of the third
        # derivative, below 1e-5 of the gradient here
        slack = float((ref[name][1] * d.abs()).sum()) + 1e-5 * float(
            (ref[name][0] * d).abs().sum())
        assert abs(got - want) < slack, (name, got, want, slack)


def _out64(q, k, v, mask):
    K, V = (t.transpose(1, 2).repeat_interleave(2, 1) for t in (k, v))
    s = torch.where(mask, q.transpose(1, 2) @ K.transpose(2, 3) / 8.0, -math.inf)
    return (torch.softmax(s, -1).nan_to_num(0.0) @ V).transpose(1, 2)


def test_runs_on_the_current_stream(cuda_device):
    from gs3d_b200.attention import cross_attention

    q, k, v, g = draw(cuda_device, torch.bfloat16, 1, 300, 500, 4, 4, 64, seed=11)
    ref = attention64(q, k, v)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        busy = torch.randn(4096, 4096, device=cuda_device)
        for _ in range(4):
            busy = busy @ busy * 1e-3
        o = cross_attention(q + 0, k + 0, v + 0)
        one = cross_attention(q[:, :1] + 0, k + 0, v + 0)
    s.synchronize()
    assert_within(o, *ref["out"], "other stream")
    assert_within(one, ref["out"][0][:, :1], ref["out"][1][:, :1], "other stream, one query")


def test_calls_recorded_in_a_graph(cuda_device):
    """Every kernel of the token operators, the masked and split ones and those that overlap the end
    of the one before included, replays in a CUDA graph on new inputs."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm, rms_norm_8bit
    from gs3d_b200.rotary import rotary_axes

    q, k, v, _ = draw(cuda_device, torch.bfloat16, 2, 150, 900, 4, 2, 64, seed=12)
    mask = masks(cuda_device, 2, 4, 150, 900, "query")
    lengths = torch.tensor([900, 411], dtype=torch.int32, device=cuda_device)
    w = torch.ones(64, device=cuda_device, dtype=torch.bfloat16)
    pos = torch.rand(2, 150, 1, device=cuda_device) * 30

    def chain():
        x, h = rms_norm(q, w, residual=q)
        x = rotary_axes(x, pos, (64,))
        o = cross_attention(x, k, v, lengths=lengths, mask=mask)
        one = cross_attention(o[:, :1], k, v, lengths=lengths)
        q8, s = rms_norm_8bit(o, w)
        return x, h, o, one, q8, s

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            chain()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for seed in (13, 14):
        fresh = draw(cuda_device, torch.bfloat16, 2, 150, 900, 4, 2, 64, seed=seed)
        for old, new in zip((q, k, v), fresh):
            old.copy_(new)
        lengths.copy_(torch.tensor([900 - seed, 300 + seed], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, chain()):
            assert torch.equal(a.float(), b.float())


def test_back_to_back_calls_do_not_overtake_one_another(cuda_device):
    """Kernels that may start before the one in front has ended still see its results: a chain of
    dependent calls, its buffers reused by the allocator, gives the same bits as one that waits
    after every call."""
    from gs3d_b200.attention import cross_attention
    from gs3d_b200.norm import rms_norm
    from gs3d_b200.rotary import rotary_axes

    q, k, v, _ = draw(cuda_device, torch.bfloat16, 1, 300, 700, 4, 2, 64, seed=15)
    w = torch.ones(64, device=cuda_device, dtype=torch.bfloat16)
    pos = torch.rand(1, 300, 1, device=cuda_device) * 30
    mask = masks(cuda_device, 1, 4, 300, 700, "query")

    def chain(wait):
        x, n = q, torch.full((1,), 700, dtype=torch.int32, device=cuda_device)
        for i in range(12):
            x = rotary_axes(x, pos, (64,), inverse=bool(i % 2))
            wait()
            x = cross_attention(x, k, v, lengths=n, mask=mask if i % 3 else None)
            wait()
            x, _ = rms_norm(x, w, residual=q)
            wait()
            one = cross_attention(x[:, :2], k, v, lengths=n)
            wait()
            x = torch.cat((one, x[:, 2:]), 1)
            n = n - 13
        return x

    apart = chain(torch.cuda.synchronize)
    for _ in range(5):
        assert torch.equal(chain(lambda: None), apart)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(2, 1, 900, 48, 2, 64), (1, 1, 2000, 128, 1, 128),
                                  (1, 5, 700, 16, 4, 80), (2, 10, 1333, 24, 2, 64),
                                  (1, 30, 5000, 12, 2, 64), (40, 64, 257, 4, 1, 128),
                                  (1, 1, 600, 130, 1, 64), (1, 3, 290, 43, 1, 64),
                                  (30, 9, 70, 16, 2, 96), (1, 12, 1000, 2, 2, 128)])
def test_few_queries_of_many_shared_heads(cuda_device, dtype, size):
    """More rows for each key head than the single-query form takes, fewer queries than a tile."""
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=8)
    apart = q.transpose(1, 2).contiguous().transpose(1, 2)  # heads outside of queries
    check(apart, k, v, g)
    t = torch.arange(B, device=cuda_device, dtype=torch.int32) * 131 % (Lk + 1)
    for kind in ("key", "query", "head", "full"):
        check(q, k, v, lengths=t, mask=masks(cuda_device, B, Hq, Lq, Lk, kind))


def test_no_second_derivative(cuda_device):
    from gs3d_b200.attention import cross_attention

    q, k, v, _ = draw(cuda_device, torch.bfloat16, 1, 4, 6, 1, 1, 8)
    q.requires_grad_()
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(cross_attention(q, k, v).sum(), q, create_graph=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(3, 300, 900, 28, 7, 64), (2, 600, 800, 30, 5, 128),
                                  (32, 257, 500, 5, 5, 40), (1, 5000, 700, 8, 2, 80)])
def test_more_blocks_of_queries_than_run_at_once(cuda_device, dtype, size):
    """Between one and three waves of CTAs, with every kind of mask."""
    B, Lq, Lk, Hq, Hkv, D = size
    q, k, v, g = draw(cuda_device, dtype, *size, seed=9)
    check(q, k, v, g)
    t = torch.arange(B, device=cuda_device, dtype=torch.int32) * 131 % (Lk + 1)
    for kind in ("key", "query", "head"):
        check(q, k, v, lengths=t if B > 1 else None,
              mask=masks(cuda_device, B, Hq, Lq, Lk, kind))


@pytest.mark.parametrize("D", (64, 128))
def test_one_item_much_longer_than_the_others(cuda_device, D):
    """Items without keys beside one with many, infinities past the ends."""
    lengths = [0, 1, 4000, 0, 130, 128, -3, 129, 1] + [1] * 10 + [0]
    B, Lk = len(lengths), 4000
    q, k, v, _ = draw(cuda_device, torch.bfloat16, B, 257, Lk, 4, 2, D, seed=10)
    for b, n in enumerate(lengths):
        k[b, max(n, 0):] = float("nan") if b % 2 else float("inf")
        v[b, max(n, 0):] = float("inf") if b % 2 else float("nan")
    t = torch.tensor(lengths, dtype=torch.int32, device=cuda_device)
    check(q, k, v, lengths=t)
    check(q, k, v, lengths=t.clamp(max=1), mask=masks(cuda_device, B, 4, 257, Lk, "key"))
