"""The token operators of the framework, case by case: what a decoder that predicts Gaussians from
images spends its time on besides matrix products.

An image is cut into the rasterizer's 16 x 16 tiles, one token each: a 1920 x 1080 view has
120 x 68 = 8,160 tokens, a 1280 x 720 view 80 x 45 = 3,600, a 128 x 128 view 64. Gaussian tokens
(the queries) look at the image tokens (the encoder's states) of one or several views.

* rotary: rotary positions with the axes (view, row, column); an image token sits at whole
  coordinates, a Gaussian at those of its projected mean.
* norm: root-mean-square norm with the residual's addition; for training with its gradients, for
  prediction with an 8-bit output (e4m3) and a scale for each row or group of 128.
* attention: cross attention of the Gaussian tokens to the image tokens, with key lengths for each
  batch item, masks, shared key heads, training and single queries.

`run` computes a case in plain torch operations in 32 bits, or, where `own` is true, through the
framework's entry points.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = 100.0  # rotary base: coordinates go up to a few hundred, not to hundreds of thousands
EPS = 1e-6
E4M3_MAX = 448.0


def _package():
    """The framework's package, imported on the first call that needs it."""
    path = str(ROOT / "custom-3dgs-cuda_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from gs3d_b200 import attention, norm, rotary

    return attention.cross_attention, norm.rms_norm, norm.rms_norm_8bit, rotary.rotary_axes


_calls = []


def _own():
    if not _calls:
        _calls.extend(_package())
    return _calls


# ---- the cases -----------------------------------------------------------------------------
def _rotary(name, train, B, L, H, D, dtype, whole, interleaved):
    return {"name": name, "op": "rotary", "train": train, "B": B, "L": L, "H": H, "D": D,
            "dtype": dtype, "whole": whole, "interleaved": interleaved}


def _norm(name, form, rows, width, dtype, residual, group=0):
    return {"name": name, "op": "norm", "form": form, "rows": rows, "width": width,
            "dtype": dtype, "residual": residual, "group": group}


def _attention(name, train, B, Lq, Lk, Hq, Hkv, D, dtype, lengths=False, mask="none"):
    return {"name": name, "op": "attention", "train": train, "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq,
            "Hkv": Hkv, "D": D, "dtype": dtype, "lengths": lengths, "mask": mask}


def listed():
    return [
        # four scenes, each asking for one more Gaussian: the rotation of that token's queries
        _rotary("rotary one token", False, 4, 1, 16, 64, "bf16", False, False),
        # the keys of one 720p view in full precision, pairs side by side
        _rotary("rotary 720p fp32", False, 1, 3600, 12, 64, "fp32", True, True),
        # training on eight 1080p views: the keys' rotation and its gradient
        _rotary("rotary 8 views train", True, 8, 8160, 16, 64, "bf16", True, False),
        # the 64 tokens of a 128 x 128 view, full precision, no residual
        _norm("norm 64 rows fp32", "forward", 64, 768, "fp32", False),
        # a training step's norm over one 1080p view, residual added, all gradients
        _norm("norm 1080p train", "train", 8160, 1024, "bf16", True),
        # prediction over eight 1080p views: residual added, 8-bit rows for the next product
        _norm("norm 8 views 8-bit", "8bit", 65280, 1024, "bf16", True),
        # four scenes, one new Gaussian each, over the scene's own part of a 720p view
        _attention("attention one query", False, 4, 1, 3600, 16, 16, 64, "bf16", lengths=True),
        # one new Gaussian over eight 1080p views, key heads shared by four query heads
        _attention("attention one query long", False, 2, 1, 65280, 32, 8, 128, "fp16"),
        # 4,096 Gaussians (the smallest scene of the benchmark) over a 1080p view
        _attention("attention 4096 x 8160", False, 1, 4096, 8160, 16, 16, 64, "bf16"),
        # a ragged set of Gaussians that each see some of the tokens only, a few of them none
        _attention("attention masked odd", False, 3, 1111, 777, 12, 4, 80, "fp16", mask="query"),
        # training on two scenes of different lengths, key heads shared
        _attention("attention train ragged", True, 2, 999, 3600, 8, 2, 64, "bf16", lengths=True),
        # training: 8,192 Gaussians over two 1080p views
        _attention("attention train large", True, 1, 8192, 16320, 16, 16, 128, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rotary", "norm", "attention", "attention"))
    if op == "rotary":
        H, D = rng.choice((8, 12, 16)), rng.choice((64, 96, 128))
        return {k: v for k, v in _rotary("", rng.random() < 0.4, rng.randint(1, 4),
                                         _log(rng, 1, 65280 * 16 * 64 / (H * D) * 0.5), H, D,
                                         rng.choice(("bf16", "bf16", "fp16", "fp32")),
                                         rng.random() < 0.5, rng.random() < 0.5).items()
                if k != "name"}
    if op == "norm":
        form = rng.choice(("forward", "train", "8bit"))
        width = rng.choice((256, 384, 768, 1000, 1024, 1536, 2048))
        rows = _log(rng, 1, 65280 * 1024 / width)
        group = 128 if form == "8bit" and width % 128 == 0 and rng.random() < 0.5 else 0
        return {k: v for k, v in _norm("", form, rows, width,
                                       rng.choice(("bf16", "bf16", "fp16", "fp32")),
                                       rng.random() < 0.7, group).items() if k != "name"}
    kind = rng.choice(("single", "forward", "train"))
    Hkv, shared, D = rng.choice((2, 4, 8)), rng.choice((1, 1, 2, 4)), rng.choice((64, 64, 80, 128))
    if kind == "single":
        B, Lq, Lk = rng.randint(1, 8), rng.choice((1, 1, 2, 3)), _log(rng, 64, 65280)
    else:
        B, Lq, Lk = rng.randint(1, 3), _log(rng, 16, 6000), _log(rng, 16, 10000)
    dtype = "bf16" if kind == "train" else rng.choice(("bf16", "bf16", "fp16"))
    mask = rng.choice(("none", "none", "key", "query"))
    if mask == "query" and Lk > 20000:
        mask = "key"
    return {k: v for k, v in _attention("", kind == "train", B, Lq, Lk, Hkv * shared, Hkv, D,
                                        dtype, rng.random() < 0.4, mask).items() if k != "name"}


# ---- inputs --------------------------------------------------------------------------------
def _axes(D):
    """The part of a head's D numbers that each axis turns: a quarter for the view, three eighths
    for the row and for the column."""
    return (D // 4, D * 3 // 8, D * 3 // 8)


def _normal(g, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * gain).to(dtype)


def _columns(L):
    """Tokens in a row of an image: that of the framework's image sizes that holds L of them."""
    return 8 if L <= 64 else 80 if L <= 3600 else 120


def _positions(g, B, L, whole):
    i = torch.arange(L, device="cuda")
    w = _columns(L)
    per_view = 8160
    view, row, col = i // per_view, (i % per_view) // w, (i % per_view) % w
    p = torch.stack((view, row, col), -1)[None].expand(B, L, 3)
    if whole:  # image tokens: one grid for all batch items
        p = p + torch.randint(0, 4, (B, 1, 3), generator=g, device="cuda")
        return p.to(torch.int32).contiguous()
    return (p + torch.rand(B, L, 3, generator=g, device="cuda")).float().contiguous()


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    c = dict(case)
    t = TYPES[c["dtype"]]
    if c["op"] == "rotary":
        shape = (c["B"], c["L"], c["H"], c["D"])
        c["x"] = _normal(g, shape, t).requires_grad_(c["train"])
        c["positions"] = _positions(g, c["B"], c["L"], c["whole"])
        if c["train"]:
            c["dy"] = _normal(g, shape, t, 0.1)
    elif c["op"] == "norm":
        shape = (c["rows"], c["width"])
        train = c["form"] == "train"
        c["x"] = _normal(g, shape, t).requires_grad_(train)
        c["weight"] = (1.0 + 0.2 * torch.randn(c["width"], generator=g, device="cuda")) \
            .to(t).requires_grad_(train)
        # a residual stream is larger than what one layer adds to it
        c["r"] = _normal(g, shape, t, 3.0).requires_grad_(train) if c["residual"] else None
        if train:
            c["dy"] = _normal(g, shape, t, 0.1)
            c["dh"] = _normal(g, shape, t, 0.1) if c["residual"] else None
    else:
        B, Lq, Lk = c["B"], c["Lq"], c["Lk"]
        train = c["train"]
        # queries of a trained model single out some of the keys: scores of deviation 1.5
        c["q"] = _normal(g, (B, Lq, c["Hq"], c["D"]), t, 1.5).requires_grad_(train)
        c["k"] = _normal(g, (B, Lk, c["Hkv"], c["D"]), t).requires_grad_(train)
        c["v"] = _normal(g, (B, Lk, c["Hkv"], c["D"]), t).requires_grad_(train)
        lengths = mask = None
        if c["lengths"]:
            lengths = torch.randint(Lk // 2, Lk + 1, (B,), generator=g, device="cuda")
            lengths = lengths.to(torch.int32)
        if c["mask"] == "key":  # tokens of the sky or of a mask image are left out
            mask = torch.rand(B, 1, 1, Lk, generator=g, device="cuda") < 0.8
        elif c["mask"] == "query":  # each Gaussian sees some of the tokens; a few see none
            mask = torch.rand(B, 1, Lq, Lk, generator=g, device="cuda") < 0.6
            mask &= torch.rand(B, 1, Lq, 1, generator=g, device="cuda") < 0.98
        c["key_lengths"], c["key_mask"] = lengths, mask
        if train:
            c["dy"] = _normal(g, (B, Lq, c["Hq"], c["D"]), t, 0.1)
    return c


# ---- the plain forms: 32 bits, rounded once at the end ---------------------------------------
def _plain_rotary(x, positions, axes, interleaved):
    angles = []
    for a, d in enumerate(axes):
        i = torch.arange(d // 2, device=x.device, dtype=torch.float32)
        angles.append(positions[..., a:a + 1].float() * torch.pow(BASE, -2.0 * i / d))
    parts, at = [], 0
    for d, angle in zip(axes, angles):
        z = x[..., at:at + d].float()
        cos, sin = torch.cos(angle)[:, :, None], torch.sin(angle)[:, :, None]
        if interleaved:
            u, v = z[..., 0::2], z[..., 1::2]
            parts.append(torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(-2))
        else:
            u, v = z[..., :d // 2], z[..., d // 2:]
            parts.append(torch.cat((u * cos - v * sin, u * sin + v * cos), -1))
        at += d
    if at < x.shape[-1]:
        parts.append(x[..., at:].float())
    return torch.cat(parts, -1).to(x.dtype)


def _plain_norm(x, weight, r):
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * weight.float()
    return y, h


def _plain_8bit(y, group):
    rows, width = y.shape
    z = y.view(rows, -1, group or width)
    scale = z.abs().amax(-1, keepdim=True) / E4M3_MAX
    q = (z / torch.where(scale > 0, scale, 1.0)).to(torch.float8_e4m3fn)
    return q.view(rows, width), scale.squeeze(-1)


def _plain_attention(q, k, v, lengths, mask):
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    shared = Hq // Hkv
    # query heads that share a key head are rows of one product
    z = q.float().view(B, Lq, Hkv, shared, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    s = (z @ k.float().permute(0, 2, 3, 1)) * (D ** -0.5)
    keep = None
    if lengths is not None:
        keep = (torch.arange(Lk, device=q.device) < lengths[:, None]).view(B, 1, 1, Lk)
    if mask is not None:
        keep = mask if keep is None else keep & mask
    if keep is not None:
        s = s.view(B, Hkv, shared, Lq, Lk)
        s = torch.where(keep[:, :, None], s, -math.inf).view(B, Hkv, -1, Lk)
    top = s.detach().amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    o = (e / torch.where(total > 0, total, 1.0)) @ v.float().permute(0, 2, 1, 3)
    o = o.view(B, Hkv, shared, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D)
    return o.to(q.dtype)


def run(s):
    if s["op"] == "rotary":
        x, positions, axes = s["x"], s["positions"], _axes(s["D"])
        if own:
            y = _own()[3](x, positions, axes, base=BASE, interleaved=s["interleaved"])
        else:
            y = _plain_rotary(x, positions, axes, s["interleaved"])
        if not s["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (x,), s["dy"]))
    if s["op"] == "norm":
        x, w, r, t = s["x"], s["weight"], s["r"], s["x"].dtype
        if s["form"] == "8bit":
            if own:
                return _own()[2](x, w, residual=r, eps=EPS, group=s["group"])
            y, h = _plain_norm(x, w, r)
            q8, scale = _plain_8bit(y, s["group"])
            return (q8, scale) if r is None else (q8, scale, h.to(t))
        if own:
            out = _own()[1](x, w, residual=r, eps=EPS)
        else:
            y, h = _plain_norm(x, w, r)
            out = y.to(t) if r is None else (y.to(t), h.to(t))
        if s["form"] == "forward":
            return out
        if r is None:
            return (out.detach(), *torch.autograd.grad(out, (x, w), s["dy"]))
        y, h = out
        grads = torch.autograd.grad((y, h), (x, r, w), (s["dy"], s["dh"]))
        return (y.detach(), h.detach(), *grads)
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        y = _own()[0](q, k, v, lengths=s["key_lengths"], mask=s["key_mask"])
    else:
        y = _plain_attention(q, k, v, s["key_lengths"], s["key_mask"])
    if not s["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, (q, k, v), s["dy"]))


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "rotary":
        n = c["B"] * c["L"] * c["H"] * c["D"]
        passes = 2 if c["train"] else 1
        return {"bytes": passes * (2 * n * size + c["B"] * c["L"] * 12), "flops": passes * 3 * n}
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        reads = writes = 2 if c["residual"] else 1  # x (and r), y (and h)
        if c["form"] == "8bit":
            scales = c["rows"] * (c["width"] // c["group"] if c["group"] else 1) * 4
            out = n + scales + (n * size if c["residual"] else 0)
            return {"bytes": reads * n * size + out + c["width"] * size, "flops": 6 * n}
        if c["form"] == "forward":
            return {"bytes": (reads + writes) * n * size + c["width"] * size, "flops": 5 * n}
        # forward, then dy (and dh) and h read, the gradient of x and r written (one and the same)
        b = (reads + writes + reads + 1 + 1) * n * size + 3 * c["width"] * size
        return {"bytes": b, "flops": 15 * n}
    B, Lq, Lk, Hq, Hkv, D = (c[k] for k in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    keys = 0.75 * Lk if c["lengths"] else Lk  # lengths are drawn from half of Lk to Lk
    nq, nk = B * Lq * Hq * D * size, B * keys * Hkv * D * size
    pairs = B * Hq * Lq * keys
    mask = B * Lq * keys if c["mask"] == "query" else B * keys if c["mask"] == "key" else 0
    bytes_ = 2 * nq + 2 * nk + mask
    if c["train"]:  # q, k, v, out, dout read again, dq, dk, dv written
        bytes_ += 3 * nq + 2 * nk + mask + nq + 2 * B * Lk * Hkv * D * size
    return {"bytes": bytes_, "flops": pairs * D * (14 if c["train"] else 4)}


# ---- the definitions in 64 bits ---------------------------------------------------------------
def _exact_rotary(c):
    """Each pair (u, v) as a complex number times exp(i position base^(-2 j / d))."""
    def turn(x, sign):
        out, at = x.double().clone(), 0
        for a, d in enumerate(_axes(c["D"])):
            f = torch.tensor([BASE ** (-2.0 * j / d) for j in range(d // 2)], dtype=torch.float64,
                             device=x.device)
            w = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                            sign * c["positions"][..., a].double()[..., None] * f)[:, :, None]
            j = torch.arange(d // 2, device=x.device)
            i0, i1 = (at + 2 * j, at + 2 * j + 1) if c["interleaved"] else (at + j, at + j + d // 2)
            z = torch.complex(x[..., i0].double(), x[..., i1].double()) * w
            out[..., i0], out[..., i1] = z.real, z.imag
            at += d
        return out

    with torch.no_grad():
        y = turn(c["x"], 1.0)
        return (y, turn(c["dy"], -1.0)) if c["train"] else y


def _exact_norm(c):
    with torch.no_grad():
        w = c["weight"].double()
        h = c["x"].double() + (c["r"].double() if c["residual"] else 0.0)
        rms = torch.sqrt(torch.sum(h ** 2, -1, keepdim=True) / c["width"] + EPS)
        u = h / rms
        y = u * w
        if c["form"] == "8bit":  # which 8-bit value is nearest hangs on the last bit of y
            z = y.view(c["rows"], -1, c["group"] or c["width"])
            scale = z.abs().amax(-1) / E4M3_MAX
            return (None, scale, h) if c["residual"] else (None, scale)
        if c["form"] == "forward":
            return (y, h) if c["residual"] else y
        dy = c["dy"].double()
        g = dy * w
        dx = (g - u * (g * u).sum(-1, keepdim=True) / c["width"]) / rms
        dw = (dy * u).sum(0)
        if not c["residual"]:
            return y, dx, dw
        dx = dx + c["dh"].double()
        return y, h, dx, dx, dw


def _exact_attention(c):
    B, Lq, Lk, Hq, Hkv, D = (c[k] for k in ("B", "Lq", "Lk", "Hq", "Hkv", "D"))
    q, k, v = (c[n].detach() for n in ("q", "k", "v"))
    out = torch.zeros(B, Lq, Hq, D, dtype=torch.float64, device=q.device)
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros(B, Lk, Hkv, D, dtype=torch.float64,
                                                      device=q.device) for _ in range(2))
    for b in range(B):
        n = Lk if c["key_lengths"] is None else int(c["key_lengths"][b])
        for h in range(Hq):
            n_h = h // (Hq // Hkv)
            K, V, Q = k[b, :n, n_h].double(), v[b, :n, n_h].double(), q[b, :, h].double()
            s = Q @ K.T / math.sqrt(D)
            if c["key_mask"] is not None:
                s = s.masked_fill(~c["key_mask"][b, 0, :, :n].expand(Lq, n), -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)  # a row without keys weighs nothing
            out[b, :, h] = p @ V
            if c["train"]:
                dO = c["dy"][b, :, h].double()
                dp = dO @ V.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) / math.sqrt(D)
                dq[b, :, h] = ds @ K
                dk[b, :n, n_h] += ds.T @ Q
                dv[b, :n, n_h] += p.T @ dO
                del dp, ds
            del s, p
    return (out, dq, dk, dv) if c["train"] else out


def exact(case, seed):
    c = prepare(case, seed)
    return {"rotary": _exact_rotary, "norm": _exact_norm, "attention": _exact_attention}[c["op"]](c)
