"""64-bit plain forms of the token operators (rotary positions, norms, cross attention), their
gradients by the formulas, and elementwise error bounds for kernels that hold sums, statistics and
scores in 32 bits."""

from __future__ import annotations

import math

import torch

# the largest relative error of one rounding (half a unit in the last place)
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# half the smallest step, where numbers are too small for the relative bound
STEP = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def assert_within(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(ref.shape)}"
    g = got.double()
    assert bool(torch.isfinite(g).all()), f"{what}: {int((~torch.isfinite(g)).sum())} not finite"
    over = (g - ref).abs() - bound
    worst = float(over.max()) if over.numel() else -1.0
    if worst > 0:
        i = int(over.argmax())
        raise AssertionError(f"{what}: at {i}: {float(g.flatten()[i])} vs "
                             f"{float(ref.flatten()[i])}, bound {float(bound.flatten()[i])}; "
                             f"{int((over > 0).sum())} of {over.numel()} outside")


def rotary64(x, positions, dims, bases, interleaved=False, inverse=False):
    """(y, |u| + |v| of each number's pair)."""
    y, mag = x.double().clone(), x.double().abs()
    at = 0
    for a, d in enumerate(dims):
        j = torch.arange(d // 2, device=x.device)
        f = torch.tensor([bases[a] ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64,
                         device=x.device)
        angle = (positions[..., a].double()[..., None] * f)[:, :, None]
        if inverse:
            angle = -angle
        iu, iv = (at + 2 * j, at + 2 * j + 1) if interleaved else (at + j, at + j + d // 2)
        u, v = x[..., iu].double(), x[..., iv].double()
        y[..., iu] = u * angle.cos() - v * angle.sin()
        y[..., iv] = u * angle.sin() + v * angle.cos()
        mag[..., iu] = mag[..., iv] = u.abs() + v.abs()
        at += d
    return y, mag


def norm64(x, w, r, eps):
    h = x.double() + (0.0 if r is None else r.double())
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h * rstd * w.double(), h, rstd


def norm_backward64(dy, dh, h, w, eps):
    """Gradients for the h given (a kernel that keeps h in fewer bits differentiates there)."""
    h, dy, w = h.double(), dy.double(), w.double()
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    u, g = h * rstd, dy * w
    dx = rstd * (g - u * (g * u).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.double()
    return dx, (dy * u).reshape(-1, h.shape[-1]).sum(0)


def keep_mask(B, Hq, Lq, Lk, lengths, mask, device):
    keep = torch.ones(B, Hq, Lq, Lk, dtype=torch.bool, device=device)
    if lengths is not None:
        n = lengths.clamp(0, Lk)
        keep &= (torch.arange(Lk, device=device) < n[:, None]).view(B, 1, 1, Lk)
    if mask is not None:
        keep &= mask
    return keep


def attention64(q, k, v, lengths=None, mask=None, scale=None, dout=None):
    """Output, lse and (with dout) gradients in 64 bits, with bounds for a kernel that rounds P and
    dS to q's type once, holds the rest in 32 bits and rounds results once. All [B, L, H, D]."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1], k.shape[2]
    rep = Hq // max(Hkv, 1)
    scale = D ** -0.5 if scale is None else scale
    Q = q.double().transpose(1, 2)
    K = k.double().transpose(1, 2).repeat_interleave(rep, 1)
    V = v.double().transpose(1, 2).repeat_interleave(rep, 1)
    keep = keep_mask(B, Hq, Lq, Lk, lengths, mask, q.device)
    # what lies at a key that all queries leave out is not part of the result
    used = keep.any(2, keepdim=True).transpose(2, 3)
    K, V = torch.where(used, K, 0.0), torch.where(used, V, 0.0)
    s = torch.where(keep, Q @ K.transpose(2, 3) * scale, -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full((B, Hq, Lq), -math.inf,
                                                       dtype=torch.float64, device=q.device)
    p = torch.exp(s - torch.where(lse > -math.inf, lse, 0.0)[..., None])
    p = torch.where(keep, p, 0.0)
    o = p @ V
    eps = ROUND[q.dtype]
    # a score's error in 32 bits: D products added, and the exponent's rounding
    mag = (Q.abs() @ K.abs().transpose(2, 3)) * abs(scale)
    top = torch.where(keep, s, 0.0).abs().amax() if s.numel() else 0.0
    es = D * 2.0 ** -24 * mag + 2.0 ** -21 * (1.0 + top)
    ep = p * (eps + 2.0 * es) + 2.0 ** -24 * (eps if q.dtype == torch.float16 else 0.0)
    eo = ep @ V.abs() + p.sum(-1, keepdim=True) * 0.0
    # the sum that normalises p has its own error, a mean of those of the scores
    ez = (p * (2.0 * es + 2.0 ** -20)).sum(-1, keepdim=True)
    eo = eo + ez * (p @ V.abs()) + eps * o.abs() + STEP[q.dtype] + eps * eo
    res = {"out": (o.transpose(1, 2), eo.transpose(1, 2)), "lse": lse,
           "lse_bound": ez.squeeze(-1) + 2.0 ** -20 * (1.0 + lse.abs().nan_to_num(posinf=0.0))}
    if dout is None:
        return res
    G = dout.double().transpose(1, 2)
    dp = G @ V.transpose(2, 3)
    delta = (G * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_dp = D * 2.0 ** -24 * (G.abs() @ V.abs().transpose(2, 3))
    e_delta = (G.abs() * eo).sum(-1, keepdim=True) + D * 2.0 ** -24 * (G.abs() * o.abs()).sum(
        -1, keepdim=True)
    rel = 2.0 * es + ez
    e_ds = ds.abs() * (eps + rel) + p * (e_dp + e_delta)
    if q.dtype == torch.float16:
        e_ds = torch.where(keep, e_ds + 2.0 ** -25, e_ds)
    n_k = Lk * 2.0 ** -24
    n_q = Lq * rep * 2.0 ** -24

    def heads(t):  # the query heads that share a key head
        return t.view(B, max(Hkv, 1), rep, Lk, D).sum(2).transpose(1, 2) if Hkv else t

    dq = scale * (ds @ K)
    b_q = abs(scale) * ((e_ds + ds.abs() * n_k) @ K.abs())
    Tds, Te = ds.transpose(2, 3), (e_ds + ds.abs() * n_q).transpose(2, 3)
    dk, b_k = scale * (Tds @ Q), abs(scale) * (Te @ Q.abs())
    Tp = p.transpose(2, 3)
    dv = Tp @ G
    b_v = (p * (eps + rel + n_q) + (ep - p * eps).clamp(min=0.0)).transpose(2, 3) @ G.abs()
    dk, b_k, dv, b_v = heads(dk), heads(b_k), heads(dv), heads(b_v)
    fin = lambda g, b: (g, b * (1.0 + eps) + eps * g.abs() + STEP[q.dtype])  # noqa: E731
    res["dq"] = fin(dq.transpose(1, 2), b_q.transpose(1, 2))
    res["dk"], res["dv"] = fin(dk, b_k), fin(dv, b_v)
    return res
