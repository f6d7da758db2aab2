"""A small decoder that predicts Gaussians from views, on the token operators: the path that runs
rotary positions, norms and cross attention together and ends in the rasterizer.

Views are cut into the rasterizer's 16 x 16 tiles, one token each, at the whole coordinates (view,
row, column). Each Gaussian is a query token at the coordinates of its mean projected into the
first view. A layer adds to the Gaussian's stream what its cross attention to the image tokens
finds, then what a two-layer product makes of it; every addition is taken by the next norm. A last
product gives each Gaussian's change of mean, log-scale, quaternion, opacity logit and colour, and
`gaussian_splatting.rasterizer` renders the result, so the photometric loss trains all of it.

`predict` answers without gradients: the norms before the wide products write 8-bit rows, which
torch's 8-bit matrix product takes with their scales.

    python -m gs3d_b200.decoder --steps 30     # trains on a synthetic scene, prints the loss
"""

from __future__ import annotations

import argparse

import torch
import torch.nn.functional as F

from gaussian_splatting.rasterizer.rasterize import RasterizeFunction

from .attention import cross_attention
from .loss import l1_ssim_loss
from .norm import rms_norm, rms_norm_8bit
from .rotary import rotary_axes

TILE = 16
# numbers of one Gaussian: mean 3, quaternion 4, log-scale 3, opacity logit 1, SH DC 3
OUT = 14
E4M3_MAX = 448.0


def view_tokens(images: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[V, H, W, 3] images -> the pixels of each 16 x 16 tile [1, V * rows * columns, 768], zero
    past the image's edge, and the tiles' (view, row, column) [1, ., 3] int32."""
    V, H, W, _ = images.shape
    rows, cols = -(-H // TILE), -(-W // TILE)
    x = F.pad(images, (0, 0, 0, cols * TILE - W, 0, rows * TILE - H))
    x = x.view(V, rows, TILE, cols, TILE, 3).permute(0, 1, 3, 2, 4, 5)
    axes = [torch.arange(n, device=images.device, dtype=torch.int32) for n in (V, rows, cols)]
    at = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1)
    return x.reshape(1, V * rows * cols, TILE * TILE * 3), at.view(1, -1, 3)


def gaussian_positions(mu: torch.Tensor, view) -> torch.Tensor:
    """Coordinates [1, N, 3] of means in `view`: (0, row, column) in tiles; where the mean lies
    behind the camera, the image's centre."""
    cam = mu @ view.R.to(mu).T + view.T.to(mu)
    z = cam[:, 2]
    ahead = z > 0.2
    z = torch.where(ahead, z, 1.0)
    col = torch.where(ahead, view.fx * cam[:, 0] / z + view.cx, view.cx) / TILE
    row = torch.where(ahead, view.fy * cam[:, 1] / z + view.cy, view.cy) / TILE
    return torch.stack((torch.zeros_like(row), row, col), -1)[None]


class Layer(torch.nn.Module):
    def __init__(self, width: int, heads: int, key_heads: int, head: int):
        super().__init__()
        self.heads, self.key_heads, self.head = heads, key_heads, head
        self.norm_attention = torch.nn.Parameter(torch.ones(width))
        self.norm_mlp = torch.nn.Parameter(torch.ones(width))
        self.q = torch.nn.Linear(width, heads * head, bias=False)
        self.kv = torch.nn.Linear(width, 2 * key_heads * head, bias=False)
        self.out = torch.nn.Linear(heads * head, width, bias=False)
        self.up = torch.nn.Linear(width, 4 * width, bias=False)
        self.down = torch.nn.Linear(4 * width, width, bias=False)


class GaussianDecoder(torch.nn.Module):
    """Master weights in float32, products and token operators in bfloat16."""

    def __init__(self, width: int = 256, heads: int = 4, key_heads: int = 2, layers: int = 2,
                 base: float = 100.0):
        super().__init__()
        head = width // heads
        if head % 8 or head > 128:
            raise ValueError("width / heads must be a multiple of 8 up to 128")
        self.axes = (head // 8 * 2, head // 8 * 2, head // 8 * 2)
        self.base = base
        self.embed = torch.nn.Linear(TILE * TILE * 3, width, bias=False)
        self.query = torch.nn.Linear(OUT, width, bias=False)
        self.norm_tokens = torch.nn.Parameter(torch.ones(width))
        self.norm_out = torch.nn.Parameter(torch.ones(width))
        self.layers = torch.nn.ModuleList(Layer(width, heads, key_heads, head)
                                          for _ in range(layers))
        self.head = torch.nn.Linear(width, OUT)
        torch.nn.init.zeros_(self.head.weight)
        torch.nn.init.zeros_(self.head.bias)

    @staticmethod
    def _mul(x: torch.Tensor, linear: torch.nn.Linear) -> torch.Tensor:
        return F.linear(x, linear.weight.to(x.dtype))

    def encode(self, images: torch.Tensor):
        """What the layers attend to: per layer the rotated keys and the values, [1, L, key heads,
        head]. Made once for any number of queries."""
        x, at = view_tokens(images)
        x = self._mul(x.bfloat16(), self.embed)
        x = rms_norm(x, self.norm_tokens.to(x.dtype))
        states = []
        for m in self.layers:
            kv = self._mul(x, m.kv).view(1, x.shape[1], 2, m.key_heads, m.head)
            states.append((rotary_axes(kv[:, :, 0], at, self.axes, base=self.base), kv[:, :, 1]))
        return states

    def _queries(self, params: torch.Tensor, positions: torch.Tensor):
        x = self._mul(params.bfloat16()[None], self.query)
        return x, torch.zeros_like(x)

    def forward(self, params: torch.Tensor, positions: torch.Tensor, states) -> torch.Tensor:
        """params [N, 14] (mean, quaternion, log-scale, opacity logit, SH DC) -> refined params."""
        h, add = self._queries(params, positions)
        for m, (k, v) in zip(self.layers, states):
            y, h = rms_norm(add, m.norm_attention.to(h.dtype), residual=h)
            add = self._attend(m, y, positions, k, v)
            y, h = rms_norm(add, m.norm_mlp.to(h.dtype), residual=h)
            add = self._mul(F.gelu(self._mul(y, m.up)), m.down)
        y, _ = rms_norm(add, self.norm_out.to(h.dtype), residual=h)
        return params + self.head(y[0].float())

    def _attend(self, m: Layer, y, positions, k, v):
        q = self._mul(y, m.q).view(1, y.shape[1], m.heads, m.head)
        q = rotary_axes(q, positions, self.axes, base=self.base)
        return self._mul(cross_attention(q, k, v).flatten(2), m.out)

    def prepare_8bit(self) -> list:
        """The up products' weights in e4m3 with a scale for each output, made once for `predict`."""
        prepared = []
        for m in self.layers:
            w = m.up.weight.detach()
            scale = w.abs().amax(1, keepdim=True).clamp(min=1e-12) / E4M3_MAX
            prepared.append(((w / scale).to(torch.float8_e4m3fn), scale.float()))
        return prepared

    @torch.no_grad()
    def predict(self, params: torch.Tensor, positions: torch.Tensor, states,
                prepared: list) -> torch.Tensor:
        """forward for an answer: the norm before each wide product writes 8 bits. Any number of
        queries, one included (8-bit products want rows in multiples of 16: they are padded)."""
        h, add = self._queries(params, positions)
        for m, (k, v), (w8, sw) in zip(self.layers, states, prepared):
            y, h = rms_norm(add, m.norm_attention.to(h.dtype), residual=h)
            add = self._attend(m, y, positions, k, v)
            q8, s, h = rms_norm_8bit(add, m.norm_mlp.to(h.dtype), residual=h)
            n = q8.shape[1]
            rows, scales = q8[0], s[0]
            if n % 16:
                rows = F.pad(rows.view(torch.uint8), (0, 0, 0, -n % 16)).view(q8.dtype)
                scales = F.pad(scales, (0, 0, 0, -n % 16))
            up = torch._scaled_mm(rows, w8.t(), scale_a=scales, scale_b=sw.t(),
                                  out_dtype=torch.bfloat16)[:n][None]
            add = self._mul(F.gelu(up), m.down)
        y, _ = rms_norm(add, self.norm_out.to(h.dtype), residual=h)
        return params + self.head(y[0].float())


def pack(scene) -> torch.Tensor:
    return torch.cat((scene.mu, scene.q, scene.s, scene.alpha, scene.A), 1)


def render(params: torch.Tensor, view) -> torch.Tensor:
    """The Gaussians of `params` [N, 14] in `view`, without higher SH degrees."""
    mu, q, s, alpha, A = (t.contiguous() for t in params.split((3, 4, 3, 1, 3), 1))
    k_j = torch.zeros(params.shape[0], 15, 3, device=params.device)
    return RasterizeFunction.apply(mu, q, s, torch.sigmoid(alpha), A, k_j, view.R.to(mu.device),
                                   view.T.to(mu.device), view.fx, view.fy, view.cx, view.cy,
                                   view.height, view.width)


def train(steps: int = 30, device="cuda", seed: int = 0, views: int = 3, size: int = 128,
          gaussians: int = 1024):
    """Trains a decoder to move perturbed Gaussians back to where `views` images of a synthetic
    scene show them. Returns (decoder, losses, what predict needs)."""
    from . import scenes

    dev = torch.device(device)
    torch.manual_seed(seed)
    scene = scenes.config0(seed)
    target = pack(scene)[:gaussians].to(dev)
    target[:, 7:10] += 1.0  # larger splats: fewer of them cover the image
    cams = [scenes.pinhole((4.0 * (i - 1) / max(views - 1, 1), 0.0, 4.0), size, size, float(size))
            for i in range(views)]
    with torch.no_grad():
        images = torch.stack([render(target, v) for v in cams])
    noise = torch.randn(target.shape, generator=torch.Generator("cpu").manual_seed(seed)).to(dev)
    start = target + noise * torch.tensor([0.02] * 3 + [0.1] * 4 + [0.1] * 3 + [0.5] + [0.5] * 3,
                                          device=dev)
    decoder = GaussianDecoder().to(dev)
    positions = gaussian_positions(start[:, :3], cams[0])
    opt = torch.optim.Adam(decoder.parameters(), lr=4e-4)
    losses = []
    for _ in range(steps):
        params = decoder(start, positions, decoder.encode(images))
        loss = sum(l1_ssim_loss(render(params, v), img) for v, img in zip(cams, images)) / views
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(loss.detach())
    return decoder, [float(v) for v in losses], (start, positions, images, cams)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__,
                                 formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args()
    decoder, losses, (start, positions, images, cams) = train(args.steps, seed=args.seed)
    for i in range(0, len(losses), max(1, len(losses) // 10)):
        print(f"step {i:4d}  loss {losses[i]:.5f}")
    print(f"last       loss {losses[-1]:.5f}")
    with torch.no_grad():
        states = decoder.encode(images)
        full = decoder(start, positions, states)
        answer = decoder.predict(start, positions, states, decoder.prepare_8bit())
    off = float((answer - full).norm() / (full - start).norm())
    print(f"8-bit prediction differs from the full one by {off:.3f} of the refinement")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
