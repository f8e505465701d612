"""Trains a token network that predicts Gaussians from image patches, through the
rasterizer, on synthetic images:

    python -m blitzgs_amd.examples.train_predictor [--steps N]

A scene is one or two views; their patches are tokens of one sequence.  Two
blocks of layer normalisation, attention (eight query heads on two key heads,
normalised and rotated to their patch's row and column, scenes of unequal length
in one padded batch) and a gated feed-forward turn each token of the first view
into four Gaussians, which are rendered and compared with that view by L1 and
SSIM.  The weight matrices take orthogonalised updates, all other parameters
AdamW's, with moments in 8 bits."""
import argparse
import math

import numpy as np
import torch
from torch import nn

from .. import synth
from ..adamw import AdamW
from ..attention import attention
from ..feedforward import feed_forward
from ..norm import layer_norm
from ..orthogonal import OrthogonalMomentum
from ..rasterizer import GaussianRasterizationSettings, GaussianRasterizer
from ..rotary import norm_rotate, rotary_frequencies
from ..ssim import fused_ssim

SIDE, PATCH, PER_TOKEN = 128, 8, 4
GRID = SIDE // PATCH
TOKENS = GRID * GRID
DISTANCE, FOV = 4.0, math.radians(50.0)
HALF = DISTANCE * math.tan(FOV / 2)          # half the image's side on the plane z = 0


def _matrix(rows, columns):
    return nn.Parameter(torch.randn(rows, columns) / math.sqrt(columns))


class Block(nn.Module):
    """x + attention(norm(x)), then x + gated(norm(x)); activations in bfloat16."""

    def __init__(self, width, heads, key_heads):
        super().__init__()
        self.heads, self.key_heads, self.head_dim = heads, key_heads, width // heads
        self.norm1, self.norm2 = nn.Parameter(torch.ones(width)), nn.Parameter(torch.ones(width))
        self.norm_q, self.norm_k = (nn.Parameter(torch.ones(self.head_dim)) for _ in range(2))
        self.qkv = _matrix((heads + 2 * key_heads) * self.head_dim, width)
        self.proj = _matrix(width, width)
        self.gate, self.up, self.down = _matrix(2 * width, width), _matrix(2 * width, width), _matrix(width, 2 * width)

    def forward(self, x, key_lengths, places, frequencies):
        B, T, _ = x.shape
        mul = lambda a, w: a @ w.t().to(a.dtype)  # noqa: E731
        qkv = mul(layer_norm(x, self.norm1), self.qkv).view(B, T, -1, self.head_dim)
        q, k, v = qkv.split([self.heads, self.key_heads, self.key_heads], 2)
        q, k = norm_rotate(q.transpose(1, 2), k.transpose(1, 2), self.norm_q, self.norm_k, places, frequencies)
        o = attention(q, k, v.transpose(1, 2), key_lengths=key_lengths)
        x = x + mul(o.transpose(1, 2).reshape(B, T, -1), self.proj)
        return x + feed_forward(layer_norm(x, self.norm2), *(w.to(x.dtype) for w in (self.gate, self.up, self.down)))


class Predictor(nn.Module):
    """(B, T, 3 PATCH^2) patches to the first view's Gaussians, as the rasterizer takes them."""

    def __init__(self, width=256, depth=2, heads=8, key_heads=2, views=2):
        super().__init__()
        self.embed = _matrix(width, 3 * PATCH * PATCH)
        self.position = nn.Parameter(0.02 * torch.randn(views * TOKENS, width))
        self.blocks = nn.ModuleList(Block(width, heads, key_heads) for _ in range(depth))
        self.norm_weight, self.norm_bias = nn.Parameter(torch.ones(width)), nn.Parameter(torch.zeros(width))
        self.head = nn.Parameter(0.02 * torch.randn(PER_TOKEN * 14, width))
        at = (torch.arange(GRID) + 0.5) * 2 / GRID - 1
        y, x = torch.meshgrid(at, at, indexing="ij")
        row, column = torch.meshgrid(torch.arange(GRID), torch.arange(GRID), indexing="ij")
        self.register_buffer("places", torch.stack([row, column], -1).reshape(TOKENS, 2).repeat(views, 1))
        # half of a head's pairs turn with the row, half with the column
        self.register_buffer("frequencies", rotary_frequencies(width // heads // 4, base=100.0, axes=2, device="cpu"))
        self.register_buffer("centre", HALF * torch.stack([x, y, torch.zeros_like(x)], -1).reshape(TOKENS, 1, 3))

    def matrices(self):
        return [p for n, p in self.named_parameters() if p.dim() == 2 and n not in ("position", "head")]

    def others(self):
        ours = {id(p) for p in self.matrices()}
        return [p for p in self.parameters() if id(p) not in ours]

    def forward(self, patches, key_lengths):
        x = (patches @ self.embed.t() + self.position[:patches.shape[1]]).to(torch.bfloat16)
        for block in self.blocks:
            x = block(x, key_lengths, self.places[:x.shape[1]], self.frequencies)
        x = layer_norm(x[:, :TOKENS], self.norm_weight, self.norm_bias).float() @ self.head.t()
        move, scale, turn, opacity, colour = x.view(-1, TOKENS, PER_TOKEN, 14).split([3, 3, 4, 1, 3], -1)
        P = TOKENS * PER_TOKEN
        step = 2 * HALF / GRID
        return [dict(means3D=(self.centre + step * torch.tanh(m)).reshape(P, 3),
                     scales=(0.4 * step * torch.exp(s.clamp(-3, 1))).reshape(P, 3),
                     rotations=nn.functional.normalize(t + t.new_tensor([1.0, 0, 0, 0]), dim=-1).reshape(P, 4),
                     opacities=torch.sigmoid(a).reshape(P, 1), shs=c.reshape(P, 1, 3))
                for m, s, t, a, c in zip(move, scale, turn, opacity, colour)]


def images(count, generator, device):
    """Smooth random images (count, 3, SIDE, SIDE) in [0, 1]."""
    at = torch.linspace(0, 1, SIDE, device=device)
    f = 1 + 3 * torch.rand((count, 3, 2, 1, 1), generator=generator, device=device)
    p = 2 * math.pi * torch.rand((count, 3, 2, 1, 1), generator=generator, device=device)
    return 0.5 + 0.25 * (torch.sin(2 * math.pi * f[:, :, 0] * at + p[:, :, 0])
                         + torch.cos(2 * math.pi * f[:, :, 1] * at[:, None] + p[:, :, 1]))


def patches_of(views):
    """(V, 3, SIDE, SIDE) to (V TOKENS, 3 PATCH^2)."""
    v = views.unfold(2, PATCH, PATCH).unfold(3, PATCH, PATCH)
    return v.permute(0, 2, 3, 1, 4, 5).reshape(-1, 3 * PATCH * PATCH)


def rasterizer(device):
    cam = synth.make_camera(np.eye(3), (0.0, 0.0, -DISTANCE), SIDE, SIDE, FOV)
    t = lambda a: torch.as_tensor(np.ascontiguousarray(a), device=device)  # noqa: E731
    return GaussianRasterizer(GaussianRasterizationSettings(
        image_height=SIDE, image_width=SIDE, tanfovx=cam["tanfovx"], tanfovy=cam["tanfovy"],
        bg=torch.full((3,), 0.5, device=device), scale_modifier=1.0, viewmatrix=t(cam["viewmatrix"]),
        projmatrix=t(cam["projmatrix"]), sh_degree=0, campos=t(cam["campos"]), prefiltered=False, debug=False))


def render(raster, g):
    args = {"avoid_pixel_all2all": False, "stats_collector": {}}
    means2D, rgb, conic, radii, depths = raster.preprocess_gaussians(g["means3D"], g["scales"], g["rotations"],
                                                                     g["shs"], g["opacities"], args)
    P = means2D.shape[0]
    empty = lambda c, grad: torch.zeros((P, c), device=means2D.device, requires_grad=grad)  # noqa: E731
    return raster.render_gaussians(means2D, empty(3, True), conic, rgb, empty(5, False), depths, radii, None, None,
                                   args)[0]


def train(steps=60, seed=0, device="cuda", report=None):
    """The losses of `steps` training steps."""
    torch.manual_seed(seed)
    g = torch.Generator(device=device).manual_seed(seed)
    net, raster = Predictor().to(device), rasterizer(device)
    opt = [OrthogonalMomentum(net.matrices(), lr=0.01), AdamW(net.others(), lr=2e-3, weight_decay=0.0, bits=8)]
    # two scenes: one of two views, one of a single view, whose second half is padding
    scenes = [images(2, g, device), images(1, g, device)]
    tokens = [patches_of(v) for v in scenes]
    lengths = torch.tensor([len(t) for t in tokens], dtype=torch.int32, device=device)
    batch = nn.utils.rnn.pad_sequence(tokens, batch_first=True)
    target = torch.stack([v[0] for v in scenes])
    losses = []
    for step in range(steps):
        for o in opt:
            o.zero_grad(set_to_none=True)
        image = torch.stack([render(raster, gaussians) for gaussians in net(batch, lengths)])
        loss = 0.8 * (image - target).abs().mean() + 0.2 * (1.0 - fused_ssim(image, target))
        loss.backward()
        for o in opt:
            o.step()
        losses.append(loss.item())
        if report:
            report(step, losses[-1])
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=60)
    steps = ap.parse_args().steps
    train(steps, report=lambda i, loss: print(f"step {i}: loss {loss:.4f}", flush=True)
          if i % 10 == 0 or i + 1 == steps else None)


if __name__ == "__main__":
    main()
