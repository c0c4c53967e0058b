"""An autoregressive decoder of point patches, trained and sampled with this package.

    python examples/patch_decoder.py [--steps 50] [--clouds 8] [--width 256] [--dtype bf16]

Clouds are cut into patches: furthest point samples as centres, in the order of a curve
through space, and the nearest points of each.  A transformer reads the patches of a cloud
in order and predicts the next one; the loss is the Chamfer distance to it.  Clouds have
different numbers of patches, and their tokens lie packed, one cloud after the other: layer
norm, packed attention and the gated projection see no padding.  Afterwards the model
continues clouds one patch at a time over a cache of keys and values.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(REPO, "torch-point-ops_amd"))

import torch_point_ops as tpo  # noqa: E402


class Block(torch.nn.Module):
    """Attention and gated feed-forward, each after a norm and added to what came in."""

    def __init__(self, width, heads, key_heads, **kw):
        super().__init__()
        self.heads, self.key_heads, self.size = heads, key_heads, width // heads
        self.norm1, self.norm2 = (tpo.LayerNorm(width, **kw) for _ in range(2))
        self.qkv = torch.nn.Linear(width, (heads + 2 * key_heads) * self.size, bias=False, **kw)
        self.out = torch.nn.Linear(width, width, bias=False, **kw)
        self.ff = tpo.GatedFeedForward(width, 2 * width, **kw)

    def project(self, x):
        """q, k and v as slices of one product."""
        y = self.qkv(self.norm1(x)).view(len(x), -1, self.size)
        return y.split([self.heads, self.key_heads, self.key_heads], 1)

    def finish(self, x, attended):
        x = x + self.out(attended.flatten(1))
        return x + self.ff(self.norm2(x))

    def forward(self, x, offsets):
        return self.finish(x, tpo.packed_attention(*self.project(x), offsets))

    def step(self, x, keys, values, one, rooms, used):
        """One new token of every sequence; keys and values (B, room, heads, size) get its own."""
        q, k, v = self.project(x)
        b = torch.arange(len(x), device=x.device)
        keys[b, used], values[b, used] = k, v
        a = tpo.packed_attention(q, keys.flatten(0, 1), values.flatten(0, 1), one, rooms,
                                 lengths_k=used + 1)
        return self.finish(x, a)


class PatchDecoder(torch.nn.Module):
    """Tokens (T, 3 + 3 K): a patch's centre and its points about it -> the next patch."""

    def __init__(self, points, width=256, heads=8, key_heads=2, depth=4, **kw):
        super().__init__()
        self.embed = torch.nn.Linear(3 + 3 * points, width, **kw)
        self.blocks = torch.nn.ModuleList(Block(width, heads, key_heads, **kw)
                                          for _ in range(depth))
        self.norm = tpo.LayerNorm(width, **kw)
        self.head = torch.nn.Linear(width, 3 + 3 * points, **kw)

    def forward(self, tokens, offsets):
        x = self.embed(tokens.to(self.embed.weight.dtype))
        for block in self.blocks:
            x = block(x, offsets)
        return self.head(self.norm(x)).float()

    @torch.no_grad()
    def generate(self, prompt, patches):
        """Continues each of the prompts (B, 3 + 3 K), one patch each, to `patches` patches."""
        B, dev, dt = len(prompt), prompt.device, self.embed.weight.dtype
        block = self.blocks[0]
        cache = [torch.empty(2, B, patches, block.key_heads, block.size, device=dev, dtype=dt)
                 for _ in self.blocks]
        one = torch.arange(B + 1, device=dev)
        rooms, used = one * patches, torch.zeros(B, dtype=torch.int64, device=dev)
        tokens = [prompt]
        for _ in range(patches - 1):
            x = self.embed(tokens[-1].to(dt))
            for b, (keys, values) in zip(self.blocks, cache):
                x = b.step(x, keys, values, one, rooms, used)
            tokens.append(self.head(self.norm(x)).float())
            used = used + 1
        return torch.stack(tokens, 1)


def patches_of(clouds, counts, points):
    """Packed tokens (T, 3 + 3 K) of clouds (B, P, 3), counts[b] patches each, and offsets."""
    most = max(counts)
    centres = tpo.farthest_point_sample_and_gather(clouds, most)[1]
    # along a curve: by octants of [-1, 1]^3, eight to a side
    cell = ((centres + 1) * 4).long().clamp(0, 7)
    key = sum(((cell[..., d] >> bit) & 1) << (3 * bit + d) for bit in range(3) for d in range(3))
    kept = torch.arange(most, device=clouds.device) < torch.tensor(counts, device=clouds.device)[:, None]
    order = torch.where(kept, key, 1 << 30).argsort(dim=1, stable=True)  # the first counts[b] samples
    centres = torch.gather(centres, 1, order[..., None].expand(-1, -1, 3))
    near = tpo.knn_gather(clouds, tpo.knn_points(centres, clouds, K=points)[0])
    tokens = torch.cat([centres, (near - centres[:, :, None]).flatten(2)], 2)
    offsets = torch.nn.functional.pad(torch.tensor(counts, device=clouds.device).cumsum(0), (1, 0))
    return tokens[kept], offsets


def next_patch_loss(model, tokens, offsets):
    """Chamfer distance of every patch but each cloud's first to its prediction."""
    out = model(tokens, offsets)
    there = torch.ones(len(tokens), dtype=torch.bool, device=tokens.device)
    there[offsets[1:] - 1] = False  # the last token of a cloud predicts nothing
    at = there.nonzero()[:, 0]
    want, have = tokens[at + 1], out[at]
    points = [t[:, None, :3] + t[:, 3:].unflatten(1, (-1, 3)) for t in (have, want)]
    return tpo.ChamferDistance("mean")(*points) + (have[:, :3] - want[:, :3]).square().mean()


def shapes(g, B, P, device):
    """Ellipsoid shells of random axes and centres, their points in random order."""
    d = torch.randn(B, P, 3, generator=g)
    d = d / d.norm(dim=-1, keepdim=True)
    axes = 0.3 + 0.5 * torch.rand(B, 1, 3, generator=g)
    return (d * axes + 0.2 * (torch.rand(B, 1, 3, generator=g) - 0.5)).to(device)


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--clouds", type=int, default=8)
    ap.add_argument("--points", type=int, default=16, help="points of a patch")
    ap.add_argument("--width", type=int, default=256)
    ap.add_argument("--dtype", choices=["f32", "f16", "bf16"], default="bf16")
    a = ap.parse_args(argv)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    torch.manual_seed(0)
    g = torch.Generator().manual_seed(0)
    model = PatchDecoder(a.points, a.width, device="cuda", dtype=dtype)
    # the optimiser's weights are float: half types lose small updates
    masters = [p.detach().float().requires_grad_(True) for p in model.parameters()]
    optimiser = torch.optim.AdamW(masters, lr=1e-3)
    losses = []
    for step in range(a.steps):
        clouds = shapes(g, a.clouds, 2048, "cuda")
        counts = torch.randint(24, 97, (a.clouds,), generator=g).tolist()
        loss = next_patch_loss(model, *patches_of(clouds, counts, a.points))
        model.zero_grad()
        loss.backward()
        for m, p in zip(masters, model.parameters()):
            m.grad = p.grad.float()
        optimiser.step()
        with torch.no_grad():
            for m, p in zip(masters, model.parameters()):
                p.copy_(m)
        losses.append(loss.item())
        if step % 10 == 0 or step == a.steps - 1:
            print(f"step {step}: loss {losses[-1]:.4f}", flush=True)
    tokens, offsets = patches_of(shapes(g, 4, 2048, "cuda"), [32] * 4, a.points)
    made = model.generate(tokens[offsets[:-1]], 32)
    print(f"generated {tuple(made.shape)}: four clouds of 32 patches of {a.points} points")
    return losses


if __name__ == "__main__":
    main()
