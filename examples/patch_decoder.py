"""An autoregressive decoder of point patches, trained and sampled with this package.

    python examples/patch_decoder.py [--steps 50] [--clouds 8] [--width 256] [--dtype bf16]
        [--positions none|places|centres] [--paged]

Clouds are cut into patches: furthest point samples as centres, in the order of a curve
through space, and the nearest points of each.  A transformer reads the patches of a cloud
in order and predicts the next one; the loss is the Chamfer distance to it.  Clouds have
different numbers of patches, and their tokens lie packed, one cloud after the other: layer
norm, packed attention and the gated projection see no padding.  Afterwards the model
continues clouds one patch at a time over a cache of keys and values, with --paged one of
8 bits in pages.  With --positions queries and keys are turned by the patches' places in their
clouds, or by their centres' coordinates.
"""
from __future__ import annotations

import argparse
import math
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

    def project(self, x, rotary=None, positions=None):
        """q, k and v as slices of one product, queries and keys turned by their positions."""
        y = self.qkv(self.norm1(x)).view(len(x), -1, self.size)
        if rotary is None:
            return y.split([self.heads, self.key_heads, self.key_heads], 1)
        qk, v = y.split([self.heads + self.key_heads, self.key_heads], 1)
        return *rotary(qk, positions).split([self.heads, self.key_heads], 1), v

    def finish(self, x, attended):
        x = x + self.out(attended.flatten(1))
        return x + self.ff(self.norm2(x))

    def forward(self, x, offsets, rotary=None, positions=None):
        return self.finish(x, tpo.packed_attention(*self.project(x, rotary, positions), offsets))

    def step(self, x, keys, values, one, rooms, used, rotary=None, positions=None):
        """One new token of every sequence; keys and values (B, room, heads, size) get its own."""
        q, k, v = self.project(x, rotary, positions)
        b = torch.arange(len(x), device=x.device)
        keys[b, used], values[b, used] = k, v
        a = tpo.packed_attention(q, keys.flatten(0, 1), values.flatten(0, 1), one, rooms,
                                 lengths_k=used + 1)
        return self.finish(x, a)

    def step_paged(self, x, cache, one, rotary=None, positions=None):
        """One new token of every sequence; the cache, whose lengths count it already, gets its
        key and value."""
        q, k, v = self.project(x)
        if rotary is None:
            tpo.cache_append(cache, k, v, one)
        else:
            q = tpo.cache_append(cache, k, v, one, q, rotary.frequencies, positions)
        return self.finish(x, tpo.cached_attention(q, cache, one))


class PatchDecoder(torch.nn.Module):
    """Tokens (T, 3 + 3 K): a patch's centre and its points about it -> the next patch.

    positions: "none", or what queries and keys are turned by: "places" of tokens in their
    sequences, or the coordinates of patches' "centres".
    """

    def __init__(self, points, width=256, heads=8, key_heads=2, depth=4, positions="none", **kw):
        super().__init__()
        size, dev = width // heads, kw.get("device")
        self.positions, self.rotary = positions, None
        if positions == "places":
            self.rotary = tpo.RotaryPositions(size // 2 * 2, device=dev)
        elif positions == "centres":  # (half a turn and more over [-1, 1], finer by octaves)
            octaves = 2.0 ** torch.arange(size // 6, dtype=torch.float64)
            self.rotary = tpo.RotaryPositions(
                size // 6 * 6, frequencies=(math.pi / 2 * octaves).repeat(3), device=dev)
        self.embed = torch.nn.Linear(3 + 3 * points, width, **kw)
        self.blocks = torch.nn.ModuleList(Block(width, heads, key_heads, **kw)
                                          for _ in range(depth))
        self.norm = tpo.LayerNorm(width, **kw)
        self.head = torch.nn.Linear(width, 3 + 3 * points, **kw)

    def positions_of(self, tokens, offsets):
        """What the tokens of packed sequences are turned by."""
        if self.positions == "centres":
            return tokens[:, :3].float().contiguous()
        if self.positions == "places":
            at = torch.arange(len(tokens), device=tokens.device)
            return at - offsets[torch.searchsorted(offsets, at, right=True) - 1]
        return None

    def forward(self, tokens, offsets):
        x = self.embed(tokens.to(self.embed.weight.dtype))
        positions = self.positions_of(tokens, offsets)
        for block in self.blocks:
            x = block(x, offsets, self.rotary, positions)
        return self.head(self.norm(x)).float()

    @torch.no_grad()
    def generate(self, prompt, patches, paged=False):
        """Continues each of the prompts (B, 3 + 3 K), one patch each, to `patches` patches.
        paged: over caches of 8 bits in pages."""
        B, dev, dt = len(prompt), prompt.device, self.embed.weight.dtype
        block = self.blocks[0]
        if paged:
            return self.generate_paged(prompt, patches)
        cache = [torch.empty(2, B, patches, block.key_heads, block.size, device=dev, dtype=dt)
                 for _ in self.blocks]
        one = torch.arange(B + 1, device=dev)
        rooms, used = one * patches, torch.zeros(B, dtype=torch.int64, device=dev)
        tokens = [prompt]
        for _ in range(patches - 1):
            x = self.embed(tokens[-1].to(dt))
            at = used if self.positions == "places" else self.positions_of(tokens[-1], one)
            for b, (keys, values) in zip(self.blocks, cache):
                x = b.step(x, keys, values, one, rooms, used, self.rotary, at)
            tokens.append(self.head(self.norm(x)).float())
            used = used + 1
        return torch.stack(tokens, 1)

    @torch.no_grad()
    def generate_paged(self, prompt, patches):
        B, dev, dt = len(prompt), prompt.device, self.embed.weight.dtype
        caches = [tpo.PagedCache.empty(B, patches, b.key_heads, b.size, page=32, device=dev)
                  for b in self.blocks]
        one, tokens = torch.arange(B + 1, device=dev), [prompt]
        for _ in range(patches - 1):
            x = self.embed(tokens[-1].to(dt))
            # (places are the cache's to know)
            at = self.positions_of(tokens[-1], one) if self.positions == "centres" else None
            for b, cache in zip(self.blocks, caches):
                cache.lengths += 1
                x = b.step_paged(x, cache, one, self.rotary, at)
            tokens.append(self.head(self.norm(x)).float())
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
    ap.add_argument("--positions", choices=["none", "places", "centres"], default="none")
    ap.add_argument("--paged", action="store_true", help="generate over an 8-bit cache in pages")
    a = ap.parse_args(argv)
    dtype = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    torch.manual_seed(0)
    g = torch.Generator().manual_seed(0)
    model = PatchDecoder(a.points, a.width, positions=a.positions, device="cuda", dtype=dtype)
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
    made = model.generate(tokens[offsets[:-1]], 32, a.paged)
    print(f"generated {tuple(made.shape)}: four clouds of 32 patches of {a.points} points")
    return losses


if __name__ == "__main__":
    main()
