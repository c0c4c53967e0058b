"""The example's decoder with rotary positions and the 8-bit cache: gradients, a token at a time
against the whole sequence, and a block over the cache against plain operations."""
import pytest
import torch

from tests import cache64, nn64
from tests.test_patch_decoder_gpu import example  # noqa: F401

pytestmark = pytest.mark.gpu


def _plain(p, rotary, positions, tokens, offsets):
    """The model's output by operations in float64 on the CPU: its own, with places turned."""
    x = tokens @ p["embed.weight"].t() + p["embed.bias"]
    o, f = offsets.tolist(), rotary.frequencies.cpu()
    for n in range(2):
        b = {k.split(".", 2)[2]: t for k, t in p.items() if k.startswith(f"blocks.{n}.")}
        y = nn64.layer_norm(x, b["norm1.weight"], b["norm1.bias"], 1e-5) @ b["qkv.weight"].t()
        q, k, v = y.view(len(x), -1, 16).split([4, 2, 2], 1)
        q, k = (cache64.turn(t, positions, f) for t in (q, k))
        x = x + nn64.attention(q, k, v, o, o, None, None, True, 0.25).flatten(1) @ b["out.weight"].t()
        y = nn64.layer_norm(x, b["norm2.weight"], b["norm2.bias"], 1e-5)
        x = x + nn64.gated(y, b["ff.gate.weight"], b["ff.up.weight"], "silu") @ b["ff.down.weight"].t()
    return nn64.layer_norm(x, p["norm.weight"], p["norm.bias"], 1e-5) @ p["head.weight"].t() + p["head.bias"]


@pytest.mark.parametrize("positions", ["places", "centres"])
def test_whole_model_against_plain_operations(example, dev, positions):  # noqa: F811
    torch.manual_seed(1)
    model = example.PatchDecoder(4, 64, 4, 2, 2, positions, device="cuda")
    tokens, offsets = torch.randn(75, 15), torch.tensor([0, 40, 41, 75])
    at = tokens[:, :3].double() if positions == "centres" else \
        torch.cat([torch.arange(n) for n in (40, 1, 34)])
    assert torch.equal(model.positions_of(tokens.to(dev), offsets.to(dev)).cpu().double(), at.double())
    leaves = {n: t.detach().cpu().double().requires_grad_(True) for n, t in model.named_parameters()}
    want = _plain(leaves, model.rotary, at, tokens.double(), offsets)
    out = model(tokens.to(dev), offsets.to(dev))
    # as without positions: a turn's rounding is one more of the operators' in float
    nn64.near(out, want.detach(), floats=1e-5)
    grad = torch.randn(75, 15)
    out.backward(grad.to(dev))
    want.backward(grad.double())
    for n, t in model.named_parameters():
        nn64.near(t.grad, leaves[n].grad, floats=5e-5)


@pytest.mark.parametrize("positions", ["places", "centres"])
def test_a_token_at_a_time_is_the_whole_sequence(example, dev, positions):  # noqa: F811
    torch.manual_seed(2)
    model = example.PatchDecoder(4, 64, 4, 2, 2, positions, device="cuda")
    made = model.generate(torch.randn(3, 15, device=dev), 20)
    offsets = torch.arange(4, device=dev) * 20
    with torch.no_grad():
        out = model(made.flatten(0, 1), offsets).view(3, 20, 15)
    # token t + 1 is what the whole sequence predicts at t; twenty steps feed on each other
    nn64.near(made[:, 1:], out[:, :-1].cpu().double(), floats=1e-4)


@pytest.mark.parametrize("positions", ["none", "places", "centres"])
def test_a_block_over_the_8_bit_cache(tpo, example, dev, positions):  # noqa: F811
    """Forty tokens one at a time: each step's attention is that of its own queries over the
    codes of the keys and values so far."""
    torch.manual_seed(3)
    model = example.PatchDecoder(4, 64, 4, 2, 1, positions, device="cuda")
    block, rotary = model.blocks[0], model.rotary
    cache = tpo.PagedCache.empty(3, 40, 2, 16, page=32, device=dev)
    plain = cache64.Cache(cache)
    one = torch.arange(4, device=dev)
    f = None if rotary is None else rotary.frequencies.cpu()
    with torch.no_grad():
        for t in range(40):
            x = torch.randn(3, 64, device=dev)
            at = torch.randn(3, 3, device=dev) if positions == "centres" else None
            cache.lengths += 1
            plain.lengths += 1
            got = block.step_paged(x, cache, one, rotary, at)
            q, k, v = (y.cpu() for y in block.project(x))
            turned = plain.append(k, v, [0, 1, 2, 3], q=q, f=f, at=None if at is None else at.cpu())
            if f is None:
                turned = q.double()
            a = plain.attention(turned, [0, 1, 2, 3])
            want = block.finish(x, a.float().to(dev))
            # the queries' turn and attention in float, through two products
            nn64.near(got, want.cpu().double(), floats=1e-5)


def test_example_runs(example, dev):  # noqa: F811
    for positions in ("places", "centres"):
        losses = example.main(["--steps", "2", "--clouds", "2", "--width", "128", "--paged",
                               "--positions", positions])
        assert len(losses) == 2 and all(x == x for x in losses)
