"""The example's decoder: it learns, its gradients are those of plain operations, and tokens
one at a time over the cache give what the whole sequence gives."""
import importlib.util
import os

import pytest
import torch

from tests import nn64
from tests.conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(tpo):
    spec = importlib.util.spec_from_file_location(
        "patch_decoder", os.path.join(REPO, "examples", "patch_decoder.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _plain(model, tokens, offsets):
    """The model's output by operations in float64 on the CPU."""
    p = {n: t for n, t in model.items()}
    x = tokens @ p["embed.weight"].t() + p["embed.bias"]
    o = offsets.tolist()
    n = 0
    while f"blocks.{n}.qkv.weight" in p:
        b = {k.split(".", 2)[2]: t for k, t in p.items() if k.startswith(f"blocks.{n}.")}
        y = nn64.layer_norm(x, b["norm1.weight"], b["norm1.bias"], 1e-5) @ b["qkv.weight"].t()
        q, k, v = y.view(len(x), -1, 16).split([4, 2, 2], 1)
        x = x + nn64.attention(q, k, v, o, o, None, None, True, 0.25).flatten(1) @ b["out.weight"].t()
        y = nn64.layer_norm(x, b["norm2.weight"], b["norm2.bias"], 1e-5)
        x = x + nn64.gated(y, b["ff.gate.weight"], b["ff.up.weight"], "silu") @ b["ff.down.weight"].t()
        n += 1
    return nn64.layer_norm(x, p["norm.weight"], p["norm.bias"], 1e-5) @ p["head.weight"].t() + p["head.bias"]


def test_whole_model_against_plain_operations(example, dev):
    torch.manual_seed(1)
    model = example.PatchDecoder(4, 64, 4, 2, 2, device="cuda")
    tokens, offsets = torch.randn(75, 15), torch.tensor([0, 40, 41, 75])
    leaves = {n: t.detach().cpu().double().requires_grad_(True) for n, t in model.named_parameters()}
    want = _plain(leaves, tokens.double(), offsets)
    out = model(tokens.to(dev), offsets.to(dev))
    # three operators a layer, two layers, in float
    nn64.near(out, want.detach(), floats=1e-5)
    grad = torch.randn(75, 15)
    out.backward(grad.to(dev))
    want.backward(grad.double())
    for n, t in model.named_parameters():
        nn64.near(t.grad, leaves[n].grad, floats=5e-5)


def test_a_token_at_a_time_is_the_whole_sequence(example, dev):
    torch.manual_seed(2)
    model = example.PatchDecoder(4, 64, 4, 2, 2, device="cuda")
    made = model.generate(torch.randn(3, 15, device=dev), 20)
    offsets = torch.arange(4, device=dev) * 20
    with torch.no_grad():
        out = model(made.flatten(0, 1), offsets).view(3, 20, 15)
    # token t + 1 is what the whole sequence predicts at t; twenty steps feed on each other
    nn64.near(made[:, 1:], out[:, :-1].cpu().double(), floats=1e-4)


def test_example_learns(example, dev):
    losses = example.main(["--steps", "30", "--clouds", "4", "--width", "128"])
    assert sum(losses[-5:]) < 0.7 * sum(losses[:5])
