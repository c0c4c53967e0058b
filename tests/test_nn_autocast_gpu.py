"""The transformer operators under torch.autocast: float parameters, inputs of either type."""
import pytest
import torch

from tests import nn64

pytestmark = pytest.mark.gpu
HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("half", HALVES)
@pytest.mark.parametrize("given", ["half", "float"])
def test_gated_feed_forward(tpo, dev, half, given):
    g = torch.Generator().manual_seed(1)
    m = tpo.GatedFeedForward(64, 96, "gelu", device=dev)
    x = torch.randn(30, 64, generator=g).to(half)
    gy = torch.randn(30, 64, generator=g).to(half)
    names = [n for n, _ in m.named_parameters()]
    W = [p.detach().cpu().to(half) for _, p in m.named_parameters()]
    X = x.to(dev, half if given == "half" else torch.float32).requires_grad_(True)
    with torch.autocast("cuda", half):
        y = m(X)
    assert y.dtype == half
    want, gwant = nn64.grads(lambda x, a, b, c: nn64.gated(x, a, b, "gelu") @ c.t(), (x, *W), gy)
    # h, then the result of the product with the third weight
    nn64.near(y, want, roundings=2)
    y.backward(gy.to(dev))
    assert names == ["gate.weight", "up.weight", "down.weight"]
    # gradients come back in the parameters' type; h, its gradient and those at the two
    # projections are rounded between the products
    for got, e in zip([X.grad] + [p.grad for p in m.parameters()], gwant):
        assert got.dtype == (X.dtype if got is X.grad else torch.float32)
        nn64.near(got.to(half), e, roundings=4)


@pytest.mark.parametrize("half", HALVES)
def test_attention_of_mixed_types(tpo, dev, half):
    """Queries and keys that a float operation left in float, values in the half type."""
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(50, h, 32, generator=g).to(half) for h in (4, 2, 2))
    go = torch.randn(50, 4, 32, generator=g).to(half)
    o = [0, 20, 50]
    idx = torch.tensor(o, device=dev)
    ins = [t.to(dev, d).requires_grad_(True)
           for t, d in ((q, torch.float32), (k, torch.float32), (v, half))]
    with pytest.raises(RuntimeError, match="one type"):
        tpo.packed_attention(*ins, idx)
    with torch.autocast("cuda", half):
        out = tpo.packed_attention(*ins, idx)
    assert out.dtype == half
    want, gwant = nn64.grads(
        lambda a, b, c: nn64.attention(a, b, c, o, o, None, None, True, 32 ** -0.5), (q, k, v), go)
    nn64.near(out, want, roundings=2)
    for a, e, t in zip(torch.autograd.grad(out, ins, go.to(dev)), gwant, ins):
        assert a.dtype == t.dtype
        nn64.near(a.to(half), e, roundings=3, floats=1e-5)


@pytest.mark.parametrize("half", HALVES)
def test_layer_norm_between_types(tpo, dev, half):
    """Float weights, x as it comes: the result is of x's type with autocast and without."""
    g = torch.Generator().manual_seed(3)
    m = tpo.LayerNorm(96, device=dev)
    x = torch.randn(20, 96, generator=g)
    for t in (half, torch.float32):
        X = x.to(dev, t)
        with torch.autocast("cuda", half):
            y = m(X)
        assert y.dtype == t and torch.equal(y, m(X))


def test_autocast_leaves_double_refused(tpo, dev):
    x, w = torch.ones(4, 16, device=dev).double(), torch.ones(8, 16, device=dev).double()
    with torch.autocast("cuda", torch.bfloat16):
        with pytest.raises(RuntimeError, match="not implemented for"):
            tpo.gated_projection(x, w, w)
