"""The transformer operators inside torch's own machinery: opcheck, torch.compile, vmap,
checkpointing, hooks."""
import pytest
import torch
from torch.library import opcheck

from tests import nn64

pytestmark = pytest.mark.gpu


def _cases(dev, dtype):
    """name: operator, differentiable inputs, other arguments."""
    g = torch.Generator().manual_seed(7)

    def r(*shape):
        return torch.randn(*shape, generator=g).to(dev, dtype).requires_grad_(True)

    o = torch.tensor([0, 9, 20], device=dev)
    n = torch.tensor([9, 4], device=dev)
    ops = torch.ops
    return {
        "layer_norm": (ops.torch_point_ops_norm.layer_norm, [r(2, 10, 48), r(48), r(48)], (1e-5,)),
        "packed_attention": (ops.torch_point_ops_attention.packed_attention,
                             [r(20, 4, 32), r(20, 2, 32), r(20, 2, 32)],
                             (o, o, None, n, True, 32 ** -0.5)),
        "gated_projection": (ops.torch_point_ops_gated.gated_projection,
                             [r(2, 10, 48), r(40, 48), r(40, 48)], (0,)),
    }


NAMES = ["layer_norm", "packed_attention", "gated_projection"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_opcheck(tpo, dev, name, dtype):
    op, ins, more = _cases(dev, dtype)[name]
    opcheck(op.default, (*ins, *more), raise_exception=True)
    opcheck(op.default, (*[t.detach() for t in ins], *more), raise_exception=True)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled(tpo, dev, name, dtype):
    op, ins, more = _cases(dev, dtype)[name]
    f = torch.compile(lambda *a: op(*a, *more))
    want, got = op(*ins, *more), f(*ins)
    assert torch.equal(got, want)
    g = torch.randn_like(want)
    for a, b in zip(torch.autograd.grad(got, ins, g), torch.autograd.grad(want, ins, g)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("name", NAMES)
def test_vmap(tpo, dev, name):
    """Without gradients the operators run under vmap, one slice after another."""
    op, ins, more = _cases(dev, torch.float32)[name]
    x, *rest = [t.detach() for t in ins]
    xs = torch.stack([x, 2 * x, -x])
    got = torch.vmap(lambda t: op(t, *rest, *more))(xs)
    assert torch.equal(got, torch.stack([op(t, *rest, *more) for t in xs]))


@pytest.mark.parametrize("name", NAMES)
def test_checkpoint_and_hooks(tpo, dev, name):
    from torch.utils.checkpoint import checkpoint

    op, ins, more = _cases(dev, torch.bfloat16)[name]
    want = torch.autograd.grad(op(*ins, *more).float().square().sum(), ins)
    y = checkpoint(lambda *a: op(*a, *more), *ins, use_reentrant=False)
    got = torch.autograd.grad(y.float().square().sum(), ins)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    seen, packed = [], []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (packed.append(1), t.cpu())[1],
                                                  lambda t: t.to(dev)):
        y = op(*ins, *more)
    ins[0].register_hook(lambda g: seen.append(g))
    got = torch.autograd.grad(y.float().square().sum(), ins)
    assert packed and len(seen) == 1 and torch.equal(seen[0], want[0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_one_gradient_flows_through_all(tpo, dev):
    """A block of the three under autograd with inputs that are views and used twice."""
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(30, 64, generator=g), torch.randn(96, 64, generator=g) / 8
    wu = torch.randn(96, 64, generator=g) / 8
    o = [0, 12, 30]

    def plain(x, w, wu):
        n = nn64.layer_norm(x, None, None, 1e-5).view(30, 2, 32)
        a = nn64.attention(n, n, n, o, o, None, None, True, 32 ** -0.5).flatten(1)
        return nn64.gated(a + x, w, wu, "gelu")

    gy = torch.randn(30, 96, generator=g)
    want, gwant = nn64.grads(plain, (x, w, wu), gy)
    X, W, U = ins = [t.to(dev).requires_grad_(True) for t in (x, w, wu)]
    n = tpo.layer_norm(X).view(30, 2, 32)
    a = tpo.packed_attention(n, n, n, torch.tensor(o, device=dev)).flatten(1)
    y = tpo.gated_projection(a + X, W, U, "gelu")
    nn64.near(y, want, floats=5e-6)
    for got, e in zip(torch.autograd.grad(y, ins, gy.to(dev)), gwant):
        nn64.near(got, e, floats=2e-5)
