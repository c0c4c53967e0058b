"""layer_norm where the float range ends, and rows of all widths over few workgroups."""
import pytest
import torch

from tests import nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


# widths that leave lanes without a value, in every build of the backward, and one that
# leaves none; powers of two, and levels of few bits, so that sums of equal values are exact
@pytest.mark.parametrize("width", [16, 64, 128, 256, 512, 2048, 16384])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_constant_rows_of_any_size(tpo, dev, width, dtype):
    """Equal values are their own mean whatever their size: the gradient is the row's
    1 / sqrt(eps) times the output gradient less its mean."""
    level = 2.0 ** (126 - width.bit_length())  # the largest whose sum over a row is a float
    x = torch.tensor([level, -level, 0.0, 2.0 ** 60])[:, None].expand(4, width).to(dtype)
    g = torch.Generator().manual_seed(width)
    gy = torch.randn(4, width, generator=g).to(dtype)
    w = torch.ones(width, dtype=dtype, device=dev, requires_grad=True)
    X = x.to(dev).contiguous().requires_grad_(True)
    y = tpo.layer_norm(X, w)
    gx, gw = torch.autograd.grad(y, (X, w), gy.to(dev))
    assert (y == 0).all() and (gw == 0).all()
    d = gy.double()
    nn64.near(gx, (d - d.mean(1, keepdim=True)) / 1e-5 ** 0.5, floats=4e-6)


# a row a workgroup, two, several; one wave a row and sixteen; each set of results
@pytest.mark.parametrize("shape", [(1, 8192), (3, 1100), (129, 8192), (130, 2100), (257, 16384),
                                   (513, 1500), (1100, 700), (2300, 4100)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_over_workgroups(tpo, dev, shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x, gy = (torch.randn(*shape, generator=g).to(dtype) for _ in range(2))
    w, b = ((f + 0.2 * torch.randn(shape[1], generator=g)).to(dtype) for f in (1, 0))
    _, want = nn64.grads(lambda x, w, b: nn64.layer_norm(x, w, b, 1e-5), (x, w, b), gy)
    ins = [t.to(dev).requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(tpo.layer_norm(*ins), ins, gy.to(dev))
    for a, e in zip(got, want):
        # sums over the rows of terms of either sign
        nn64.near(a, e, floats=2e-6 + 1e-7 * x.numel() ** 0.5 / max(1.0, e.norm().item()))
    X = ins[0].detach().requires_grad_(True)
    alone, = torch.autograd.grad(tpo.layer_norm(X, *[t.detach() for t in ins[1:]]), X, gy.to(dev))
    assert torch.equal(alone, got[0])
