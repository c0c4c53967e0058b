"""layer_norm against its definition in float64: values, gradients, layouts, refusals."""
import pytest
import torch

from tests import nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(shape, dtype, weights, seed, shift=0.3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * 1.5 + shift
    wt = {"none": None, "same": dtype, "float": torch.float32}[weights]
    w = b = None
    if wt is not None:
        w = (1 + 0.2 * torch.randn(shape[-1], generator=g)).to(wt)
        b = (0.2 * torch.randn(shape[-1], generator=g)).to(wt)
    return x.to(dtype), w, b, torch.randn(*shape, generator=g).to(dtype)


def _on(dev, *ts, grad=True):
    return [t if t is None else t.to(dev).requires_grad_(grad) for t in ts]


# one value, odd widths, the edges of a wave's loads, rows held in registers or
# not; one row, a few, many
@pytest.mark.parametrize("shape", [(1, 1), (3, 2), (5, 63), (1, 64), (7, 65), (4, 255), (130, 256),
                                   (3, 511), (2, 3, 512), (9, 771), (257, 1000), (17, 1024),
                                   (6, 2047), (5, 4104), (3, 8192), (2, 8193), (4, 20000),
                                   (1500, 96), (5000, 8)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weights", ["none", "same", "float"])
def test_values_and_gradients(tpo, dev, shape, dtype, weights):
    x, w, b, gy = _inputs(shape, dtype, weights, sum(shape))
    eps = 1e-5
    ins = [t for t in (x, w, b) if t is not None]
    want, gwant = nn64.grads(lambda x, *p: nn64.layer_norm(x, *(p or (None, None)), eps), ins, gy)
    X, W, B = _on(dev, x, w, b)
    y = tpo.layer_norm(X, W, B, eps)
    assert y.dtype == dtype
    nn64.near(y, want)
    with torch.no_grad():
        assert torch.equal(tpo.layer_norm(X, W, B, eps), y)
    got = torch.autograd.grad(y, [t for t in (X, W, B) if t is not None], gy.to(dev))
    if shape[-1] == 1:  # x is its own mean: nothing but rounding
        assert got[0].abs().max() <= 1e-2
        got, gwant = got[1:], gwant[1:]
    for a, e in zip(got, gwant):
        # sums over the rows of terms of either sign
        nn64.near(a, e, floats=2e-6 + 1e-7 * x.numel() ** 0.5 / max(1.0, e.norm().item()))


# rows that several waves hold, the last of them in part, and more rows than workgroups
@pytest.mark.parametrize("shape", [(600, 1030), (700, 1500), (300, 2048), (600, 2049), (300, 2500),
                                   (600, 4097), (600, 5000), (300, 9000), (300, 16384), (70, 16390),
                                   (70, 32769)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_rows(tpo, dev, shape, dtype):
    x, w, b, gy = _inputs(shape, dtype, "same", sum(shape))
    want, gwant = nn64.grads(lambda x, w, b: nn64.layer_norm(x, w, b, 1e-5), (x, w, b), gy)
    X, W, B = _on(dev, x, w, b)
    y = tpo.layer_norm(X, W, B)
    nn64.near(y, want)
    for a, e in zip(torch.autograd.grad(y, (X, W, B), gy.to(dev)), gwant):
        # sums over the rows of terms of either sign
        nn64.near(a, e, floats=2e-6 + 1e-7 * x.numel() ** 0.5 / max(1.0, e.norm().item()))


def test_each_gradient_alone(tpo, dev):
    x, w, b, gy = _inputs((37, 200), torch.bfloat16, "same", 5)
    X, W, B = _on(dev, x, w, b)
    full = torch.autograd.grad(tpo.layer_norm(X, W, B), (X, W, B), gy.to(dev))
    for at in range(3):
        part = [t.detach().requires_grad_(i == at) for i, t in enumerate((X, W, B))]
        g, = torch.autograd.grad(tpo.layer_norm(*part), part[at], gy.to(dev))
        assert torch.equal(g, full[at])
    # a bias without a weight, a weight without a bias
    B2, W2 = B.detach().requires_grad_(True), W.detach().requires_grad_(True)
    g, = torch.autograd.grad(tpo.layer_norm(X.detach(), None, B2), B2, gy.to(dev))
    assert torch.equal(g, full[2])
    g, = torch.autograd.grad(tpo.layer_norm(X.detach(), W2, None), W2, gy.to(dev))
    assert torch.equal(g, full[1])


def test_gradient_against_differences(tpo, dev):
    x, w, b, gy = _inputs((6, 40), torch.float32, "same", 9)
    X, W, B = _on(dev, x, w, b)
    got = torch.autograd.grad(tpo.layer_norm(X, W, B), (X, W, B), gy.to(dev))
    g = torch.Generator().manual_seed(1)
    for at in range(3):
        d = [torch.randn(t.shape, generator=g, dtype=torch.float64) * (i == at)
             for i, t in enumerate((x, w, b))]
        want = nn64.slope(lambda x, w, b: (nn64.layer_norm(x, w, b, 1e-5) * gy.double()).sum(),
                          [t.double() for t in (x, w, b)], d, 1e-5)
        have = (got[at].cpu().double() * d[at]).sum()
        # the difference quotient is good to 1e-8; the float gradient to 1e-6 of its norm
        assert abs(have - want) <= 1e-5 * got[at].norm().item() * d[at].norm().item()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_far_from_zero(tpo, dev, dtype):
    """The variance is taken about the mean: a large level costs nothing beyond x's own type."""
    x, w, b, _ = _inputs((64, 384), dtype, "same", 3, shift=1000.0)
    nn64.near(tpo.layer_norm(*_on(dev, x, w, b, grad=False)), nn64.layer_norm(x, w, b, 1e-5),
              floats=1e-4)  # x - mean cancels 1000 to 1.5: 2^-24 * 1000 of it


def test_constant_and_nonfinite_rows(tpo, dev):
    x = torch.zeros(4, 100)
    x[1] = 7.0
    x[2, 50] = float("nan")
    x[3, 7] = float("inf")
    y = tpo.layer_norm(x.to(dev)).cpu()
    assert (y[:2] == 0).all()
    assert y[2:].isnan().all()


def test_layouts_streams_and_empty(tpo, dev):
    g = torch.Generator().manual_seed(4)
    big = torch.randn(70, 33, generator=g)
    w = torch.randn(33, 2, generator=g)
    want = nn64.layer_norm(big.t()[:, 1:69], None, None, 1e-5)
    nn64.near(tpo.layer_norm(big.to(dev).t()[:, 1:69]), want)  # strided, unaligned rows
    nn64.near(tpo.layer_norm(big.to(dev)[1:], w.to(dev)[:, 1]),
              nn64.layer_norm(big[1:], w[:, 1], None, 1e-5))
    flat = torch.randn(1 + 12 * 96, generator=g, dtype=torch.float32).to(torch.bfloat16)
    nn64.near(tpo.layer_norm(flat.to(dev)[1:].view(12, 96)),
              nn64.layer_norm(flat[1:].view(12, 96), None, None, 1e-5))
    side = torch.cuda.Stream()
    X = big.to(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = tpo.layer_norm(X)
    torch.cuda.current_stream().wait_stream(side)
    nn64.near(y, nn64.layer_norm(big, None, None, 1e-5))
    e = torch.empty(0, 48, device=dev, requires_grad=True)
    W = torch.ones(48, device=dev, requires_grad=True)
    y = tpo.layer_norm(e, W)
    ge, gw = torch.autograd.grad(y, (e, W), torch.empty(0, 48, device=dev))
    assert y.shape == ge.shape == (0, 48) and (gw == 0).all()


def test_more_than_32_bits_of_values(tpo, dev):
    rows, width = (1 << 31) // 4096 + 5, 4096
    x = torch.empty(rows, width, dtype=torch.bfloat16, device=dev)
    g = torch.Generator().manual_seed(3)
    tail = torch.randn(7, width, generator=g).to(torch.bfloat16)
    x.zero_()
    x[-7:] = tail
    y = tpo.layer_norm(x)
    nn64.near(y[-7:], nn64.layer_norm(tail, None, None, 1e-5))
    assert (y[:3] == 0).all()


def test_gradient_sums_repeat(tpo, dev):
    x, w, b, gy = _inputs((9000, 130), torch.float32, "same", 8)
    X, W, B = _on(dev, x, w, b)
    first = torch.autograd.grad(tpo.layer_norm(X, W, B), (X, W, B), gy.to(dev))
    for _ in range(3):
        again = torch.autograd.grad(tpo.layer_norm(X, W, B), (X, W, B), gy.to(dev))
        assert all(torch.equal(a, c) for a, c in zip(first, again))


def test_graph_replays(tpo, dev):
    x, w, b, gy = _inputs((300, 192), torch.bfloat16, "same", 6)
    X, W, B = _on(dev, x, w, b)
    G = gy.to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(tpo.layer_norm(X, W, B), (X, W, B), G)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tpo.layer_norm(X, W, B)
        gs = torch.autograd.grad(y, (X, W, B), G)
    for seed in range(3):
        with torch.no_grad():
            X.copy_(_inputs((300, 192), torch.bfloat16, "same", 60 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        e = tpo.layer_norm(X, W, B)
        es = torch.autograd.grad(e, (X, W, B), G)
        assert torch.equal(y, e) and all(torch.equal(a, c) for a, c in zip(gs, es))


def test_module_and_refusals(tpo, dev):
    m = tpo.LayerNorm(96, device=dev)
    x = torch.randn(5, 96, device=dev)
    nn64.near(m(x), nn64.layer_norm(x.cpu(), m.weight.cpu().detach(), m.bias.cpu().detach(), 1e-5))
    m(x).sum().backward()
    assert m.weight.grad.shape == m.bias.grad.shape == (96,)
    w = torch.ones(96, device=dev)
    for bad, words in [((x.double(),), "not implemented for"), ((x, w[:95]), "must have shape"),
                       ((x, w.half()), "x's type or float32"), ((x, w.cpu()), "same device"),
                       ((x.half(), w, w.half()), "one type"),
                       ((torch.empty(3, 0, device=dev),), "empty"), ((x, None, None, -1.0), "eps")]:
        with pytest.raises(RuntimeError, match=words):
            tpo.layer_norm(*bad)
