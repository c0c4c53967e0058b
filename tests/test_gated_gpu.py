"""gated_projection against its definition in float64: sizes, activations, gradients, refusals."""
import pytest
import torch

from tests import nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = ["silu", "gelu", "relu", "sigmoid"]


def _inputs(M, K, F, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * size
    wg, wu = (torch.randn(F, K, generator=g) / K ** 0.5 for _ in range(2))
    return tuple(t.to(dtype) for t in (x, wg, wu, torch.randn(M, F, generator=g)))


def _check(tpo, dev, M, K, F, dtype, name, seed=0):
    x, wg, wu, gh = _inputs(M, K, F, dtype, seed)
    want, gwant = nn64.grads(lambda a, b, c: nn64.gated(a, b, c, name), (x, wg, wu), gh)
    X, G, U = (t.to(dev).requires_grad_(True) for t in (x, wg, wu))
    h = tpo.gated_projection(X, G, U, name)
    assert h.dtype == dtype
    # float sums of K terms: the error grows with the root of their number
    nn64.near(h, want, floats=2e-6 + 2e-7 * K ** 0.5)
    got = torch.autograd.grad(h, (X, G, U), gh.to(dev))
    for a, e in zip(got, gwant):
        nn64.near(a, e, roundings=2, floats=2e-6 + 2e-7 * max(M, K, F) ** 0.5)
    return (h, *got)


# one row, few rows (a step of generation), tiles' edges, odd widths, widths
# that end inside a 16-byte load, one feature
@pytest.mark.parametrize("M,K,F", [
    (1, 1, 1), (1, 64, 128), (2, 8, 16), (3, 7, 5), (16, 512, 96), (17, 40, 33), (31, 100, 129),
    (33, 136, 72), (64, 64, 64), (65, 72, 130), (127, 130, 127), (128, 128, 256), (129, 257, 255),
    (200, 385, 300), (256, 320, 512), (257, 96, 513), (700, 33, 1000), (40, 1031, 40), (5, 2048, 700),
    (1000, 8, 24), (32, 1536, 264),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_and_gradients(tpo, dev, M, K, F, dtype):
    _check(tpo, dev, M, K, F, dtype, "silu", seed=M + K + F)


# enough of two of the axes for the largest tiles in one product each (the
# projections; x's gradient; the weights'), and for the middle ones in all, with
# sums that are shared and ends inside tiles
@pytest.mark.parametrize("M,K,F", [
    (5000, 99, 2203), (8180, 2041, 66), (131, 2041, 4090), (1999, 2050, 1027), (4097, 100, 2050),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_tiles(tpo, dev, M, K, F, dtype):
    _check(tpo, dev, M, K, F, dtype, "gelu", seed=M + K + F)


# more workgroups of few tokens than CUs, but few tiles: the smallest ones
@pytest.mark.parametrize("M,K,F", [(600, 72, 1100), (900, 131, 701), (1025, 520, 640)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_small_tiles(tpo, dev, M, K, F, dtype):
    _check(tpo, dev, M, K, F, dtype, "relu", seed=M + K + F)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_activations(tpo, dev, name, dtype):
    _check(tpo, dev, 70, 96, 200, dtype, name, seed=4)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_far_activations(tpo, dev, name, dtype):
    """Gates of up to a hundred in size: no overflow inside, saturated values exact."""
    x, wg, wu, gh = _inputs(30, 64, 48, dtype, 11, size=30.0)
    want, gwant = nn64.grads(lambda a, b, c: nn64.gated(a, b, c, name), (x, wg, wu), gh)
    X, G, U = (t.to(dev).requires_grad_(True) for t in (x, wg, wu))
    h = tpo.gated_projection(X, G, U, name)
    # an activation's relative slope grows with its argument (30 to 100 here)
    nn64.near(h, want, floats=1e-4)
    for a, e in zip(torch.autograd.grad(h, (X, G, U), gh.to(dev)), gwant):
        nn64.near(a, e, roundings=2, floats=1e-4)


def test_each_gradient_alone(tpo, dev):
    x, wg, wu, gh = _inputs(50, 64, 80, torch.bfloat16, 5)
    ins = [t.to(dev).requires_grad_(True) for t in (x, wg, wu)]
    full = torch.autograd.grad(tpo.gated_projection(*ins), ins, gh.to(dev))
    for at in range(3):
        part = [t.detach().requires_grad_(i == at) for i, t in enumerate(ins)]
        g, = torch.autograd.grad(tpo.gated_projection(*part), part[at], gh.to(dev))
        assert torch.equal(g, full[at])


def test_one_weight_for_both(tpo, dev):
    x, w, _, gh = _inputs(40, 64, 72, torch.float32, 6)
    want, gwant = nn64.grads(lambda a, b: nn64.gated(a, b, b, "silu"), (x, w), gh)
    X, W = (t.to(dev).requires_grad_(True) for t in (x, w))
    h = tpo.gated_projection(X, W, W)
    nn64.near(h, want, floats=4e-6)
    for a, e in zip(torch.autograd.grad(h, (X, W), gh.to(dev)), gwant):
        nn64.near(a, e, floats=4e-6)


def test_gradient_against_differences(tpo, dev):
    x, wg, wu, gh = _inputs(9, 24, 17, torch.float32, 7)
    ins = [t.to(dev).requires_grad_(True) for t in (x, wg, wu)]
    for name in ("silu", "gelu", "sigmoid"):
        got = torch.autograd.grad(tpo.gated_projection(*ins, name), ins, gh.to(dev))
        g = torch.Generator().manual_seed(1)
        for at in range(3):
            d = [torch.randn(t.shape, generator=g, dtype=torch.float64) * (i == at)
                 for i, t in enumerate((x, wg, wu))]
            want = nn64.slope(lambda *a: (nn64.gated(*a, name) * gh.double()).sum(),
                              [t.double() for t in (x, wg, wu)], d, 1e-5)
            have = (got[at].cpu().double() * d[at]).sum()
            assert abs(have - want) <= 1e-5 * got[at].norm().item() * d[at].norm().item()


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_shapes(tpo, dev, dtype):
    x, wg, wu, _ = _inputs(60, 72, 40, dtype, 8)
    want = nn64.gated(x, wg, wu, "silu")
    f = dict(roundings=1, floats=4e-6)
    X, G, U = (t.to(dev) for t in (x, wg, wu))
    nn64.near(tpo.gated_projection(X.view(3, 4, 5, 72), G, U).view(60, 40), want, **f)
    nn64.near(tpo.gated_projection(X[7], G, U), want[7], **f)
    nn64.near(tpo.gated_projection(X.t().contiguous().t(), G.t().contiguous().t(), U), want, **f)
    wide = torch.zeros(60, 75, dtype=dtype, device=dev)
    wide[:, 1:73] = X
    nn64.near(tpo.gated_projection(wide[:, 1:73], G, U), want, **f)
    flat = torch.cat([torch.zeros(1, dtype=dtype, device=dev), G.flatten()])
    nn64.near(tpo.gated_projection(X, flat[1:].view(40, 72), U), want, **f)  # off the 16-byte grid


def test_more_than_32_bits_of_values(tpo, dev):
    """Outputs beyond 2^31 values; one weight's rows and the last tokens are checked."""
    M, F = (1 << 31) // 8192 + 100, 8192
    x, wg, wu, _ = _inputs(200, 64, F, torch.bfloat16, 13)
    X = torch.zeros(M, 64, dtype=torch.bfloat16, device=dev)
    X[-200:] = x.to(dev)
    h = tpo.gated_projection(X, wg.to(dev), wu.to(dev))
    nn64.near(h[-200:], nn64.gated(x, wg, wu, "silu"), floats=4e-6)
    assert (h[:3] == 0).all()


def test_nonfinite_rows_stay_apart(tpo, dev):
    x, wg, wu, _ = _inputs(40, 64, 48, torch.bfloat16, 9)
    X, G, U = (t.to(dev) for t in (x, wg, wu))
    clean = tpo.gated_projection(X, G, U)
    X[3] = float("nan")
    X[11] = float("inf")
    got = tpo.gated_projection(X, G, U)
    keep = [i for i in range(40) if i not in (3, 11)]
    assert torch.equal(got[keep], clean[keep]) and got[3].isnan().all()


def test_empty_calls(tpo, dev):
    for M, F in ((0, 5), (4, 0), (0, 0)):
        x = torch.ones(M, 8, device=dev, requires_grad=True)
        g, u = (torch.ones(F, 8, device=dev, requires_grad=True) for _ in range(2))
        h = tpo.gated_projection(x, g, u)
        gs = torch.autograd.grad(h, (x, g, u), torch.ones_like(h))
        assert h.shape == (M, F) and all((t == 0).all() for t in gs)
        assert [t.shape for t in gs] == [x.shape, g.shape, u.shape]


def test_repeats_streams_and_graph(tpo, dev):
    x, wg, wu, gh = _inputs(150, 136, 200, torch.bfloat16, 10)
    ins = [t.to(dev).requires_grad_(True) for t in (x, wg, wu)]
    GH = gh.to(dev)

    def both():
        # detached: a graph that is kept holds its leaves to the stream they were used on
        h = tpo.gated_projection(*ins)
        return (h.detach(), *torch.autograd.grad(h, ins, GH))

    e = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(e, r))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = both()
    for seed in range(3):
        with torch.no_grad():
            ins[0].copy_(_inputs(150, 136, 200, torch.bfloat16, 20 + seed)[0])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(both(), r))


def test_module_and_refusals(tpo, dev):
    m = tpo.GatedFeedForward(64, 96, "gelu", device=dev)
    x = torch.randn(5, 7, 64, device=dev)
    h = nn64.gated(x.cpu(), m.gate.weight.detach().cpu(), m.up.weight.detach().cpu(), "gelu")
    nn64.near(m(x), h @ m.down.weight.detach().cpu().double().t(), floats=1e-5)
    m(x).sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    x, w = torch.ones(4, 16, device=dev), torch.ones(8, 16, device=dev)
    for bad, words in [((x, w, w[:7]), "same shape"), ((x[:, :15], w, w), "features"),
                       ((x.half(), w, w), "one type"), ((x, w[0], w[0]), "expects x"),
                       ((x.double(), w.double(), w.double()), "not implemented for"),
                       ((x, w.cpu(), w.cpu()), "same device")]:
        with pytest.raises(RuntimeError, match=words):
            tpo.gated_projection(*bad)
    with pytest.raises(RuntimeError, match="unknown activation"):
        torch.ops.torch_point_ops_gated.gated_projection(x, w, w, 9)
    with pytest.raises(ValueError, match="activation must be"):
        tpo.gated_projection(x, w, w, "tanh")
