"""rotary_positions against its definition in float64: layouts, parts, places, gradients."""
import pytest
import torch

from tests import cache64, nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _inputs(T, H, D, pairs, axes, dtype, seed, places=20000):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, D, generator=g).to(dtype)
    if axes == 0:  # places
        at = torch.randint(-places, places, (T,), generator=g)
    else:
        at = 2 * torch.rand(T, axes, generator=g) - 1
    f = 1e4 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))
    return x, at, f if axes == 0 else 40 * f, torch.randn(T, H, D, generator=g).to(dtype)


def _check(tpo, dev, T, H, D, pairs, dtype, interleaved=False, axes=0, amplitude=1.0, seed=0):
    x, at, f, gy = _inputs(T, H, D, pairs, axes, dtype, seed)
    X = x.to(dev).requires_grad_(True)
    y = tpo.rotary_positions(X, at.to(dev), f.to(dev), interleaved, amplitude)
    assert y.dtype == dtype and y.is_contiguous()
    nn64.near(y, cache64.turn(x, at, f, interleaved, amplitude))
    assert torch.equal(y.detach().cpu()[..., 2 * pairs:], x[..., 2 * pairs:])
    gx, = torch.autograd.grad(y, X, gy.to(dev))
    nn64.near(gx, cache64.turn(gy, at, f, interleaved, amplitude, back=True))
    return y


@pytest.mark.parametrize("D", [2, 3, 8, 16, 20, 40, 63, 64, 80, 96, 128, 129, 256, 512])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(tpo, dev, D, interleaved, dtype):
    for pairs in sorted({0, 1, D // 4, D // 2}):
        _check(tpo, dev, 37, 3, D, pairs, dtype, interleaved, seed=D + pairs)


@pytest.mark.parametrize("T,H", [(1, 1), (1, 40), (2, 300), (255, 7), (5000, 2), (33000, 1)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_and_heads(tpo, dev, T, H, dtype):
    _check(tpo, dev, T, H, 24, 12, dtype, seed=T + H)


@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(tpo, dev, axes, interleaved):
    _check(tpo, dev, 100, 4, 56, 24, torch.float32, interleaved, axes=axes, amplitude=1.3)


def test_places_far_away(tpo, dev):
    """Angles are those of 64 bits: places of millions turn as exactly as the first."""
    x, _, f, _ = _inputs(64, 2, 32, 16, 0, torch.float32, 5)
    for top in (10, 2 ** 20, 2 ** 31, 2 ** 40):
        at = torch.arange(64) + top
        y = tpo.rotary_positions(x.to(dev), at.to(dev), f.to(dev))
        # an angle of 64 bits is off by 2^-53 of itself in either place
        nn64.near(y, cache64.turn(x, at, f), floats=nn64.FLOAT + top * 2.0 ** -51)
    at = torch.tensor([float("nan"), float("inf"), 2.0 ** 60, 1.0])
    y = tpo.rotary_positions(x[:4].to(dev), at.to(dev), f.to(dev)).cpu()
    assert y[:2].isnan().all() and y[2, :, 0].isnan().all() and y[3].isfinite().all()


def test_values_that_are_not_finite(tpo, dev):
    """A NaN or an infinity reaches its pair and nothing else."""
    x, at, f, _ = _inputs(9, 2, 40, 16, 0, torch.float16, 6)
    clean = tpo.rotary_positions(x.to(dev), at.to(dev), f.to(dev)).cpu()
    x[3, 1, 5], x[4, 0, 35] = float("nan"), float("inf")
    y = tpo.rotary_positions(x.to(dev), at.to(dev), f.to(dev)).cpu()
    bad = torch.zeros(y.shape, dtype=torch.bool)
    bad[3, 1, 5] = bad[3, 1, 21] = bad[4, 0, 35] = True
    assert torch.equal(y[~bad], clean[~bad]) and not y[bad].isfinite().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(tpo, dev, dtype):
    """Slices of a projection, heads first, rows at odd places, every other value, broadcast."""
    g = torch.Generator().manual_seed(7)
    f = torch.rand(10, generator=g, dtype=torch.float64)
    at = torch.arange(30)
    y = torch.randn(30, 9, 41, generator=g).to(dtype)
    views = [lambda t: t[:, 2:5, :24], lambda t: t[:9].transpose(0, 1)[:, :, 1:],
             lambda t: t[:, :, 1:40:2][..., :20], lambda t: t[:, :1].expand(30, 5, 41),
             lambda t: t[:1].expand(30, 9, 41)]
    for view in views:
        x, X = view(y), view(y.to(dev))
        n = len(x)
        nn64.near(tpo.rotary_positions(X, at[:n].to(dev), f.to(dev)),
                  cache64.turn(x, at[:n], f))
    x = y[:, :, 1:40:2][..., :20]
    # gradients that are broadcast or turned round
    X = x.to(dev).requires_grad_(True)
    out = tpo.rotary_positions(X, at.to(dev), f.to(dev))
    gx, = torch.autograd.grad(out.sum(), X)
    nn64.near(gx, cache64.turn(torch.ones(30, 9, 20), at, f, back=True))


def test_nothing_to_turn(tpo, dev):
    f = torch.ones(4, dtype=torch.float64, device=dev)
    for shape in ((0, 3, 16), (5, 0, 16)):
        x = torch.ones(*shape, device=dev, requires_grad=True)
        y = tpo.rotary_positions(x, torch.zeros(shape[0], dtype=torch.int64, device=dev), f)
        assert y.shape == x.shape
        y.sum().backward()
        assert x.grad.shape == x.shape


def test_gradient_against_differences(tpo, dev):
    x, at, f, gy = _inputs(5, 2, 12, 4, 0, torch.float32, 8)
    X = x.to(dev).requires_grad_(True)
    gx, = torch.autograd.grad(tpo.rotary_positions(X, at.to(dev), f.to(dev), True), X, gy.to(dev))
    d = torch.randn(x.shape, generator=torch.Generator().manual_seed(9)).to(dev)
    with torch.no_grad():
        hi, lo = (tpo.rotary_positions(X + s * d, at.to(dev), f.to(dev), True).double()
                  for s in (0.5, -0.5))
    # a linear map: the difference is exact but for float's rounding of values of about 1
    assert abs(((hi - lo) * gy.to(dev)).sum() - (gx.double() * d).sum()) < 1e-4


def test_module(tpo, dev):
    m = tpo.RotaryPositions(32, base=500.0, stretch=4.0, trained=256, interleaved=True,
                            amplitude=1.1).to(dev).to(torch.bfloat16)
    assert m.frequencies.dtype == torch.float64 and m.frequencies.device.type == "cuda"
    x, at, _, _ = _inputs(50, 2, 40, 16, 0, torch.bfloat16, 3)
    f = tpo.rotary_frequencies(16, 500.0, 4.0, 256)
    nn64.near(m(x.to(dev), at.to(dev)), cache64.turn(x, at, f, True, 1.1))


def test_captured(tpo, dev):
    x, at, f, _ = _inputs(40, 3, 64, 32, 0, torch.bfloat16, 4)
    X, A, F = x.to(dev), at.to(dev), f.to(dev)
    tpo.rotary_positions(X, A, F)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = tpo.rotary_positions(X, A, F)
    for step in range(3):
        A.add_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, tpo.rotary_positions(X, A, F))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_queries_of_append_are_the_same(tpo, dev, dtype, interleaved):
    """Bit for bit, in each of the kernels that turn them, however often a rounding is close."""
    g = torch.Generator().manual_seed(5)
    for B, new, H in ((200, 3, 8), (2, 700, 8), (1, 3000, 96)):  # (the last past the caches)
        T = B * new
        q, k = (torch.randn(T, h, 128, generator=g).to(dev, dtype) for h in (H, 1))
        f = tpo.rotary_frequencies(64, device=dev)
        cache = tpo.PagedCache.empty(B, new, 1, 128, device=dev)
        cache.lengths += new
        o = torch.arange(B + 1, device=dev) * new
        got = tpo.cache_append(cache, k, k, o, q, f, interleaved=interleaved)
        at = torch.arange(T, device=dev) % new
        assert torch.equal(got, tpo.rotary_positions(q, at, f, interleaved))
