"""cache_append against its definition in float64: every code, scale and byte that stays."""
import pytest
import torch

from tests import cache64, nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _offsets(counts, before=0):
    o = [before]
    for n in counts:
        o.append(o[-1] + n)
    return o


def _rows(T, Hq, Hk, D, dtype, seed, level=1.0):
    g = torch.Generator().manual_seed(seed)
    y = torch.randn(T, Hq + 2 * Hk, D, generator=g)
    y = y * torch.exp(level * torch.randn(T, 1, 1, generator=g))
    return y.to(dtype).split([Hq, Hk, Hk], 1)


def _same(cache, want):
    """The GPU's cache holds exactly what the definition gives."""
    got = cache64.Cache(cache)
    assert torch.equal(got.ks, want.ks) and torch.equal(got.vs, want.vs)
    assert torch.equal(got.k.nan_to_num(999), want.k.nan_to_num(999))
    assert torch.equal(got.v.nan_to_num(999), want.v.nan_to_num(999))


def _check(tpo, dev, new, held, Hq, Hk, D, dtype, page=64, pairs=None, interleaved=False, seed=0,
           lengths_new=None, before=0, after=0, at=None, amplitude=1.0, level=1.0, cache=None):
    """Appends `new` tokens a sequence to `held`; returns the cache, the queries and inputs."""
    used = new if lengths_new is None else [min(a, max(0, b)) for a, b in zip(new, lengths_new)]
    if cache is None:
        cache = cache64.paged(tpo, dev, [a + b for a, b in zip(used, held)], Hk, D, page, seed)
    want = cache64.Cache(cache)
    o = _offsets(new, before)
    q, k, v = _rows(o[-1] + after, Hq, Hk, D, dtype, seed, level)
    pairs = D // 2 if pairs is None else pairs
    f = 1e4 ** (-torch.arange(pairs, dtype=torch.float64) / max(1, pairs))
    ln = None if lengths_new is None else torch.tensor(lengths_new, device=dev)
    wq = want.append(k, v, o, lengths_new, q, f, at, interleaved, amplitude)
    gq = tpo.cache_append(cache, k.to(dev), v.to(dev), torch.tensor(o, device=dev), q.to(dev),
                          f.to(dev), None if at is None else at.to(dev), interleaved, amplitude, ln)
    assert gq.dtype == dtype
    nn64.near(gq, wq)
    assert (gq.cpu()[(wq == 0).all(-1)] == 0).all()
    _same(cache, want)
    return cache, (q, k, v, o, f)


# (new tokens, tokens held): pages and blocks that begin, end and go on inside
CASES = [([1], [0]), ([1], [63]), ([1, 1, 1], [64, 31, 130]), ([0, 2, 0, 1], [5, 62, 0, 0]),
         ([100], [0]), ([64, 128, 1], [0, 64, 0]), ([33, 70, 0, 5], [31, 60, 9, 127]),
         ([300], [17]), ([3] * 70, list(range(70))), ([0, 0], [3, 0])]


@pytest.mark.parametrize("new,held", CASES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_places(tpo, dev, new, held, dtype):
    _check(tpo, dev, new, held, 4, 2, 64, dtype, seed=len(new))


@pytest.mark.parametrize("D", [1, 2, 8, 16, 17, 24, 40, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(tpo, dev, D, interleaved, dtype):
    for pairs in sorted({0, D // 4, D // 2}):
        for new, held in (([2, 3], [40, 0]), ([90], [20])):
            _check(tpo, dev, new, held, 3, 3, D, dtype, pairs=pairs, interleaved=interleaved,
                   seed=D + pairs)


@pytest.mark.parametrize("page", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("D", [32, 128])
def test_pages(tpo, dev, page, D):
    for new, held in (([1, 4], [page - 1, 7]), ([2 * page + 5, 3, page], [page // 2, 0, 0])):
        _check(tpo, dev, new, held, 2, 1, D, torch.bfloat16, page=page, seed=page)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (5, 5), (6, 3), (16, 2), (17, 17), (64, 8)])
def test_heads(tpo, dev, Hq, Hk):
    for new in ([1, 2], [70, 40]):
        _check(tpo, dev, new, [10, 60], Hq, Hk, 32, torch.float16, seed=Hq)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_grow(tpo, dev, dtype):
    """Token after token, each larger than all before it, then smaller ones."""
    cache = cache64.paged(tpo, dev, [0, 0], 2, 40, 32, seed=3, extra=2)
    cache.table.copy_(torch.tensor([[0, 1, -1], [-1, -1, -1]]))
    g = torch.Generator().manual_seed(4)
    for i in range(40):
        cache.lengths.copy_(torch.tensor([i + 1, 0]))
        want = cache64.Cache(cache)
        k, v = (torch.randn(1, 2, 40, generator=g) * 2.0 ** (8 - abs(i - 20) / 2) for _ in range(2))
        k, v = k.to(dtype), v.to(dtype)
        want.append(k, v, [0, 1, 1])
        assert tpo.cache_append(cache, k.to(dev), v.to(dev),
                                torch.tensor([0, 1, 1], device=dev)) is None
        _same(cache, want)


def test_every_code(tpo, dev):
    """Values on, next to and half-way between codes, normal and subnormal ones, at several
    scales."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    x = torch.cat([x, -x, torch.full((1024 - 2 * len(x),), 448.0, dtype=torch.float64)])
    for e in (-30, -3, 0, 11, 38):
        k = (x.view(8, 1, 128) * 2.0 ** e).float()
        cache = cache64.paged(tpo, dev, [8], 1, 128, 32)
        want = cache64.Cache(cache)
        want.append(k, -k, [0, 8])
        assert want.ks[int(cache.table[0, 0]), 0] == 2.0 ** e
        tpo.cache_append(cache, k.to(dev), -k.to(dev), torch.tensor([0, 8], device=dev))
        _same(cache, want)


def test_extreme_values(tpo, dev):
    """Zeros, the least and the largest, what is not finite: the page's other values keep their
    scale."""
    k = torch.zeros(12, 1, 32)
    k[1, 0, 3], k[2] = 1.0, 1e-30
    v = torch.ones(12, 1, 32)
    v[4, 0, 0], v[5, 0, 1], v[6, 0, 2] = float("inf"), float("-inf"), float("nan")
    v[7, 0, 3], v[8, 0, 4] = 3e38, -3e38
    for n in (1, 12):
        for start in (0, 3):
            cache = cache64.paged(tpo, dev, [start + n], 1, 32, 32)
            want = cache64.Cache(cache)
            want.append(k[:n], v[:n], [0, n])
            tpo.cache_append(cache, k[:n].to(dev), v[:n].to(dev), torch.tensor([0, n], device=dev))
            _same(cache, want)
    # what is not finite in a key reaches its pair
    cache = cache64.paged(tpo, dev, [12], 1, 32, 32)
    want = cache64.Cache(cache)
    f = torch.ones(8, dtype=torch.float64)
    want.append(v, k, [0, 12], f=f)
    tpo.cache_append(cache, v.to(dev), k.to(dev), torch.tensor([0, 12], device=dev), None, f.to(dev))
    _same(cache, want)


@pytest.mark.parametrize("many", [False, True])
def test_rows_not_in_use(tpo, dev, many):
    """A padded batch, rows before the first sequence and behind the last, offsets outside."""
    new, lengths = ([3, 2, 4], [1, 0, 9]) if not many else ([90, 40, 70], [50, -3, 70])
    _check(tpo, dev, new, [20, 33, 0], 2, 2, 48, torch.float32, lengths_new=lengths, before=2,
           after=3, seed=5)
    g = torch.Generator().manual_seed(6)
    T = 6 if not many else 60
    k, v = (torch.randn(T, 1, 16, generator=g) for _ in range(2))
    for o in ([-5, 3, 2 * T], [4, 2, T], [T + 1, T + 2, T + 9], [0, T, T - 1]):
        cache = cache64.paged(tpo, dev, [70, 80], 1, 16, 32)
        want = cache64.Cache(cache)
        want.append(k, v, o)
        tpo.cache_append(cache, k.to(dev), v.to(dev), torch.tensor(o, device=dev))
        _same(cache, want)


@pytest.mark.parametrize("many", [False, True])
def test_pages_that_are_not_there(tpo, dev, many):
    """Nothing is written for entries outside of the pool, nor for tokens before the first place;
    lengths stop at the table's room."""
    n = 40 if many else 2
    cache = cache64.paged(tpo, dev, [100, 100, 100, 100, 100], 2, 32, 32)
    P = cache.keys.shape[0]
    cache.table[0, 2:] = -1
    cache.table[1, 3] = P
    cache.table[2, 1:] = torch.tensor([2 ** 31 - 1, -2 ** 31, P + 7], dtype=torch.int32)
    cache.lengths.copy_(torch.tensor([100, 97, 64, n - 1, 10 ** 12]))
    _check(tpo, dev, [n] * 5, [0] * 5, 2, 2, 32, torch.float32, cache=cache, seed=8)
    cache.lengths.copy_(torch.tensor([0, -4, 1, 33, 128]))
    _check(tpo, dev, [n] * 5, [0] * 5, 2, 2, 32, torch.float32, cache=cache, seed=9)
    empty = tpo.PagedCache.empty(2, 64, 2, 32, page=32, pages=0, device=dev)
    empty.lengths.fill_(50)
    o = torch.tensor([0, 1, 3], device=dev)
    tpo.cache_append(empty, torch.ones(3, 2, 32, device=dev), torch.ones(3, 2, 32, device=dev), o)
    none = tpo.PagedCache.empty(0, 64, 2, 32, device=dev)
    q = tpo.cache_append(none, torch.ones(3, 2, 32, device=dev), torch.ones(3, 2, 32, device=dev),
                         o[:1], q=torch.ones(3, 4, 32, device=dev),
                         frequencies=torch.ones(4, dtype=torch.float64, device=dev))
    assert (q == 0).all()


def test_given_positions(tpo, dev):
    g = torch.Generator().manual_seed(10)
    for many in (False, True):
        new = [50, 20] if many else [2, 3]
        at = torch.randint(0, 10 ** 6, (sum(new),), generator=g)
        _check(tpo, dev, new, [5, 40], 4, 2, 32, torch.bfloat16, at=at, amplitude=0.9)
        at = torch.rand(sum(new), 2, generator=g)
        _check(tpo, dev, new, [5, 40], 4, 2, 40, torch.bfloat16, pairs=12, at=at, interleaved=True)


def test_strides(tpo, dev):
    """k, v and q as slices of one projection, at odd places, and with values apart."""
    g = torch.Generator().manual_seed(11)
    y = torch.randn(50, 7, 81, generator=g).to(torch.float16)
    f = torch.rand(13, generator=g, dtype=torch.float64)
    for new in ([1, 2, 1], [30, 20]):
        o, T = _offsets(new), sum(new)
        for view in (lambda t: (t[:T, 0:3, 1:41], t[:T, 3:5, 1:41], t[:T, 5:7, 3:43]),
                     lambda t: (t[:T, 0:3, ::2], t[:T, 3:5, ::2], t[:T, 5:7, ::2]),
                     lambda t: (t[:T, :4, :40], t[:T, :1, :40].expand(T, 2, 40), t[:T, 1:3, :40])):
            cache = cache64.paged(tpo, dev, [9 + n for n in new], 2, view(y)[1].shape[2])
            want = cache64.Cache(cache)
            q, k, v = view(y)
            wq = want.append(k, v, o, None, q, f)
            Q, K, V = view(y.to(dev))
            nn64.near(tpo.cache_append(cache, K, V, torch.tensor(o, device=dev), Q, f.to(dev)), wq)
            _same(cache, want)


def test_again_and_in_pieces(tpo, dev):
    """The same tokens twice leave what the first time left; a prompt in pieces that end with
    pages is the prompt at once."""
    cache, (q, k, v, o, f) = _check(tpo, dev, [70, 3], [40, 31], 2, 2, 64, torch.bfloat16, seed=12)
    kept = [t.clone() for t in (cache.keys.view(torch.uint8), cache.values.view(torch.uint8),
                                cache.key_scales, cache.value_scales)]
    tpo.cache_append(cache, k.to(dev), v.to(dev), torch.tensor(o, device=dev), None, f.to(dev))
    for a, b in zip(kept, (cache.keys.view(torch.uint8), cache.values.view(torch.uint8),
                           cache.key_scales, cache.value_scales)):
        assert torch.equal(a, b)
    one, two = (cache64.paged(tpo, dev, [200], 2, 64, 64, seed=13) for _ in range(2))
    _, K, V = (t.to(dev) for t in _rows(200, 1, 2, 64, torch.float16, 13))
    tpo.cache_append(one, K, V, torch.tensor([0, 200], device=dev), None, f.to(dev))
    for a, b in ((0, 64), (64, 192), (192, 200)):
        two.lengths.fill_(b)
        tpo.cache_append(two, K[a:b], V[a:b], torch.tensor([0, b - a], device=dev), None, f.to(dev))
    assert torch.equal(one.keys.view(torch.uint8), two.keys.view(torch.uint8))
    assert torch.equal(one.values.view(torch.uint8), two.values.view(torch.uint8))


def test_few_rule_with_many_tokens(tpo, dev):
    """Many sequences of one token and one of many: a page's tokens in several rounds."""
    new = [1] * 30 + [150] + [0] * 10
    _check(tpo, dev, new, [3 * b for b in range(41)], 4, 4, 128, torch.bfloat16, seed=14)
    _check(tpo, dev, new, [3 * b for b in range(41)], 5, 5, 40, torch.float32, seed=15, page=128)


def test_captured_with_lengths_that_grow(tpo, dev):
    cache = cache64.paged(tpo, dev, [3, 40], 2, 32, 32, seed=16, extra=2, spare=6)
    cache.table.copy_(torch.arange(cache.table.numel()).view_as(cache.table) % cache.keys.shape[0])
    g = torch.Generator().manual_seed(17)
    f, o = torch.rand(16, generator=g, dtype=torch.float64), torch.tensor([0, 1, 2], device=dev)
    k, v, q = (torch.randn(2, 2, 32, generator=g).to(dev) for _ in range(3))
    cache.lengths.add_(1)
    tpo.cache_append(cache, k, v, o, q, f.to(dev))
    F = f.to(dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.lengths.add_(1)
        out = tpo.cache_append(cache, k, v, o, q, F)
    for _ in range(5):
        want = cache64.Cache(cache)
        want.lengths += 1
        for t in (k, v, q):
            t.copy_(torch.randn(2, 2, 32, generator=g))
        wq = want.append(k.cpu(), v.cpu(), [0, 1, 2], None, q.cpu(), f)
        graph.replay()
        torch.cuda.synchronize()
        nn64.near(out, wq)
        _same(cache, want)


def test_versions_and_derivatives(tpo, dev):
    cache = cache64.paged(tpo, dev, [2], 1, 16)
    k, o = torch.ones(1, 1, 16, device=dev), torch.tensor([0, 1], device=dev)
    was = cache.keys._version
    tpo.cache_append(cache, k, k, o)
    assert cache.keys._version == was + 1
    with torch.inference_mode():
        tpo.cache_append(cache, k, k, o)
    with pytest.raises(RuntimeError, match="has no derivative"):
        tpo.cache_append(cache, k.requires_grad_(True), k, o)
    with torch.no_grad():
        tpo.cache_append(cache, k, k, o)


def test_scales_from_elsewhere(tpo, dev):
    """Older codes of a page whose scale is above the largest: what does not fit is the largest
    value, as of new tokens; in both kernels."""
    for new in (1, 30):
        cache = tpo.PagedCache.empty(1, 64, 1, 16, device=dev)
        cache.lengths.fill_(20)
        k = torch.ones(20, 1, 16, device=dev)
        k[3], k[4], k[5, 0, 2] = -2.0, 0.0, float("nan")
        tpo.cache_append(cache, k, k, torch.tensor([0, 20], device=dev))
        old = cache.rows()[0][0, 0, :20].clone() / cache.key_scales[0, 0]
        cache.key_scales.fill_(2.0 ** 44)
        cache.value_scales.fill_(2.0 ** 44)
        cache.lengths += new
        z = torch.zeros(new, 1, 16, device=dev)
        tpo.cache_append(cache, z, z, torch.tensor([0, new], device=dev))
        assert (cache.key_scales == 2.0 ** 40).all() and (cache.value_scales == 2.0 ** 40).all()
        want = (old * 16).clamp(-448, 448) * 2.0 ** 40
        for rows in cache.rows():
            assert torch.equal(rows[0, 0, :20].nan_to_num(1.0), want.nan_to_num(1.0))
            assert rows[0, 0, 5, 2].isnan() and (rows[0, 0, 20:20 + new] == 0).all()
