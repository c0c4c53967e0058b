"""cache_append and cached_attention where numbers end: keys next to nothing, the largest."""
import math

import pytest
import torch

from tests import cache64, nn64

pytestmark = pytest.mark.gpu


def _same(cache, want):
    """The GPU's cache holds exactly what the definition gives."""
    got = cache64.Cache(cache)
    assert torch.equal(got.ks, want.ks) and torch.equal(got.vs, want.vs)
    assert torch.equal(got.k.nan_to_num(999), want.k.nan_to_num(999))
    assert torch.equal(got.v.nan_to_num(999), want.v.nan_to_num(999))


def _append(tpo, dev, k, f, at, interleaved, amplitude=1.0):
    """k (T, H, D) as keys and values of one sequence, against the definition; few tokens and many
    take kernels of their own."""
    T, H, D = k.shape
    cache = cache64.paged(tpo, dev, [T + 3], H, D, 32, seed=T)
    want = cache64.Cache(cache)
    want.append(k, k, [0, T], f=f, at=at, interleaved=interleaved, amplitude=amplitude)
    tpo.cache_append(cache, k.to(dev), k.to(dev), torch.tensor([0, T], device=dev), None, f.to(dev),
                     at.to(dev), interleaved, amplitude)
    _same(cache, want)
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [4, 40])
def test_turned_keys_next_to_nothing(tpo, dev, dtype, interleaved, T):
    """Finite keys whose turned values are under the least float, of either sign: their codes are
    0, alone in a page and beside larger ones."""
    tiny = torch.tensor([1e-30, 1e-40, 1.4e-45, 6e-8, 0.0, 1e-38])
    f = torch.tensor([1e-9, 1e-7, 1e-20, 1e-40, math.pi / 2, 1.2, 3.0, 1e-300], dtype=torch.float64)
    for larger in (False, True):
        k = tiny.repeat(T * 6)[:T * 32].view(T, 2, 16) * torch.tensor([1.0, -1.0])[:, None]
        k[:, :, 1::3] *= -1
        if larger:
            k[T // 2, 1] = torch.linspace(-3, 3, 16)
        for at in (torch.ones(T, dtype=torch.int64), torch.arange(T) - T // 2):
            want = _append(tpo, dev, k.to(dtype), f, at, interleaved)
            assert want.k.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T", [4, 40])
def test_turned_keys_beyond_the_largest_float(tpo, dev, dtype, interleaved, T):
    """Finite keys whose turned values no float holds: the largest value that the cache has, and
    only what is not finite is NaN."""
    f = torch.tensor([math.pi / 4, 1.0, 3.0, 0.0], dtype=torch.float64)
    k = torch.full((T, 1, 16), 3e38).to(dtype)
    k[::2] *= -1
    k[T // 2], k[T // 2 + 1] = 1.0, 1e30
    at = torch.arange(T) % 3
    for amplitude in (1.0, 8.0):
        want = _append(tpo, dev, k, f, at, interleaved, amplitude)
        assert want.k.isfinite().all() and (want.ks == 2.0 ** 40).any()
    k[1, 0, 2], k[3, 0, 5], k[3, 0, 12] = float("inf"), float("nan"), float("-inf")
    want = _append(tpo, dev, k, f, at, interleaved)
    assert want.k.isnan().any()


# Tables of an odd number of pages that are an odd number of blocks, the last sequence as long as
# its table: the last two blocks of 32 tokens that go together are not both there.
# (page, pages of a sequence); tests/test_cache_table_cpu.py looks up which kernel takes them.
FULL = [(32, 1), (32, 7), (96, 1), (96, 3), (160, 1), (224, 3)]
FULL_NEW, FULL_HEADS, FULL_D = 16 * [30], 32, 72


@pytest.mark.parametrize("page,M", FULL)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_over_full_tables(tpo, dev, page, M, dtype, causal):
    B, T = len(FULL_NEW), sum(FULL_NEW)
    lengths = [max(30, page * M - 11 * b) for b in reversed(range(B))]
    lengths[3] = page * M
    cache = cache64.paged(tpo, dev, lengths, FULL_HEADS, FULL_D, page, seed=page)
    assert cache.table.shape == (B, M) and lengths[-1] == page * M
    g = torch.Generator().manual_seed(M)
    q = torch.randn(T, 2 * FULL_HEADS, FULL_D, generator=g).to(dtype)
    o = torch.arange(B + 1) * 30
    got = tpo.cached_attention(q.to(dev), cache, o.to(dev), causal=causal)
    want = cache64.Cache(cache).attention(q, o.tolist(), causal=causal)
    nn64.near(got, want, roundings=2)  # probabilities and the result


def _levels(tpo, dev, lengths, Hk, D, page, apart, order, seed):
    """A cache whose pages are of two kinds: small values in all of a head's channels, and values
    2^apart times as large in channel 3 and nothing in the others."""
    cache = cache64.paged(tpo, dev, lengths, Hk, D, page, seed)
    cache.value_scales.fill_(2.0 ** -19)
    for row in cache.table.tolist():
        for i, p in enumerate(row):
            if p >= 0 and order(i):
                codes = cache.values.view(torch.uint8)[p]
                kept = codes[:, :, 3].clone()
                codes.zero_()
                codes[:, :, 3] = kept
                cache.value_scales[p] = 2.0 ** (apart - 19)
    return cache


def _channels(cache, got, q, o, causal=True):
    """Every value by itself: probabilities are off by a rounding each, and by 2^-24 of their sum,
    which is 1; then the result is rounded (half's steps end at 2^-24).  Floats end at 2^-126, and
    bfloat16 with them: a result under that is 0, and so is a weight, the probability times the
    page's scale against the row's largest such product.  With scales at most 2^80 apart that
    probability is under 2^-126 2^80, so that a key's part of the result is off by 2^-46 of its
    value at most."""
    model = cache64.Cache(cache)
    want = model.attention(q, o, causal=causal)
    model.v = model.v.abs()
    sums = model.attention(q, o, causal=causal)
    G = q.shape[1] // model.Hk
    most = (model.v * model.vs[..., None, None]).amax((0, 2))[:, :q.shape[2]]
    most = most.repeat_interleave(G, 0)
    n = max(cache.lengths.tolist())
    tol = (2 * nn64.U[q.dtype] + 1e-5) * sums + n * 2.0 ** -46 * most + 2.0 ** -126
    if q.dtype == torch.float16:
        tol = tol + n * 2.0 ** -24 * most + 2.0 ** -25
    got = got.cpu().double()
    there = want.abs() < 6e4  # (more is infinite in half, and no case of this test)
    assert there[..., [c for c in range(q.shape[2]) if c != 3]].all()
    off = ((got - want).abs() / tol)[there]
    assert off.max() <= 1, off.max().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("apart", [1, 3, 8, 16, 24, 40, 59, 80])
def test_small_values_beside_large_ones(tpo, dev, dtype, apart):
    """A page of large values in one channel leaves the others' small ones their bits, whatever
    comes first and however many workgroups and waves have the keys."""
    orders = (lambda i: i == 0, lambda i: i % 2 == 1, lambda i: i % 3 != 1, lambda i: i >= 3)
    for n, order in enumerate(orders):
        for lengths, new, page in (([500, 70, 1], [3, 40, 1], 32), ([3000], [2], 64)):
            cache = _levels(tpo, dev, lengths, 2, 32, page, apart, order, 7 * n)
            g = torch.Generator().manual_seed(n)
            q = torch.randn(sum(new), 4, 32, generator=g).to(dtype)
            o = [0]
            for c in new:
                o.append(o[-1] + c)
            got = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
            _channels(cache, got, q, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("apart", [3, 16, 40, 80])
@pytest.mark.parametrize("page", [32, 96])
def test_small_values_beside_large_ones_in_prompts(tpo, dev, dtype, apart, page):
    """The same by 128 rows, whose blocks of 32 go two at a time: of one page and of two."""
    B = len(FULL_NEW)
    for n, order in enumerate((lambda i: i == 0, lambda i: i % 2 == 1, lambda i: i % 3 != 1)):
        lengths = [30 + 13 * b for b in range(B)]
        cache = _levels(tpo, dev, lengths, FULL_HEADS, FULL_D, page, apart, order, n)
        g = torch.Generator().manual_seed(n)
        q = torch.randn(sum(FULL_NEW), 2 * FULL_HEADS, FULL_D, generator=g).to(dtype)
        o = (torch.arange(B + 1) * 30).tolist()
        got = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
        _channels(cache, got, q, o)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("gone", [0, 1, 2])
def test_small_values_beside_a_page_that_is_not_there(tpo, dev, dtype, gone):
    """A block of small values next to one whose page is not there, with scores beyond half's
    range: what is not there weighs nothing, also before a row has seen a key."""
    B = len(FULL_NEW)
    lengths = [100 + 13 * b for b in range(B)]
    cache = _levels(tpo, dev, lengths, FULL_HEADS, FULL_D, 32, 20, lambda i: i >= 2, gone)
    cache.table[:, gone] = -1
    g = torch.Generator().manual_seed(gone)
    q = (4 * torch.randn(sum(FULL_NEW), 2 * FULL_HEADS, FULL_D, generator=g)).to(dtype)
    o = (torch.arange(B + 1) * 30).tolist()
    got = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
    assert got.isfinite()[..., [c for c in range(FULL_D) if c != 3]].all()
    _channels(cache, got, q, o)
