"""cached_attention against its definition in float64: lengths, masks, pages, what lies behind."""
import pytest
import torch

from tests import cache64, nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _q(T, Hq, D, dtype, seed):
    return torch.randn(T, Hq, D, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _offsets(counts, before=0):
    o = [before]
    for n in counts:
        o.append(o[-1] + n)
    return o


def _check(tpo, dev, new, lengths, Hq, Hk, D, dtype, page=64, causal=True, scale=None, lq=None,
           before=0, after=0, seed=0, cache=None, spread=0.5):
    if cache is None:
        cache = cache64.paged(tpo, dev, lengths, Hk, D, page, seed, spread=spread)
    o = _offsets(new, before)
    q = _q(o[-1] + after, Hq, D, dtype, seed)
    want = cache64.Cache(cache).attention(q, o, lq, causal, scale)
    ln = None if lq is None else torch.tensor(lq, device=dev)
    out = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev), ln, causal, scale)
    assert out.dtype == dtype and out.shape == q.shape
    # float16 ends at 65504, and what rounds to more (from 65520 on) is infinite in it; the sums of
    # pages with scales of 2^36 are beyond.  A result that is off by two roundings has to be
    # infinite from two roundings over the end on, and may be from two roundings under it on.
    got, end, off = out.cpu(), torch.finfo(dtype).max, 2 * nn64.U[dtype]
    over = got.isinf()
    assert (want.abs()[over] > end * (1 - off)).all() and (want.sign() == got.sign())[over].all()
    assert over[want.abs() > end * (1 + off)].all()
    nn64.near(got.masked_fill(over, 0), want.masked_fill(over, 0),
              roundings=2)  # probabilities and the result
    assert (out.cpu()[(want == 0).all(-1)] == 0).all()
    return out


# (new tokens, tokens in all): none, one, edges of blocks, pages and tiles, long ones
CASES = [([1], [1]), ([1, 1], [31, 32]), ([1, 1, 1], [33, 64, 65]), ([0, 2, 1], [7, 2, 0]),
         ([5], [300]), ([1], [1000]), ([40, 1, 0, 33], [40, 129, 5, 200]), ([130, 70], [140, 70]),
         ([1] * 40, [3 * i for i in range(40)]), ([0, 0], [4, 0])]


@pytest.mark.parametrize("new,lengths", CASES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(tpo, dev, new, lengths, dtype, causal):
    _check(tpo, dev, new, lengths, 4, 2, 64, dtype, causal=causal, seed=len(new))


@pytest.mark.parametrize("D", [1, 7, 8, 16, 20, 24, 32, 40, 63, 64, 72, 80, 96, 100, 127, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(tpo, dev, D, dtype):
    _check(tpo, dev, [3, 1, 50], [70, 1, 130], 3, 1, D, dtype, seed=D)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (3, 3), (8, 1), (12, 4), (33, 1), (40, 8), (17, 17)])
@pytest.mark.parametrize("new", [[1, 1], [20, 3]])
def test_grouped_heads(tpo, dev, Hq, Hk, new):
    _check(tpo, dev, new, [90, 41], Hq, Hk, 32, torch.bfloat16, seed=Hq)


@pytest.mark.parametrize("page", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages(tpo, dev, page, dtype):
    for n in (page - 1, page, page + 1, 3 * page + 33):
        _check(tpo, dev, [1, 2], [n, n // 2 + 2], 2, 2, 48, dtype, page=page, seed=n)


@pytest.mark.parametrize("dtype", DTYPES)
def test_levels_of_pages(tpo, dev, dtype):
    """Pages whose scales lie far apart, keys and values: sums are those of 32 bits."""
    _check(tpo, dev, [1, 4], [500, 700], 4, 2, 64, dtype, seed=3, spread=3.0, scale=0.02)
    cache = cache64.paged(tpo, dev, [640], 2, 32, 64, seed=4)
    cache.value_scales.copy_(2.0 ** (torch.arange(cache.value_scales.numel(), device=dev)
                                     .view_as(cache.value_scales) * 4.0 - 36))
    _check(tpo, dev, [3], [640], 2, 2, 32, dtype, cache=cache, seed=4)
    # pages of nothing but zeros weigh in the sum
    cache.values.view(torch.uint8)[1:7] = 0
    cache.value_scales[1:7] = 2.0 ** -40
    _check(tpo, dev, [3], [640], 2, 2, 32, dtype, cache=cache, seed=5)
    # scales that are no powers of two
    cache.value_scales.copy_(torch.rand(cache.value_scales.shape) + 0.1)
    cache.key_scales.copy_(torch.rand(cache.key_scales.shape) * 0.02 + 0.001)
    _check(tpo, dev, [3], [640], 2, 2, 32, dtype, cache=cache, seed=6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-30])
def test_scales_of_scores(tpo, dev, dtype, scale):
    _check(tpo, dev, [2, 35], [100, 64], 4, 2, 32, dtype, scale=scale, seed=7)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shares(tpo, dev, dtype):
    """Few rows over long caches: several workgroups share the keys."""
    _check(tpo, dev, [1], [5000], 2, 2, 32, dtype, seed=8)
    _check(tpo, dev, [2, 1, 1], [9000, 40, 2048], 2, 1, 64, dtype, page=256, seed=9)
    # a table with far more room than is used
    cache = cache64.paged(tpo, dev, [70, 1], 2, 32, 64, seed=10, extra=300)
    _check(tpo, dev, [1, 1], [70, 1], 4, 2, 32, dtype, cache=cache, seed=10)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_pages_a_wave(tpo, dev, dtype):
    """More tiles than a wave looks up at a time, of sequences that share their pages."""
    B, n = 40, 9000
    cache = cache64.paged(tpo, dev, [n], 32, 16, 256, seed=11)
    cache.table = cache.table.expand(B, -1).contiguous()
    cache.lengths = torch.full((B,), n, device=dev)
    cache.lengths[3], cache.lengths[7] = 8192 + 33, 8190
    q = _q(B, 32, 16, dtype, 11)
    o = list(range(B + 1))
    out = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
    model = cache64.Cache(cache)
    nn64.near(out, model.attention(q, o), roundings=2)


@pytest.mark.parametrize("B", [61, 62, 63, 64, 130])
def test_numbers_of_sequences(tpo, dev, B):
    new = [(7 * b) % 5 for b in range(B)]
    _check(tpo, dev, new, [(13 * b) % 90 + 4 for b in range(B)], 2, 1, 16, torch.float16, page=32,
           before=3, after=2, seed=B)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_not_in_use(tpo, dev, dtype):
    _check(tpo, dev, [4, 3, 40], [50, 9, 100], 4, 2, 32, dtype, lq=[2, -1, 77], before=5, after=40,
           seed=12)
    cache = cache64.paged(tpo, dev, [50, 60], 2, 32)
    for o in ([-5, 3, 99], [4, 2, 9], [10, 11, 12], [0, 8, 5]):
        q = _q(9, 4, 32, dtype, 13)
        out = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
        nn64.near(out, cache64.Cache(cache).attention(q, o), roundings=2)


@pytest.mark.parametrize("dtype", DTYPES)
def test_more_rows_than_tokens(tpo, dev, dtype):
    """Rows before a sequence's first token see nothing."""
    _check(tpo, dev, [5, 40, 3], [2, 33, 0], 2, 1, 32, dtype, seed=14)
    _check(tpo, dev, [5, 40, 3], [2, 33, 0], 2, 1, 32, dtype, seed=14, causal=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_lies_behind_counts_for_nothing(tpo, dev, dtype):
    """NaN codes and scales everywhere but in the sequences' tokens change no bit."""
    new, lengths = [1, 3, 40], [70, 33, 100]
    cache = cache64.paged(tpo, dev, lengths, 2, 32, 64, seed=15, extra=1)
    q = _q(sum(new), 4, 32, dtype, 15).to(dev)
    o = torch.tensor(_offsets(new), device=dev)
    want = tpo.cached_attention(q, cache, o)
    keys, values = cache.keys.view(torch.uint8), cache.values.view(torch.uint8)
    k, v = torch.full_like(keys, 0x7f), torch.full_like(values, 0xff)
    ks, vs = (torch.full_like(t, float("nan")) for t in (cache.key_scales, cache.value_scales))
    for b, n in enumerate(lengths):
        for j in range(n):
            p, s = int(cache.table[b, j // 64]), j % 64
            k[p, :, s // 32, :, s % 32] = keys[p, :, s // 32, :, s % 32]
            v[p, :, s // 32, :, s % 32] = values[p, :, s // 32, :, s % 32]
            ks[p], vs[p] = cache.key_scales[p], cache.value_scales[p]
    other = tpo.PagedCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs,
                           cache.table, cache.lengths)
    assert torch.equal(tpo.cached_attention(q, other, o), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_reaches_those_that_see_it(tpo, dev, dtype):
    """A NaN of a key or value reaches the rows that see it, and no other."""
    for which in ("keys", "values"):
        for place in (70, 95, 99):
            cache = cache64.paged(tpo, dev, [100, 40], 1, 32, 64, seed=16)
            q = _q(41, 2, 32, dtype, 16).to(dev)
            o = torch.tensor([0, 40, 41], device=dev)
            clean = tpo.cached_attention(q, cache, o)
            p, s = int(cache.table[0, place // 64]), place % 64
            if which == "keys":
                cache.keys.view(torch.uint8)[p, 0, s // 32, 0, s % 32, 5] = 0x7f
            else:
                cache.values.view(torch.uint8)[p, 0, s // 32, 5, s % 32] = 0xff
            got = tpo.cached_attention(q, cache, o)
            first = place - 60  # the row whose own token it is
            assert torch.equal(got[:first], clean[:first]) and torch.equal(got[40:], clean[40:])
            bad = got[first:40].isnan()
            assert bad[..., 5].all()
            assert bad.all() if which == "keys" else not bad[..., torch.arange(32) != 5].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_that_are_not_there(tpo, dev, dtype):
    cache = cache64.paged(tpo, dev, [200, 200, 200, 10], 2, 32, 32, seed=17)
    P = cache.keys.shape[0]
    cache.table[0, 1] = -1
    cache.table[1, 5:] = torch.tensor([P, 2 ** 31 - 1], dtype=torch.int32)
    cache.table[2] = -2 ** 31
    cache.lengths[3] = 10 ** 15
    _check(tpo, dev, [2, 40, 1, 1], None, 4, 2, 32, dtype, cache=cache, seed=17)
    empty = tpo.PagedCache.empty(2, 64, 2, 32, page=32, pages=0, device=dev)
    empty.lengths.fill_(50)
    o = torch.tensor([0, 1, 3], device=dev)
    q = torch.ones(3, 2, 32, device=dev, dtype=dtype)
    assert (tpo.cached_attention(q, empty, o) == 0).all()
    none = tpo.PagedCache.empty(0, 64, 2, 32, device=dev)
    assert (tpo.cached_attention(q, none, o[:1]) == 0).all()
    assert tpo.cached_attention(q[:0], empty, o).shape == (0, 2, 32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides(tpo, dev, dtype):
    cache = cache64.paged(tpo, dev, [60, 90], 2, 24, seed=18)
    y = _q(30, 9, 40, dtype, 18)
    o = [0, 20, 30]
    for view in (lambda t: t[:, 3:7, 8:32], lambda t: t[:, 1:5, 1:25], lambda t: t[:, :8:2, 16:],
                 lambda t: t[:, 2:3, :24].expand(30, 4, 24), lambda t: t[:1, :4, :24].expand(30, 4, 24)):
        want = cache64.Cache(cache).attention(view(y), o)
        nn64.near(tpo.cached_attention(view(y.to(dev)), cache, torch.tensor(o, device=dev)), want,
                  roundings=2)


# What takes the kernel of 128 rows a workgroup (tests/test_cache_api_cpu.py looks the rule up):
# sequences' new tokens and tokens, heads of the cache, query heads of each.
PROMPTS = [([40] * 20, [40 + 7 * b for b in range(20)], 32, 1),
           ([129, 1, 0, 200, 64, 63], [129, 70, 5, 260, 64, 200], 48, 2),
           ([33] * 70, [33 + 3 * b for b in range(70)], 8, 1),
           ([300, 212], [700, 3000], 52, 2)]
HALVES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [True, False])
def test_prompts(tpo, dev, which, dtype, causal):
    new, lengths, Hk, G = PROMPTS[which]
    _check(tpo, dev, new, lengths, G * Hk, Hk, 72, dtype, causal=causal, seed=which, before=3,
           after=4)


MANY = [40] * 16  # with 32 heads: 512 workgroups


@pytest.mark.parametrize("D", [65, 72, 80, 96, 100, 112, 127, 128])
@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_head_sizes(tpo, dev, D, dtype):
    _check(tpo, dev, MANY, [40 + 9 * b for b in range(16)], 32, 32, D, dtype, seed=D,
           page=32 if D % 3 else 96)


@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_levels_scales_and_rows(tpo, dev, dtype):
    lengths = [40 + 30 * b for b in range(16)]
    for scale in (-0.2, 0.0, 0.5):
        _check(tpo, dev, MANY, lengths, 64, 32, 80, dtype, seed=3, spread=3.0, scale=scale)
    _check(tpo, dev, MANY, lengths, 64, 32, 80, dtype, lq=[3 * b for b in range(16)], seed=4)
    _check(tpo, dev, MANY, [4 * b for b in range(16)], 64, 32, 80, dtype, seed=5)
    cache = cache64.paged(tpo, dev, lengths, 32, 80, 32, seed=6)
    cache.table[3, 1], cache.table[5, 0], cache.table[8] = -1, 10 ** 6, -5
    cache.lengths[9] = 10 ** 12
    _check(tpo, dev, MANY, None, 64, 32, 80, dtype, cache=cache, seed=6)


@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_past_one_look_up(tpo, dev, dtype):
    """More blocks than a wave looks up at a time (64), of sequences that share their pages."""
    cache = cache64.paged(tpo, dev, [4200], 32, 128, 256, seed=7)
    cache.table = cache.table.expand(16, -1).contiguous()
    cache.lengths = torch.tensor([4200 - 61 * b for b in range(16)], device=dev)
    q, o = _q(640, 32, 128, dtype, 7), _offsets(MANY)
    out = tpo.cached_attention(q.to(dev), cache, torch.tensor(o, device=dev))
    model, at = cache64.Cache(cache), [0, 33, 640 - 40, 639]
    for r in at:  # some rows: the model's 64 bits take their time
        b = r // 40
        n = int(cache.lengths[b]) - 39 + r % 40
        k, v, _ = model.rows(b, 128)
        a = (q[r].double()[:, None] @ k[:, :n].transpose(1, 2)) * 128 ** -0.5
        nn64.near(out[r], (torch.softmax(a, -1) @ v[:, :n])[:, 0], roundings=2)


@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_nan(tpo, dev, dtype):
    """As test_nan_reaches_those_that_see_it and test_what_lies_behind_counts_for_nothing, by the
    other kernel."""
    for which in ("keys", "values"):
        for place in (70, 95, 99):
            cache = cache64.paged(tpo, dev, [100] * 16, 32, 80, 64, seed=16)
            q = _q(640, 32, 80, dtype, 16).to(dev)
            o = torch.tensor(_offsets(MANY), device=dev)
            clean = tpo.cached_attention(q, cache, o)
            p, s = int(cache.table[4, place // 64]), place % 64
            if which == "keys":
                cache.keys.view(torch.uint8)[p, 3, s // 32, 0, s % 32, 5] = 0x7f
            else:
                cache.values.view(torch.uint8)[p, 3, s // 32, 5, s % 32] = 0xff
            p = int(cache.table[4, 1])  # behind the sequence's last place
            cache.keys.view(torch.uint8)[p, :, 1, :, 4:] = 0x7f
            cache.values.view(torch.uint8)[p, :, 1, :, 4:] = 0x7f
            got = tpo.cached_attention(q, cache, o)
            first = 160 + place - 60  # the row whose own token it is
            bad = got[first:200, 3].isnan()
            assert bad[..., 5].all()
            assert bad.all() if which == "keys" else not bad[..., torch.arange(80) != 5].any()
            got[first:200, 3] = clean[first:200, 3]
            assert torch.equal(got, clean)


@pytest.mark.parametrize("dtype", HALVES)
def test_prompts_nan_before_the_border(tpo, dev, dtype):
    """A NaN that all rows see, in a tile that not all of them see the end of (the first row sees
    places 0 .. 100), in either of its blocks."""
    for place in (64, 70, 95, 96, 100):
        cache = cache64.paged(tpo, dev, [140] * 16, 32, 80, 64, seed=24)
        q = _q(640, 32, 80, dtype, 24).to(dev)
        o = torch.tensor(_offsets(MANY), device=dev)
        clean = tpo.cached_attention(q, cache, o)
        p, s = int(cache.table[4, place // 64]), place % 64
        cache.values.view(torch.uint8)[p, 3, s // 32, 5, s % 32] = 0x7f
        got = tpo.cached_attention(q, cache, o)
        bad = torch.zeros(got.shape, dtype=torch.bool, device=dev)
        bad[160:200, 3, 5] = True
        assert torch.equal(got.isnan(), bad) and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scale_of_nothing(tpo, dev, dtype):
    """A scale of 0 over pages of the smallest scale, or of none: the mean of what a row sees."""
    for smallest in (2.0 ** -40, 0.0):
        for lengths, heads in ([70, 33], 2), ([140] * 16, 32):
            n = 5 if heads == 2 else 40
            cache = cache64.paged(tpo, dev, lengths, heads, 80, 64, seed=6)
            q = _q(n * len(lengths), heads, 80, dtype, 6).to(dev)
            o = torch.tensor(_offsets([n] * len(lengths)), device=dev)
            want = tpo.cached_attention(q, cache, o, scale=0.0)
            assert want.isfinite().all()
            cache.key_scales.fill_(smallest)
            assert torch.equal(tpo.cached_attention(q, cache, o, scale=0.0), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_pool(tpo, dev, dtype):
    """A pool of more than 256 MB, whose codes go past the caches."""
    small = cache64.paged(tpo, dev, [300, 70], 2, 64, 64, seed=23)
    P = 70000
    big = tpo.PagedCache.empty(2, 300, 2, 64, page=64, pages=P, device=dev)
    at = torch.arange(small.keys.shape[0], device=dev) * 3001 + 17
    for n in ("keys", "values"):
        getattr(big, n).view(torch.uint8)[at] = getattr(small, n).view(torch.uint8)
    for n in ("key_scales", "value_scales"):
        getattr(big, n)[at] = getattr(small, n)
    big.table = torch.where(small.table >= 0, at[small.table.long()].int(), -1)
    big.lengths = small.lengths
    q, o = _q(3, 4, 64, dtype, 23), [0, 1, 3]
    out = tpo.cached_attention(q.to(dev), big, torch.tensor(o, device=dev))
    assert torch.equal(out, tpo.cached_attention(q.to(dev), small, torch.tensor(o, device=dev)))
    nn64.near(out, cache64.Cache(small).attention(q, o), roundings=2)


def test_past_32_bits(tpo, dev):
    """Pages beyond 2^31 and 2^32 bytes of the pool, written and read."""
    P, Hk, D, page = 140000, 1, 128, 256  # 32 KB a page and head: 4.6 GB of keys
    cache = tpo.PagedCache.empty(1, 2 * page, Hk, D, page=page, pages=P, device=dev)
    g = torch.Generator().manual_seed(19)
    k, v = (torch.randn(2 * page, Hk, D, generator=g) for _ in range(2))
    q, o = _q(1, 2, D, torch.float32, 19), torch.tensor([0, 2 * page], device=dev)
    small = tpo.PagedCache.empty(1, 2 * page, Hk, D, page=page, device=dev)
    for c, table in ((small, [[0, 1]]), (cache, [[P - 1, 2 ** 16 + 3]])):
        c.table.copy_(torch.tensor(table))
        c.lengths.fill_(2 * page)
        tpo.cache_append(c, k.to(dev), v.to(dev), o)
    for i, p in ((0, P - 1), (1, 2 ** 16 + 3)):
        assert torch.equal(small.keys.view(torch.uint8)[i], cache.keys.view(torch.uint8)[p])
        assert torch.equal(small.values.view(torch.uint8)[i], cache.values.view(torch.uint8)[p])
    one = torch.tensor([0, 1], device=dev)
    a, b = (tpo.cached_attention(q.to(dev), c, one) for c in (small, cache))
    assert torch.equal(a, b)
    nn64.near(a, cache64.Cache(small).attention(q, [0, 1]), roundings=2)


def test_captured_and_on_another_stream(tpo, dev):
    """A graph replayed as the cache fills, and calls on two streams at once."""
    cache = cache64.paged(tpo, dev, [5000, 100], 2, 64, seed=20)
    q = _q(2, 4, 64, torch.bfloat16, 20).to(dev)
    o = torch.tensor([0, 1, 2], device=dev)
    tpo.cached_attention(q, cache, o)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tpo.cached_attention(q, cache, o)
    for n in (5000, 17, 4096, 0):
        cache.lengths[0] = n
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, tpo.cached_attention(q, cache, o))
    cache.lengths[0] = 5000
    want = tpo.cached_attention(q, cache, o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(tpo.cached_attention(q, cache, o))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_autocast_and_derivatives(tpo, dev):
    cache = cache64.paged(tpo, dev, [40], 1, 32)
    q, o = _q(2, 2, 32, torch.float32, 21).to(dev), torch.tensor([0, 2], device=dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a = tpo.cached_attention(q, cache, o)
    assert torch.equal(a, tpo.cached_attention(q.bfloat16(), cache, o))
    with pytest.raises(RuntimeError, match="has no derivative"):
        tpo.cached_attention(q.requires_grad_(True), cache, o)
    with torch.no_grad():
        assert tpo.cached_attention(q, cache, o).shape == q.shape


@pytest.mark.parametrize("dtype", DTYPES)
def test_generation(tpo, dev, dtype):
    """A prompt and then token by token, as a decoder runs them: rotary positions, append,
    attention; against packed attention of what the cache holds."""
    g = torch.Generator().manual_seed(22)
    B, Hq, Hk, D = 3, 4, 2, 64
    turn = tpo.RotaryPositions(D, device=dev)
    cache = tpo.PagedCache.empty(B, 256, Hk, D, device=dev)
    prompt = [50, 1, 130]
    total = torch.tensor(prompt, device=dev)
    for step in range(5):
        new = prompt if step == 0 else [1] * B
        o = torch.tensor(_offsets(new), device=dev)
        y = torch.randn(sum(new), Hq + 2 * Hk, D, generator=g).to(dev, dtype)
        q, k, v = y.split([Hq, Hk, Hk], 1)
        cache.lengths += torch.tensor(new, device=dev)
        q2 = tpo.cache_append(cache, k, v, o, q=q, frequencies=turn.frequencies)
        at = torch.cat([torch.arange(n - m, n) for m, n in zip(new, cache.lengths.tolist())])
        assert torch.equal(q2, turn(q, at.to(dev)))
        out = tpo.cached_attention(q2, cache, o)
        nn64.near(out, cache64.Cache(cache).attention(q2.cpu(), o.tolist()), roundings=2)
        # the same with the cache's contents laid out as packed_attention takes them
        K, V = (t.permute(0, 2, 1, 3).reshape(B * 256, Hk, D).to(dtype) for t in (
            x.view(B, 4, Hk, 64, D).transpose(2, 1).reshape(B, Hk, 256, D)[:, :, :, :]
            for x in cache.rows()))
        rooms = torch.arange(B + 1, device=dev) * 256
        same = tpo.packed_attention(q2, K, V, o, rooms, lengths_k=cache.lengths)
        # both are within two roundings of the exact result
        nn64.near(out, same.cpu().double(), roundings=4)
    assert torch.equal(cache.lengths, total + 4)
