"""packed_attention against its definition in float64: lengths, masks, layouts, gradients."""
import pytest
import torch

from tests import nn64

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _offsets(lengths, before=0):
    o = [before]
    for n in lengths:
        o.append(o[-1] + n)
    return o


def _qkv(Tq, Tk, Hq, Hk, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(T, H, D, generator=g).to(dtype)
                 for T, H in ((Tq, Hq), (Tk, Hk), (Tk, Hk), (Tq, Hq)))


def _dev(dev, *lists):
    return [None if x is None else torch.tensor(x, dtype=torch.int64, device=dev) for x in lists]


def _check(tpo, dev, lens_q, lens_k, Hq, Hk, D, dtype, causal, scale=None, lq=None, lk=None,
           before=(0, 0), after=(0, 0), seed=0, grad=True):
    """Forward and gradients; returns the GPU's results."""
    oq, ok = _offsets(lens_q, before[0]), _offsets(lens_k, before[1])
    q, k, v, go = _qkv(oq[-1] + after[0], ok[-1] + after[1], Hq, Hk, D, dtype, seed)
    s = D ** -0.5 if scale is None else scale
    want, gwant = nn64.grads(
        lambda a, b, c: nn64.attention(a, b, c, oq, ok, lq, lk, causal, s), (q, k, v), go) \
        if any(a and b for a, b in zip(lens_q, lens_k)) else \
        (torch.zeros(q.shape, dtype=torch.float64), [torch.zeros(t.shape).double() for t in (q, k, v)])
    Q, K, V = (t.to(dev).requires_grad_(grad) for t in (q, k, v))
    idx = _dev(dev, oq, ok, lq, lk)
    out = tpo.packed_attention(Q, K, V, *idx, causal=causal, scale=scale)
    assert out.dtype == dtype
    nn64.near(out, want, roundings=2)  # probabilities and the result
    # what takes no part is exactly zero
    assert (out.cpu()[(want == 0).all(-1)] == 0).all()
    if not grad:
        return out
    with torch.no_grad():
        nn64.near(tpo.packed_attention(Q, K, V, *idx, causal=causal, scale=scale), want, roundings=2)
    gs = torch.autograd.grad(out, (Q, K, V), go.to(dev))
    for a, e in zip(gs, gwant):
        # the result, probabilities or scores' gradients, and the rows' sums of
        # gradient times (rounded) output
        nn64.near(a, e, roundings=3, floats=1e-5)
    return (out, *gs)


# lengths at the edges of tiles of 32, 64 and 128 rows, none, one, long ones
LENGTHS = [[1], [0, 1, 2], [31, 32, 33], [63, 64, 65, 0], [127, 1, 129], [200, 0, 0, 57], [700],
           [0, 0], [5] * 40]


@pytest.mark.parametrize("lens", LENGTHS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_whole_sequences(tpo, dev, lens, dtype, causal):
    _check(tpo, dev, lens, lens, 4, 2, 64, dtype, causal, seed=len(lens))


@pytest.mark.parametrize("D", [1, 7, 8, 16, 24, 32, 40, 63, 64, 65, 72, 80, 96, 100, 120, 127, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_head_sizes(tpo, dev, D, dtype):
    _check(tpo, dev, [70, 1, 130], [70, 1, 130], 3, 1, D, dtype, True, seed=D)


@pytest.mark.parametrize("Hq,Hk", [(1, 1), (2, 1), (3, 3), (8, 1), (8, 2), (12, 4), (33, 1), (40, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_grouped_heads(tpo, dev, Hq, Hk, causal):
    _check(tpo, dev, [50, 3, 90], [50, 3, 90], Hq, Hk, 32, torch.bfloat16, causal, seed=Hq)


# rows enough to fill the chip without sharing keys: tiles of 128 rows
@pytest.mark.parametrize("D", [8, 33, 40, 64, 96, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows(tpo, dev, D, dtype, causal):
    lens = [600, 1, 0, 437, 130, 64, 65]
    _check(tpo, dev, lens, lens, 32, 8, D, dtype, causal, seed=D, grad=D == 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_of_rooms_in_part_used(tpo, dev, dtype, causal):
    lens_q, lens_k = [300, 200, 0, 140, 500], [500, 20, 40, 140, 130]
    _check(tpo, dev, lens_q, lens_k, 32, 16, 32, dtype, causal, lq=[290, 129, 0, 0, 499],
           lk=[333, 20, 1, 140, 127], before=(3, 5), after=(7, 2), seed=33, grad=False)


# as many workgroups by heads of their own; and by sequences of a few rows each
@pytest.mark.parametrize("D", [8, 33, 64, 96, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_heads(tpo, dev, D, dtype, causal):
    lens = [600, 1, 0, 437, 130, 64, 65]
    _check(tpo, dev, lens, lens, 32, 32, D, dtype, causal, seed=D + 1, grad=D == 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_heads_of_rooms_in_part_used(tpo, dev, dtype, causal):
    lens_q, lens_k = [300, 200, 0, 140, 500], [500, 20, 40, 140, 130]
    _check(tpo, dev, lens_q, lens_k, 64, 64, 32, dtype, causal, lq=[290, 129, 0, 0, 499],
           lk=[333, 20, 1, 140, 127], before=(3, 5), after=(7, 2), seed=34, grad=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_many_short_sequences(tpo, dev, D, dtype, causal):
    lens_q, lens_k = [b % 5 for b in range(70)], [7 * b % 200 for b in range(70)]
    _check(tpo, dev, lens_q, lens_k, 16, 8, D, dtype, causal, lk=[7 * b % 200 * (b % 3) // 2 for b in range(70)],
           seed=D + 2, grad=False)


# 33 to 64 rows a key head on average, of queries or of the heads that share keys,
# over few keys and over many (in shares)
@pytest.mark.parametrize("lens_q,lens_k,Hq", [
    ([40, 64, 33], [40, 64, 33], 1), ([40, 65, 3], [2500, 1100, 3000], 1), ([5, 7, 8], [2500, 0, 3000], 8),
    ([1, 1], [5000, 1025], 40), ([3, 4], [5, 2], 16),
])
@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_pairs_of_tiles(tpo, dev, lens_q, lens_k, Hq, D, dtype, causal):
    _check(tpo, dev, lens_q, lens_k, Hq, 1, D, dtype, causal, seed=D + Hq, grad=D == 64)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shares_of_rooms_in_part_used(tpo, dev, dtype):
    """Keys are shared by their room; of some sequences whole shares are unused."""
    _check(tpo, dev, [1, 2, 1, 1], [4000, 3000, 2000, 5000], 8, 2, 64, dtype, True,
           lk=[4000, 17, 0, 2049], seed=8)


# rows and keys of different numbers: causal rows that see no key, a few rows
# over many keys, many rows over few, no keys at all
@pytest.mark.parametrize("lens_q,lens_k", [
    ([10, 40, 64], [4, 40, 100]), ([1, 1, 1], [300, 1, 0]), ([5, 2, 0, 7], [77, 129, 50, 0]),
    ([300], [3]), ([1], [5000]), ([3, 130], [2500, 140]), ([64] * 3, [1000, 2, 64]),
    ([1] * 70, list(range(70))),
])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_rows_against_other_keys(tpo, dev, lens_q, lens_k, dtype, causal):
    _check(tpo, dev, lens_q, lens_k, 4, 1, 64, dtype, causal, seed=sum(lens_q))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_rooms_in_part_used(tpo, dev, dtype, causal):
    """Lengths within the rooms, rows outside of every sequence; garbage where nothing is used."""
    lens_q, lens_k = [40, 33, 1, 70], [100, 64, 40, 200]
    lq, lk = [17, 0, 1, 99], [100, 30, 0, 77]  # one beyond its room: clamped
    oq, ok = _offsets(lens_q, 5), _offsets(lens_k, 3)
    q, k, v, go = _qkv(oq[-1] + 9, ok[-1] + 2, 4, 2, 40, dtype, 1)
    uq, uk = torch.zeros(q.shape[0], dtype=torch.bool), torch.zeros(k.shape[0], dtype=torch.bool)
    for used, o, n in ((uq, oq, lq), (uk, ok, lk)):
        for s, c in nn64.sequences(o, n, len(used)):
            used[s:s + c] = True
    s = 40 ** -0.5
    want, gwant = nn64.grads(
        lambda a, b, c: nn64.attention(a, b, c, oq, ok, lq, lk, causal, s), (q, k, v), go)
    q[~uq], k[~uk], v[~uk], go[~uq] = (float("nan"), float("inf"), float("nan"), float("inf"))
    Q, K, V = (t.to(dev).requires_grad_(True) for t in (q, k, v))
    out = tpo.packed_attention(Q, K, V, *_dev(dev, oq, ok, lq, lk), causal=causal)
    gs = torch.autograd.grad(out, (Q, K, V), go.to(dev))
    nn64.near(out, want, roundings=2)
    for a, e, u in zip(gs, gwant, (uq, uk, uk)):
        nn64.near(a, e, roundings=3, floats=1e-5)
        assert (a.cpu()[~u] == 0).all()
    assert (out.cpu()[~uq] == 0).all()


def test_padded_batch_with_lengths(tpo, dev):
    """A padded batch of clouds and its lengths, keys packed as the queries are."""
    B, P, H, D = 3, 50, 2, 32
    q, k, v, _ = _qkv(B * P, B * P, H, H, D, torch.float16, 2)
    n = [50, 20, 1]
    oq = [b * P for b in range(B + 1)]
    want = nn64.attention(q, k, v, oq, oq, n, n, True, D ** -0.5)
    o, l = _dev(dev, oq, n)
    got = tpo.packed_attention(q.to(dev), k.to(dev), v.to(dev), o, lengths_q=l)
    nn64.near(got, want, roundings=2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 40, 33])
def test_slices_of_one_projection(tpo, dev, dtype, D):
    g = torch.Generator().manual_seed(D)
    H, T = 3, 150
    one = torch.randn(T, 3, H, D, generator=g).to(dtype)
    o = [0, 100, 150]
    X = one.to(dev).requires_grad_(True)
    out = tpo.packed_attention(X[:, 0], X[:, 1], X[:, 2], *_dev(dev, o))
    go = torch.randn(T, H, D, generator=g).to(dtype)
    want, (gwant,) = nn64.grads(
        lambda x: nn64.attention(x[:, 0], x[:, 1], x[:, 2], o, o, None, None, True, D ** -0.5),
        (one,), go)
    nn64.near(out, want, roundings=2)
    gx, = torch.autograd.grad(out, X, go.to(dev))
    nn64.near(gx, gwant, roundings=3, floats=1e-5)
    # heads before rows, a reversed-order view, data off the 16-byte grid
    by_head = one.permute(2, 0, 1, 3).contiguous().to(dev).permute(1, 2, 0, 3)
    nn64.near(tpo.packed_attention(*by_head.unbind(1), *_dev(dev, o)), want, roundings=2)
    wide = torch.zeros(T, 3, H, D + 3, dtype=dtype, device=dev)
    wide[..., 1:D + 1] = X.detach()
    nn64.near(tpo.packed_attention(*wide[..., 1:D + 1].unbind(1), *_dev(dev, o)), want, roundings=2)
    inner = X.detach().transpose(2, 3).contiguous().transpose(2, 3)
    nn64.near(tpo.packed_attention(*inner.unbind(1), *_dev(dev, o)), want, roundings=2)


def test_broadcast_inputs(tpo, dev):
    """One key head expanded to all: its gradient is the sum over them."""
    q, k, v, go = _qkv(90, 90, 6, 1, 64, torch.float32, 7)
    o = [0, 60, 90]
    K, V = (t.to(dev).requires_grad_(True) for t in (k, v))
    Q, idx = q.to(dev), _dev(dev, o)
    out = tpo.packed_attention(Q, K.expand(-1, 6, -1), V.expand(-1, 6, -1), *idx)
    want, gwant = nn64.grads(lambda b, c: nn64.attention(q, b, c, o, o, None, None, True, 0.125),
                             (k, v), go)
    nn64.near(out, want)
    for a, e in zip(torch.autograd.grad(out, (K, V), go.to(dev)), gwant):
        nn64.near(a, e, floats=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_and_equal_scores(tpo, dev, dtype):
    """Scores far apart (one key takes all), all equal, and of the size where exp overflows."""
    q, k, v, _ = _qkv(100, 100, 2, 2, 64, dtype, 3)
    o = [0, 100]
    for f, s in ((0.0, 1.0), (4.0, 8.0), (8.0, -4.0)):
        a = (q * f).to(dtype)
        want = nn64.attention(a, k, v, o, o, None, None, False, s)
        got = tpo.packed_attention(a.to(dev), k.to(dev), v.to(dev), *_dev(dev, o), causal=False,
                                   scale=s)
        # a score of size |s| f |q k| ~ 1000 is off by some 2^-24 of it, and its
        # exponential by that absolutely
        nn64.near(got, want, roundings=2, floats=2e-3 if f else 2e-6)


def test_infinite_scores_stay_in_their_rows(tpo, dev):
    """A key at -infinity has no weight; an infinite query spoils no row but its own."""
    q, k, v, _ = _qkv(40, 40, 1, 1, 32, torch.float32, 3)
    q[:, 0, 0], k[:, 0, 0] = 1.0, 0.0
    k[5, 0, 0] = float("-inf")
    want = nn64.attention(q, torch.cat([k[:5], k[6:]]), torch.cat([v[:5], v[6:]]), [0, 40], [0, 39],
                          None, None, False, 1.0)
    got = tpo.packed_attention(q.to(dev), k.to(dev), v.to(dev), *_dev(dev, [0, 40]), causal=False,
                               scale=1.0)
    nn64.near(got, want, floats=1e-5)
    k[:, 0, 0] = float("-inf")  # every score: no key has weight
    got = tpo.packed_attention(q.to(dev), k.to(dev), v.to(dev), *_dev(dev, [0, 40]), causal=False)
    assert (got == 0).all()
    q, k, v, _ = _qkv(40, 40, 1, 1, 32, torch.float32, 4)
    clean = tpo.packed_attention(q.to(dev), k.to(dev), v.to(dev), *_dev(dev, [0, 40]))
    q[7] = float("inf")
    got = tpo.packed_attention(q.to(dev), k.to(dev), v.to(dev), *_dev(dev, [0, 40]))
    keep = torch.arange(40) != 7
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])


def test_gradient_against_differences(tpo, dev):
    oq, ok = [0, 9, 20], [0, 14, 22]
    q, k, v, go = _qkv(20, 22, 4, 2, 16, torch.float32, 5)
    Q, K, V = (t.to(dev).requires_grad_(True) for t in (q, k, v))
    got = torch.autograd.grad(tpo.packed_attention(Q, K, V, *_dev(dev, oq, ok)), (Q, K, V),
                              go.to(dev))
    g = torch.Generator().manual_seed(1)
    for at in range(3):
        d = [torch.randn(t.shape, generator=g, dtype=torch.float64) * (i == at)
             for i, t in enumerate((q, k, v))]
        want = nn64.slope(
            lambda a, b, c: (nn64.attention(a, b, c, oq, ok, None, None, True, 0.25)
                             * go.double()).sum(), [t.double() for t in (q, k, v)], d, 1e-5)
        have = (got[at].cpu().double() * d[at]).sum()
        assert abs(have - want) <= 1e-5 * got[at].norm().item() * d[at].norm().item()


@pytest.mark.parametrize("lens_q,lens_k", [([300, 64], [300, 64]), ([1, 2], [3000, 700])])
def test_results_repeat(tpo, dev, lens_q, lens_k):
    a = _check(tpo, dev, lens_q, lens_k, 4, 2, 64, torch.bfloat16, True, seed=3)
    b = _check(tpo, dev, lens_q, lens_k, 4, 2, 64, torch.bfloat16, True, seed=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_bad_offsets_stay_inside(tpo, dev):
    """Offsets and lengths outside of the arrays are clamped: nothing is read or written there."""
    q, k, v, _ = _qkv(64, 64, 2, 2, 32, torch.float32, 6)
    Q, K, V = (t.to(dev) for t in (q, k, v))
    out = tpo.packed_attention(Q, K, V, *_dev(dev, [0, 64], [0, 1000]), causal=False)
    nn64.near(out, nn64.attention(q, k, v, [0, 64], [0, 64], None, None, False, 32 ** -0.5))
    out = tpo.packed_attention(Q, K, V, *_dev(dev, [-5, 64], [-9, 64], None, [10 ** 12]))
    nn64.near(out, nn64.attention(q, k, v, [0, 64], [0, 64], None, None, True, 32 ** -0.5))


def test_side_stream_and_graph(tpo, dev):
    q, k, v, go = _qkv(200, 200, 4, 2, 64, torch.bfloat16, 8)
    Q, K, V = (t.to(dev).requires_grad_(True) for t in (q, k, v))
    G, (o,) = go.to(dev), _dev(dev, [0, 130, 200])

    def both():
        # detached: a graph that is kept holds its leaves to the stream they were used on
        out = tpo.packed_attention(Q, K, V, o)
        return (out.detach(), *torch.autograd.grad(out, (Q, K, V), G))

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
    for cut in (130, 1, 199):  # other lengths in the captured call
        o[1] = cut
        graph.replay()
        torch.cuda.synchronize()
        e = both()
        assert all(torch.equal(a, b) for a, b in zip(e, r))


def test_step_by_step_over_a_cache(tpo, dev):
    """Tokens fed one at a time over a growing cache give the whole prompt's rows."""
    B, P, Hq, Hk, D = 3, 37, 4, 2, 64
    q, k, v, _ = _qkv(B * P, B * P, Hq, Hk, D, torch.float32, 9)
    Q, K, V = (t.to(dev) for t in (q, k, v))
    o, one = _dev(dev, [b * P for b in range(B + 1)], list(range(B + 1)))
    whole = tpo.packed_attention(Q, K, V, o).view(B, P, Hq, D)
    ck, cv = (torch.full((B, P, Hk, D), float("nan"), device=dev) for _ in range(2))
    used = torch.zeros(B, dtype=torch.int64, device=dev)
    for t in range(P):
        ck[:, t], cv[:, t] = K.view(B, P, Hk, D)[:, t], V.view(B, P, Hk, D)[:, t]
        used += 1
        step = tpo.packed_attention(Q.view(B, P, Hq, D)[:, t], ck.view(-1, Hk, D),
                                    cv.view(-1, Hk, D), one, o, lengths_k=used)
        nn64.near(step, whole[:, t].cpu().double())


@pytest.mark.parametrize("causal", [True, False])
def test_many_sequences(tpo, dev, causal):
    """More sequences than a wave has lanes, of more than one tile each."""
    lens = [150 + b for b in range(70)]
    _check(tpo, dev, lens, lens, 2, 1, 32, torch.bfloat16, causal, seed=70)


def test_cache_beyond_32_bits(tpo, dev):
    """Sequences that begin more than 2^32 bytes into the arrays of keys and values."""
    H, D, n = 8, 128, 300
    T = (1 << 32) // (H * D * 2) + 2 * n
    q, k, v, go = _qkv(2 * n, 2 * n, H, H, D, torch.bfloat16, 12)
    K, V = (torch.empty(T, H, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for big, small in ((K, k), (V, v)):
        big[:n], big[-n:] = small[:n], small[-n:]
    oq, ok = [0, n, 2 * n], [0, T - n, T]
    want = nn64.attention(q, k, v, oq, oq, None, None, True, D ** -0.5)
    lk = [n, n]
    got = tpo.packed_attention(q.to(dev), K, V, *_dev(dev, oq, ok, None, lk))
    nn64.near(got, want, roundings=2)
    last = torch.tensor([0, n - 1, n, 2 * n - 1])  # one row a sequence: every key, by shares
    step = tpo.packed_attention(q.to(dev)[last[1::2]], K, V, *_dev(dev, [0, 1, 2], ok, None, lk))
    nn64.near(step, want[last[1::2]], roundings=2)


def test_empty_calls(tpo, dev):
    for Tq, Tk, o in ((0, 0, [0]), (0, 5, [0, 0]), (4, 0, [0, 0]), (4, 3, [0])):
        q, k, v = (torch.ones(T, 2, 16, device=dev, requires_grad=True) for T in (Tq, Tk, Tk))
        idx, = _dev(dev, o)
        out = tpo.packed_attention(q, k, v, idx)
        gs = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        assert (out == 0).all() and all((g == 0).all() for g in gs)
        assert [g.shape for g in gs] == [q.shape, k.shape, v.shape]


def test_refusals(tpo, dev):
    q, k, o = torch.ones(8, 4, 16, device=dev), torch.ones(8, 2, 16, device=dev), \
        torch.tensor([0, 8], device=dev)
    ok = lambda **kw: dict({"q": q, "k": k, "v": k, "offsets_q": o}, **kw)  # noqa: E731
    tpo.packed_attention(**ok())
    for kw, words in [
            (ok(q=q[0]), "expects q"), (ok(v=k[:7]), "same shape"), (ok(q=q[..., :8]), "head size"),
            (ok(q=q[:, :3]), "multiple"), (ok(q=q.half()), "one type"),
            (ok(q=q.double(), k=k.double(), v=k.double()), "not implemented for"),
            (ok(offsets_q=o.int()), "int64"), (ok(offsets_q=o.cpu()), "same device"),
            (ok(offsets_k=torch.cat([o, o])), "differ in length"),
            (ok(lengths_q=torch.cat([o, o])), "lengths"),
            (ok(q=torch.ones(8, 2, 129, device=dev), k=torch.ones(8, 2, 129, device=dev),
                v=torch.ones(8, 2, 129, device=dev)), "D at most 128")]:
        with pytest.raises(RuntimeError, match=words):
            tpo.packed_attention(**kw)
    with pytest.raises(ValueError, match="needs offsets_k"):
        tpo.packed_attention(**ok(lengths_k=o[1:]))
