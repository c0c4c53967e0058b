"""Rotary positions and the 8-bit cache inside torch's own machinery: opcheck, torch.compile,
vmap, checkpointing, another thread, a model under all of it."""
import threading

import pytest
import torch
from torch.library import opcheck

from tests import cache64, nn64

pytestmark = pytest.mark.gpu


def _rotary(dev, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(20, 4, 32, generator=g).to(dev, dtype).requires_grad_(True)
    return x, torch.arange(20, device=dev), torch.rand(16, generator=g, dtype=torch.float64).to(dev)


def _cache(tpo, dev):
    c = cache64.paged(tpo, dev, [70, 9], 2, 32, 64, seed=2)
    return c, (c.keys, c.values, c.key_scales, c.value_scales, c.table, c.lengths)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_opcheck(tpo, dev, dtype):
    ops = torch.ops
    x, at, f = _rotary(dev, dtype)
    for t in (x, x.detach()):
        opcheck(ops.torch_point_ops_rotary.rotary_positions.default, (t, at, f, True, 1.5))
    c, parts = _cache(tpo, dev)
    o = torch.tensor([0, 3, 5], device=dev)
    q, k = torch.randn(5, 4, 32, device=dev, dtype=dtype), torch.randn(5, 2, 32, device=dev,
                                                                       dtype=dtype)
    # test_schema multiplies every argument, which torch does not do to 8-bit floats; what
    # append writes to is looked at in test_versions.
    opcheck(ops.torch_point_ops_cache.attention.default, (q, *parts, o, None, True, 0.2),
            test_utils=("test_autograd_registration", "test_faketensor",
                        "test_aot_dispatch_dynamic"))
    for queries, frequencies in ((q, f), (None, f), (None, None)):
        opcheck(ops.torch_point_ops_cache.append.default,
                (k, k, *parts, o, None, queries, None, frequencies, False, 1.0),
                test_utils="test_faketensor")


def test_versions(tpo, dev):
    """append writes to the cache's codes and scales, as autograd is told, and to nothing else;
    attention writes to nothing."""
    c, parts = _cache(tpo, dev)
    o = torch.tensor([0, 3, 5], device=dev)
    k = torch.randn(5, 2, 32, device=dev)
    before = [t._version for t in parts]
    others = [t.clone() for t in parts[4:]]
    tpo.cached_attention(k, c, o)
    assert [t._version for t in parts] == before
    tpo.cache_append(c, k, k, o)
    assert [t._version for t in parts] == [v + (i < 4) for i, v in enumerate(before)]
    assert all(torch.equal(a, b) for a, b in zip(parts[4:], others))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled(tpo, dev, dtype):
    x, at, f = _rotary(dev, dtype)
    fn = torch.compile(lambda t: tpo.rotary_positions(t, at, f) * 2)
    want, got = tpo.rotary_positions(x, at, f) * 2, fn(x)
    assert torch.equal(got, want)
    gy = torch.randn_like(want)
    assert torch.equal(torch.autograd.grad(got, x, gy)[0], torch.autograd.grad(want, x, gy)[0])
    c, parts = _cache(tpo, dev)
    o = torch.tensor([0, 3, 5], device=dev)
    q = torch.randn(5, 4, 32, device=dev, dtype=dtype)
    with torch.no_grad():
        got = torch.compile(lambda t: tpo.cached_attention(t, c, o) + 1)(q)
        assert torch.equal(got, tpo.cached_attention(q, c, o) + 1)


def test_compiled_step(tpo, dev):
    """A step of generation as one graph: the cache is changed in place there too."""
    one, _ = _cache(tpo, dev)
    two, _ = _cache(tpo, dev)
    o = torch.tensor([0, 1, 2], device=dev)
    f = 4.0 ** -torch.arange(16, dtype=torch.float64, device=dev)

    def step(cache, q, k, v):
        cache.lengths += 1
        q = tpo.cache_append(cache, k * 2, v, o, q + 1, f)
        return tpo.cached_attention(q, cache, o) * 2

    fn = torch.compile(step)
    g = torch.Generator().manual_seed(4)
    with torch.no_grad():
        for _ in range(3):
            q, k, v = (torch.randn(2, h, 32, generator=g).to(dev) for h in (4, 2, 2))
            want, got = step(one, q, k, v), fn(two, q, k, v)
            assert torch.equal(got, want)
    for name in ("keys", "values"):
        assert torch.equal(getattr(one, name).view(torch.uint8), getattr(two, name).view(torch.uint8))
    for name in ("key_scales", "value_scales", "lengths"):
        assert torch.equal(getattr(one, name), getattr(two, name))


def test_vmap(tpo, dev):
    x, at, f = _rotary(dev, torch.float32)
    x = x.detach()
    xs = torch.stack([x, 2 * x, -x])
    got = torch.vmap(lambda t: tpo.rotary_positions(t, at, f))(xs)
    assert torch.equal(got, torch.stack([tpo.rotary_positions(t, at, f) for t in xs]))
    c, _ = _cache(tpo, dev)
    o, q = torch.tensor([0, 3, 5], device=dev), torch.randn(3, 5, 4, 32, device=dev)
    got = torch.vmap(lambda t: tpo.cached_attention(t, c, o))(q)
    assert torch.equal(got, torch.stack([tpo.cached_attention(t, c, o) for t in q]))


def test_checkpoint_and_hooks(tpo, dev):
    from torch.utils.checkpoint import checkpoint

    x, at, f = _rotary(dev, torch.bfloat16)
    want, = torch.autograd.grad(tpo.rotary_positions(x, at, f).float().square().sum(), x)
    y = checkpoint(lambda t: tpo.rotary_positions(t, at, f), x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y.float().square().sum(), x)[0], want)
    seen = []
    x.register_hook(seen.append)
    tpo.rotary_positions(x, at, f).float().square().sum().backward()
    assert torch.equal(seen[0], want) and torch.equal(x.grad, want)


def test_a_backward_pass_captured(tpo, dev):
    x, at, f = _rotary(dev, torch.bfloat16)
    gy = torch.randn(20, 4, 32, device=dev, dtype=torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            torch.autograd.grad(tpo.rotary_positions(x, at, f), x, gy)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad(tpo.rotary_positions(x, at, f), x, gy)
    for step in range(3):
        gy.mul_(1.5)
        at.add_(3)
        graph.replay()
        torch.cuda.synchronize()
        want = cache64.turn(gy.cpu(), at.cpu(), f.cpu(), back=True)
        nn64.near(g, want)


def test_threads(tpo, dev):
    """Calls of several threads, each on a stream of its own."""
    c, _ = _cache(tpo, dev)
    o, q = torch.tensor([0, 3, 5], device=dev), torch.randn(5, 4, 32, device=dev)
    x, at, f = _rotary(dev, torch.float32)
    want = tpo.cached_attention(q, c, o), tpo.rotary_positions(x.detach(), at, f)
    torch.cuda.synchronize()
    wrong = []

    def work():
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(20):
                got = tpo.cached_attention(q, c, o), tpo.rotary_positions(x.detach(), at, f)
                s.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want)):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_refusals(tpo, dev):
    """Arguments that do not fit are errors of the call, and leave the cache as it is."""
    c, parts = _cache(tpo, dev)
    o = torch.tensor([0, 3, 5], device=dev)
    k, q = torch.zeros(5, 2, 32, device=dev), torch.zeros(5, 4, 32, device=dev)
    f = torch.ones(16, dtype=torch.float64, device=dev)
    at = torch.arange(5, device=dev)
    import dataclasses as dc

    def turned(*a, **kw):
        return lambda: tpo.rotary_positions(*a, **kw)

    def append(*a, **kw):
        return lambda: tpo.cache_append(*a, **kw)

    def attend(*a, **kw):
        return lambda: tpo.cached_attention(*a, **kw)

    half_table = dc.replace(c, table=c.table.long())
    for call, text in [
            (turned(q[0], at, f), "expects x"), (turned(q.double(), at, f), "not implemented for"),
            (turned(q, at[:4], f), "positions must have shape"),
            (turned(q, at.int(), f), "int64 or float32"),
            (turned(q, at, f.float()), "must be float64"),
            (turned(q, at, torch.cat([f, f])), "pairs need heads"),
            (turned(q, torch.zeros(5, 3, device=dev), f), "do not share out"),
            (turned(q, at.cpu(), f), "same device"), (turned(q[..., :0], at, f), "empty"),
            (append(c, k, k[:4], o), "the same shape"), (append(c, k, k.half(), o), "one type"),
            (append(c, k[0], k[0], o), "expects k and v"),
            (append(c, k[:, :1], k[:, :1], o), "heads, the cache has"),
            (append(c, k[..., :9], k[..., :9], o), "need a cache of"),
            (append(c, k, k, o[:2]), "one entry more"), (append(c, k, k, o.int()), "int64"),
            (append(c, k, k, o, q=q), "needs frequencies"),
            (append(c, k, k, o, q=q[:4], frequencies=f), "q must have shape"),
            (append(c, k, k, o, q=q.half(), frequencies=f), "k's type"),
            (append(c, k, k, o, lengths_new=o), "one entry a sequence"),
            (append(c, k.double(), k.double(), o), "not implemented for"),
            (append(dc.replace(c, keys=c.keys.view(torch.uint8)), k, k, o), "float8_e4m3fn"),
            (append(dc.replace(c, values=c.values[:1]), k, k, o), "values must be"),
            (append(dc.replace(c, key_scales=c.key_scales.half()), k, k, o), "scales must be"),
            (append(dc.replace(c, keys=c.keys.transpose(4, 5)), k, k, o), "contiguous"),
            (append(dc.replace(c, lengths=c.lengths.cpu()), k, k, o), "same device"),
            (append(half_table, k, k, o), "table must be int32"),
            (attend(q[:, :3], c, o), "multiple of the"), (attend(q[0], c, o), "expects q"),
            (attend(q[..., :9], c, o), "need a cache of"), (attend(q, c, o[:2]), "one entry more"),
            (attend(q, half_table, o), "table must be int32"),
            (attend(q, dc.replace(c, lengths=c.lengths[:1]), o), "one entry a sequence"),
            (attend(q.double(), c, o), "not implemented for"),
            (attend(q, c, o, lengths_q=o), "one entry a sequence")]:
        with pytest.raises(RuntimeError, match=text):
            call()
    fresh = cache64.paged(tpo, dev, [70, 9], 2, 32, 64, seed=2)
    assert torch.equal(c.keys.view(torch.uint8), fresh.keys.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_through_a_block(tpo, dev, dtype):
    """Queries and keys of one projection, turned in one call by coordinates, into packed
    attention: gradients at the projection."""
    g = torch.Generator().manual_seed(3)
    T, Hq, Hk, D = 40, 4, 2, 48
    y, go = (torch.randn(T, n, D, generator=g).to(dtype) for n in (Hq + 2 * Hk, Hq))
    at = 2 * torch.rand(T, 3, generator=g) - 1
    f = torch.tensor([1.0, 3.0, 9.0, 27.0], dtype=torch.float64).repeat(3)
    o = [0, 25, 40]

    def plain(y):
        qk = cache64.turn(y[:, :Hq + Hk], at, f, True)
        return nn64.attention(qk[:, :Hq], qk[:, Hq:], y[:, Hq + Hk:], o, o, None, None, True,
                              D ** -0.5)

    Y = y.to(dev).requires_grad_(True)
    qk = tpo.rotary_positions(Y[:, :Hq + Hk], at.to(dev), f.to(dev), True)
    out = tpo.packed_attention(qk[:, :Hq], qk[:, Hq:], Y[:, Hq + Hk:], torch.tensor(o, device=dev))
    got, = torch.autograd.grad(out, Y, go.to(dev))
    (want, (gwant,)) = nn64.grads(plain, (y,), go)
    nn64.near(out, want, roundings=3)  # turned values, probabilities, the result
    # and of the gradients: scores', at the turned values, turned back
    nn64.near(got, gwant, roundings=5, floats=1e-5)
