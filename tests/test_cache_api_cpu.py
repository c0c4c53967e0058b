"""Rotary positions and the 8-bit cache without a GPU: fake shapes, the CPU's answer, refusals of
Python and of the C entries, derivatives, what the constructors make."""
import ctypes
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

from tests import cache64

P, I, D, C = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_int
APPEND = [C] + [P] * 5 + [I] * 10 + [P, C, I, P, I, C, D] + [P] * 6 + [I] * 5 + [P, P]
ATTEND = [C] + [P] * 3 + [I] * 6 + [P] * 6 + [I] * 5 + [C, D, P, P, I, P]


@pytest.fixture(scope="module")
def lib(tpo):
    from torch_point_ops import _native

    L = ctypes.CDLL(_native.HIP_LIB)
    L.tpo_last_error.restype = ctypes.c_char_p
    L.tpo_rotary.argtypes = [C, P, I, I, I, I, I, P, C, I, P, I, C, D, C, P, P]
    L.tpo_cache_append.argtypes = APPEND
    L.tpo_cache_attention.argtypes = ATTEND
    L.tpo_cache_attention_workspace_size.argtypes = [C] + [I] * 7
    L.tpo_cache_attention_workspace_size.restype = I
    return L


def _cache(tpo, device=None, B=2, Hk=2, size=32, page=64):
    return tpo.PagedCache.empty(B, 2 * page, Hk, size, page=page, device=device)


def _ops():
    return torch.ops.torch_point_ops_cache


def _parts(c):
    return (c.keys, c.values, c.key_scales, c.value_scales, c.table, c.lengths)


def test_fake_shapes(tpo):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, f = torch.empty(7, 4, 32, dtype=torch.bfloat16), torch.empty(16, dtype=torch.float64)
        at, o = torch.empty(7, dtype=torch.int64), torch.empty(3, dtype=torch.int64)
        y = tpo.rotary_positions(x, at, f)
        assert y.shape == x.shape and y.dtype == x.dtype
        c = _cache(tpo)
        k = torch.empty(7, 2, 32, dtype=torch.bfloat16)
        assert tpo.cache_append(c, k, k, o) is None
        assert tpo.cache_append(c, k, k, o, q=x, frequencies=f).shape == x.shape
        y = tpo.cached_attention(x, c, o)
        assert y.shape == x.shape and y.dtype == x.dtype


def test_cpu_tensors_are_refused(tpo):
    x, f, o = torch.ones(4, 2, 32), torch.ones(4, dtype=torch.float64), torch.tensor([0, 2, 4])
    for t in (x, x.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="rotary_positions is not implemented for CPU"):
            tpo.rotary_positions(t, torch.arange(4), f)
    with pytest.raises(RuntimeError, match="cache_append is not implemented for CPU"):
        tpo.cache_append(_cache(tpo), x, x, o)
    with pytest.raises(RuntimeError, match="cached_attention is not implemented for CPU"):
        tpo.cached_attention(x, _cache(tpo), o)


def test_python_refusals(tpo):
    for bad in (31, -2):
        with pytest.raises(ValueError, match="size must be even"):
            tpo.RotaryPositions(bad)
    with pytest.raises(ValueError, match="frequencies must have shape"):
        tpo.RotaryPositions(8, frequencies=torch.ones(3))
    for bad in ((-1,), (4, 0.0), (4, 1e4, -1.0)):
        with pytest.raises(ValueError, match="must be positive"):
            tpo.rotary_frequencies(*bad)
    for page in (0, 16, 48, 288):
        with pytest.raises(ValueError, match="page must be"):
            tpo.PagedCache.empty(1, 10, 1, 32, page=page)
    for bad in ((-1, 10, 1, 32), (1, -1, 1, 32), (1, 10, 0, 32), (1, 10, 1, 0), (1, 10, 1, 129)):
        with pytest.raises(ValueError, match="bad sizes"):
            tpo.PagedCache.empty(*bad)


def test_frequencies(tpo):
    f = tpo.rotary_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, 100.0 ** (-torch.arange(8) / 8).double())
    assert torch.equal(tpo.rotary_frequencies(8, 100.0, stretch=4.0), f / 4)
    # over 200 tokens the first turns 31.8 times, the last less than once
    g = tpo.rotary_frequencies(8, 100.0, stretch=4.0, trained=200)
    turns = 200 * f / (2 * math.pi)
    assert g[-1] == f[-1] / 4 if turns[-1] <= 1 else True
    assert (g <= f).all() and (g >= f / 4).all() and (g[1:] < g[:-1]).all()
    assert torch.equal(tpo.rotary_frequencies(4, 1.0, 4.0, trained=10 ** 6), torch.ones(4).double())
    m = tpo.RotaryPositions(8, interleaved=True).half()
    assert m.frequencies.dtype == torch.float64 and not list(m.parameters())
    assert tpo.RotaryPositions(6, frequencies=torch.ones(3)).frequencies.dtype == torch.float64


def test_empty_cache(tpo):
    c = tpo.PagedCache.empty(3, 130, 2, 40, page=64)
    assert c.keys.shape == (9, 2, 2, 3, 32, 16) and c.values.shape == (9, 2, 2, 48, 32)
    assert c.keys.dtype == c.values.dtype == torch.float8_e4m3fn and c.page == 64
    assert c.table.tolist() == [[0, 1, 2], [3, 4, 5], [6, 7, 8]] and c.lengths.tolist() == [0, 0, 0]
    k, v = c.rows()
    assert k.shape == v.shape == (9, 2, 64, 48) and (k == 0).all() and (v == 0).all()
    c = tpo.PagedCache.empty(3, 130, 2, 40, page=64, pages=5)
    assert c.keys.shape[0] == 5 and (c.table == -1).all()


def test_rows_are_codes_times_scales(tpo):
    c = cache64.paged(tpo, "cpu", [70, 30], 2, 40, 64, seed=1)
    want, (k, v) = cache64.Cache(c), c.rows()
    assert torch.equal(k.double(), want.k * want.ks[..., None, None])
    assert torch.equal(v.double(), want.v * want.vs[..., None, None])


def test_the_definition_rounds_as_torch_does():
    """The oracle's rounding to codes against torch's conversion, at every code and border."""
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (codes[1:] + codes[:-1]) / 2
    x = torch.cat([codes, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20)])
    x = torch.cat([x, -x])
    assert torch.equal(cache64.to_code(x), x.float().to(torch.float8_e4m3fn).double())
    assert cache64.to_code(torch.tensor([math.inf, math.nan]).double()).isnan().all()
    for top, e in ((0.0, -40), (448.0, 0), (448.5, 1), (1e-30, -40), (1e30, 40), (224.0, -1)):
        assert cache64.exponent(top) == e


def test_a_gradient_that_would_be_left_out_is_refused(tpo):
    x = torch.empty(6, 2, 32, device="meta")
    o = torch.empty(3, dtype=torch.int64, device="meta")
    at = torch.empty(6, device="meta")
    f = torch.empty(16, dtype=torch.float64, device="meta")
    c = _cache(tpo, "meta")

    def calls(t):
        yield lambda: tpo.cached_attention(t, c, o)
        yield lambda: tpo.cache_append(c, t, x, o)
        yield lambda: tpo.cache_append(c, x, t, o)
        yield lambda: tpo.cache_append(c, x, x, o, q=t, frequencies=f)

    for call in calls(torch.empty_like(x).requires_grad_(True)):
        with pytest.raises(RuntimeError, match="has no derivative"):
            call()
        with torch.no_grad():
            call()
    with fw.dual_level():
        for call in calls(fw.make_dual(torch.empty_like(x), torch.empty_like(x))):
            with pytest.raises(RuntimeError, match="has no derivative"):
                call()
    for bad in ({"positions": at.requires_grad_(True)}, {"frequencies": f.requires_grad_(True)}):
        with pytest.raises(RuntimeError, match="no derivative in positions"):
            tpo.rotary_positions(x, **{"positions": at.detach(), "frequencies": f.detach(), **bad})
    c.key_scales.requires_grad_(True)
    with pytest.raises(RuntimeError, match="has no derivative"):
        tpo.cached_attention(x, c, o)
    with pytest.raises(RuntimeError, match="has no derivative"):
        tpo.cache_append(c, x, x, o)


def test_derivatives_of_rotary_positions(tpo):
    x = torch.empty(6, 2, 32, device="meta", requires_grad=True)
    at = torch.empty(6, dtype=torch.int64, device="meta")
    f = torch.empty(16, dtype=torch.float64, device="meta")
    y = tpo.rotary_positions(x, at, f)
    # (linear: only a gradient that itself comes from x has a second derivative)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    assert g.shape == x.shape
    with pytest.raises(RuntimeError, match="_backward is not implemented"):
        torch.autograd.grad(g.sum(), x, allow_unused=True)
    for grad in (False, True):
        with fw.dual_level():
            t = fw.make_dual(x.detach().requires_grad_(grad), torch.empty_like(x))
            with pytest.raises(RuntimeError, match="jvp is not implemented"):
                tpo.rotary_positions(t, at, f)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp is not implemented"):
                tpo.rotary_positions(t, at, f)


def test_rotary_entry(lib):
    f = P(4096)  # never dereferenced: the calls fail their checks first
    good = [0, f, 4, 2, 32, 64, 32, f, 4, 1, f, 16, 0, 1.0, 0, f, None]

    def call(**changes):
        a = list(good)
        for at, v in changes.items():
            a[int(at[1:])] = v
        return lib.tpo_rotary(*a)

    for bad in ({"_2": -1}, {"_2": 1 << 31}, {"_3": -1}, {"_3": 1 << 20}, {"_4": 0}, {"_4": 513},
                {"_9": 0}, {"_9": 3}, {"_11": -1}, {"_11": 17}):
        assert call(**bad) == -1, bad
        assert b"bad sizes" in lib.tpo_last_error()
    assert call(_0=1) == -2 and call(_8=2) == -2
    assert call(_2=0) == 0 and call(_3=0) == 0
    for at in (1, 7, 10, 15):
        assert call(**{f"_{at}": None}) == -1 and b"NULL" in lib.tpo_last_error()
    assert call(_2=(1 << 31) - 1, _4=512, _11=256) == -1 and b"too many tokens" in lib.tpo_last_error()


def _append_args():
    f = P(4096)
    #       k  v  q  offsets lengths_new B T Hq D   strides                   places
    return [0, f, f, f, f, None, 2, 4, 2, 32, 64, 32, 64, 32, 64, 32, None, 4, 1, f, 16, 0, 1.0,
            f, f, f, f, f, f, 8, 2, 64, 32, 4, f, None]


def test_append_entry(lib):
    def call(**changes):
        a = _append_args()
        for at, v in changes.items():
            a[int(at[1:])] = v
        return lib.tpo_cache_append(*a)

    for bad in ({"_6": -1}, {"_7": -1}, {"_7": 1 << 31}, {"_8": 0}, {"_8": 2000}, {"_9": 0},
                {"_9": 48}, {"_9": 129}, {"_20": 17}, {"_20": -1}, {"_29": -1}, {"_30": 0},
                {"_30": 1025}, {"_31": 48}, {"_31": 0}, {"_31": 512}, {"_32": 48}, {"_33": -1},
                {"_33": 1 << 26}, {"_33": (1 << 24) + 1}):
        assert call(**bad) == -1, bad
        assert b"bad sizes" in lib.tpo_last_error(), bad
    assert call(_0=1) == -2 and call(_16=P(4096), _17=2) == -2
    assert call(_7=0) == 0
    for at in (1, 2, 4, 19, 23, 24, 25, 26, 27, 28, 34):
        assert call(**{f"_{at}": None}) == -1 and b"NULL" in lib.tpo_last_error(), at
    assert call(_23=P(4104)) == -1 and b"16-byte aligned" in lib.tpo_last_error()
    assert call(_7=(1 << 31) - 1) == -1 and b"too many tokens" in lib.tpo_last_error()


def test_attention_entry(lib):
    f = P(4096)
    good = [0, f, f, None, 2, 4, 4, 32, 128, 32, f, f, f, f, f, f, 8, 2, 64, 32, 4, 1, 1.0, f,
            None, 0, None]

    def call(**changes):
        a = list(good)
        for at, v in changes.items():
            a[int(at[1:])] = v
        return lib.tpo_cache_attention(*a)

    for bad in ({"_4": -1}, {"_5": -1}, {"_5": 1 << 30}, {"_6": 3}, {"_6": 0}, {"_7": 0},
                {"_7": 48}, {"_16": -1}, {"_17": 0}, {"_18": 40}, {"_19": 48}, {"_20": 1 << 26}):
        assert call(**bad) == -1, bad
        assert b"bad sizes" in lib.tpo_last_error(), bad
    assert call(_0=1) == -2
    assert call(_5=0) == 0
    for at in (1, 2, 10, 11, 12, 13, 14, 15, 23):
        assert call(**{f"_{at}": None}) == -1 and b"NULL" in lib.tpo_last_error(), at
    for bad in ({"_1": P(4100)}, {"_10": P(4104)}, {"_8": 130}, {"_8": 0}, {"_9": 33}):
        assert call(**bad) == -1 and b"16 bytes" in lib.tpo_last_error(), bad
    size = lib.tpo_cache_attention_workspace_size
    need = size(0, 1, 1, 4, 2, 32, 64, 256)
    assert need > 0 and need % 256 == 0 and size(0, 1, 1, 4, 2, 32, 64, 2) == 0
    assert call(_4=1, _5=1, _20=256) == -4 and b"workspace" in lib.tpo_last_error()
    assert size(0, 1, 1, 3, 2, 32, 64, 4) == -1 and size(1, 1, 1, 4, 2, 32, 64, 4) == -1
    assert call(_4=1 << 24, _5=(1 << 29) - 1) == -1 and b"too many rows" in lib.tpo_last_error()


def test_attention_kernels_of_the_gpu_tests(lib):
    """Which kernel the sizes of tests/test_cached_attention_gpu.py take, so that no change of the
    rule leaves one of them without its tests."""
    from tests import test_cached_attention_gpu as t

    lib.tpo_cache_attention_rows.argtypes = [C] + [I] * 7

    def rows(dtype, new, lengths, Hq, Hk, size, page=64, more=0):
        return lib.tpo_cache_attention_rows(dtype, len(new), sum(new) + more, Hq, Hk, size, page,
                                            max(1, -(-max(lengths) // page)))

    for dtype in (0, 2, 3):
        prompt = 32 if dtype == 0 else 128  # float's products take too long
        for new, lengths, Hk, G in t.PROMPTS:
            assert rows(dtype, new, lengths, G * Hk, Hk, 72, more=7) == prompt
            assert rows(dtype, new, lengths, G * Hk, Hk, 64, more=7) == 32
        assert rows(dtype, t.MANY, [400], 32, 32, 65) == prompt
        for new, lengths in t.CASES:
            assert rows(dtype, new, lengths, 4, 2, 64) == 32
    assert rows(0, [4], [4], 3, 2, 16) == -1 and rows(1, [4], [4], 2, 2, 16) == -2
