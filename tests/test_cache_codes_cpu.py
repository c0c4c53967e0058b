"""How a key turned in 64 bits becomes a float that has its code: on the host, from the kernels'
own header, against the definition in tests/cache64.py."""
import ctypes
import itertools
import math

import numpy as np
import pytest
import torch

from tests import cache64
from tests.cache_host import library

SOURCE = """
#include "cache_codes.hpp"
extern "C" void odd(const double* d, float* f, int64_t n) {
  for (int64_t i = 0; i < n; ++i) f[i] = tpo::to_odd(d[i]);
}
extern "C" int exponent(float top) { return tpo::exponent_for(top); }
"""
MOST, LEAST = float(np.finfo(np.float32).max), 2.0 ** -149


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    lib = library(SOURCE, tmp_path_factory.mktemp("codes"))
    lib.exponent.argtypes = [ctypes.c_float]
    return lib


def _odd(host, d):
    d = np.ascontiguousarray(d, dtype=np.float64)
    f = np.empty(d.shape, np.float32)
    host.odd(d.ctypes.data_as(ctypes.c_void_p), f.ctypes.data_as(ctypes.c_void_p),
             ctypes.c_int64(d.size))
    return f


def _values():
    """Magnitudes about every border: nothing, floats' least, normal, codes' and the largest."""
    v = [0.0, 5e-324, 1e-320, 1e-300, 1e-60, 1e-50, 1e-46, 7e-46, 1e-40, 1.4e-45, 1e-38, MOST]
    v += [m * 2.0 ** e for e in range(-160, 127) for m in (1.0, 1.25, 1 + 2.0 ** -30, 2 - 2.0 ** -40,
                                                           1.0625, 1.0625 + 2.0 ** -45)]
    return np.array([s * x for x in v for s in (1, -1)])


def test_rounding_to_odd(host):
    """The float towards zero, its last bit set where that is not the value itself."""
    d = _values()
    f = _odd(host, d)
    assert np.isfinite(f).all()
    assert (np.signbit(f) == np.signbit(d)).all()
    near = d.astype(np.float32)
    down = np.where(np.abs(near.astype(np.float64)) > np.abs(d),
                    np.nextafter(near, np.float32(0)), near)
    bits = np.where(down.astype(np.float64) == d, 0, 1) | down.view(np.int32)
    assert (f.view(np.int32) == bits).all(), d[f.view(np.int32) != bits]
    none = _odd(host, [math.nan, math.inf, -math.inf])
    assert np.isnan(none[0]) and none[1] == math.inf and none[2] == -math.inf


def test_codes_are_those_of_the_double(host):
    """Two roundings, to odd and to the code, are one; also where the scale's exponent is at its
    ends."""
    d = _values()
    f = torch.from_numpy(_odd(host, d)).double()
    d = torch.from_numpy(d)
    for e in (-40, -3, 0, 17, 40):
        assert torch.equal(cache64.to_code(f / 2.0 ** e), cache64.to_code(d / 2.0 ** e))


def test_exponents(host):
    for m, e in itertools.product((1.0, 1.75, 1.75 + 2.0 ** -23, 2 - 2.0 ** -23), range(-149, 128)):
        top = float(np.float32(m * 2.0 ** e))
        assert host.exponent(top) == cache64.exponent(top), top
    assert host.exponent(0.0) == -40 and host.exponent(MOST) == 40


def test_beyond_the_largest_float(host):
    """A finite value is never taken for one that is not: the largest float, which is odd."""
    d = np.array([s * x for x in (MOST * (1 + 2.0 ** -26), MOST * 1.0001, 4.2e38, 2.0 ** 128, 1e300)
                  for s in (1, -1)])
    assert (_odd(host, d) == np.sign(d) * MOST).all()
