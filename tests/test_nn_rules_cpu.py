"""What the transformer operators' rules choose, read from their workspaces and queries."""
import ctypes

import pytest

I = ctypes.c_int64


@pytest.fixture(scope="module")
def lib(tpo):
    from torch_point_ops import _native

    L = ctypes.CDLL(_native.HIP_LIB)
    L.tpo_layer_norm_bwd_workspace_size.argtypes = [I, I]
    L.tpo_layer_norm_bwd_workspace_size.restype = I
    return L


def _shares(lib, rows, width):
    """Workgroups of the layer norm's backward: each leaves 2 width floats."""
    return lib.tpo_layer_norm_bwd_workspace_size(rows, width) // (8 * width)


@pytest.mark.parametrize("width", [1100, 2048, 4096, 8192, 16384])
def test_wide_rows_have_a_workgroup_each(lib, width):
    for rows in (1, 4, 16, 64, 128):
        assert _shares(lib, rows, width) == rows
    for rows in (200, 500, 1000):
        assert _shares(lib, rows, width) >= rows // 2 if rows < 512 else 256


@pytest.mark.parametrize("width", [96, 512, 700, 1024])
def test_narrow_rows_have_a_wave_each(lib, width):
    for rows in (1, 5, 64, 500, 1000):
        assert _shares(lib, rows, width) == (rows + 3) // 4


@pytest.mark.parametrize("width", [1, 8, 96, 1000, 3000, 8192, 16384, 20000, 1 << 20])
def test_shares_stay_small_beside_many_rows(lib, width):
    for rows in (8192, 32768, 1 << 20, (1 << 31) - 1):
        assert 1 <= _shares(lib, rows, width) <= min(1024, rows // 8)
