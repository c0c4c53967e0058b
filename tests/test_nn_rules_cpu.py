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


def test_attention_backward_of_some(tpo, lib):
    """dK and dV go together and alone take the workspace; each operator result can be left out."""
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode

    P, C, D = ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    lib.tpo_last_error.restype = ctypes.c_char_p
    lib.tpo_attention_bwd.argtypes = [C] + [P] * 11 + [I] * 12 + [C, D, P, P, P, P, I, P]
    f = P(4096)  # never dereferenced

    def call(gq, gk, gv, rows=4, ws=None):
        return lib.tpo_attention_bwd(0, f, f, f, f, f, f, f, f, f, None, None, 1, rows, rows, 2, 2,
                                     16, *[32, 16] * 3, 1, 1.0, gq, gk, gv, ws, 0, None)

    for gk, gv in ((f, None), (None, f)):
        assert call(f, gk, gv) == -1 and b"go together" in lib.tpo_last_error()
    assert call(None, f, f) == -4
    assert call(None, None, None) == 0
    assert call(f, None, None, rows=0) == 0
    with FakeTensorMode():
        q, k, o = torch.empty(7, 4, 32), torch.empty(9, 2, 32), torch.empty(3, dtype=torch.int64)
        lse = torch.empty(4, 7)
        for mask in ([True, False, False], [False, True, False], [False, False, True]):
            g = torch.ops.torch_point_ops_attention.packed_attention_backward(
                q, q, k, k, q, lse, torch.empty(0), o, o, None, None, True, 1.0, mask)
            assert [t.shape for t in g] == [t.shape if on else (0,)
                                            for t, on in zip((q, k, k), mask)]


def test_attention_kernels_of_the_gpu_tests(tpo, lib):
    """Which kernel the sizes of tests/test_attention_more_gpu.py take, so that no change of
    the rule leaves one of them without its tests."""
    from tests import test_attention_more_gpu as t

    lib.tpo_attention_fwd_rows.argtypes = [ctypes.c_int] + [I] * 6

    def rows(dtype, lens_q, lens_k, Hq, Hk, D, more=(0, 0)):
        return lib.tpo_attention_fwd_rows(dtype, len(lens_q), sum(lens_q) + more[0],
                                          sum(lens_k) + more[1], Hq, Hk, D)

    for dtype in (0, 2, 3):
        for Hq, Hk in t.PROMPT_HEADS:
            for D in (40, 64, 128):
                assert rows(dtype, t.PROMPT, t.PROMPT, Hq, Hk, D) == 128
            assert rows(dtype, t.ROOMS_Q, t.ROOMS_K, Hq, Hk, 32, (10, 7)) == 128
        assert [rows(dtype, lens, lens, Hq, Hk, D) for lens, Hq, Hk, D in t.SCALED] == [32, 32, 128]
        for B in (61, 62, 63, 64, 65):
            for lens in (t._mixed(B, 40), t._mixed(B, 150)):
                many = lens == t._mixed(B, 150)
                assert rows(dtype, lens, lens, *((16, 8) if many else (4, 2)), 32,
                            (3, 3)) == (128 if many else 32)
    assert rows(0, [4], [4], 3, 2, 16) == -1 and rows(1, [4], [4], 2, 2, 16) == -2


def test_launches_stay_below_their_threads(lib):
    """A launch has fewer than 2^32 threads along an axis: more rows are an error of the call."""
    P, C, D = ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    lib.tpo_last_error.restype = ctypes.c_char_p
    lib.tpo_attention_fwd.argtypes = [C] + [P] * 7 + [I] * 12 + [C, D, P, P, P, P, I, P]
    lib.tpo_attention_bwd.argtypes = [C] + [P] * 11 + [I] * 12 + [C, D, P, P, P, P, I, P]
    f = P(4096)  # never dereferenced
    B, T, H = 1 << 20, 1 << 20, 16
    assert lib.tpo_attention_fwd_rows(2, B, T, T, H, H, 16) == 128
    assert lib.tpo_attention_fwd(2, f, f, f, f, f, None, None, B, T, T, H, H, 16, *[256, 16] * 3, 1,
                                 1.0, f, None, None, None, 0, None) == -1
    assert b"too many rows" in lib.tpo_last_error()
    T = 1 << 26
    assert lib.tpo_attention_bwd(2, f, f, f, f, f, None, f, f, f, None, None, 1, T, 64, H, H, 16,
                                 *[256, 16] * 3, 1, 1.0, f, None, None, None, 0, None) == -1
    assert b"too many rows" in lib.tpo_last_error()


def test_missing_arrays_are_refused(lib):
    """A NULL for an array that a call would read or write is an error of the call."""
    P, C, D = ctypes.c_void_p, ctypes.c_int, ctypes.c_double
    lib.tpo_last_error.restype = ctypes.c_char_p
    lib.tpo_layer_norm_fwd.argtypes = [C, C, P, P, P, I, I, D, P, P, P, P]
    lib.tpo_layer_norm_bwd.argtypes = [C, C, P, P, P, P, P, I, I, D, P, P, P, P, I, P]
    lib.tpo_attention_fwd.argtypes = [C] + [P] * 7 + [I] * 12 + [C, D, P, P, P, P, I, P]
    lib.tpo_attention_bwd.argtypes = [C] + [P] * 11 + [I] * 12 + [C, D, P, P, P, P, I, P]
    lib.tpo_gated_fwd.argtypes = [C, P, P, P, I, I, I, C, P, P, P, I, P]
    lib.tpo_gated_bwd.argtypes = [C, P, P, P, P, P, I, I, I, C, P, P, P, P, I, P]
    f = P(4096)  # never dereferenced
    sizes = [1, 4, 4, 2, 2, 16, *[32, 16] * 3, 1, 1.0]

    def refused(entry, args, needed):
        for at in needed:
            a = list(args)
            a[at] = None
            assert entry(*a) == -1, at
            assert b"NULL" in lib.tpo_last_error()

    refused(lib.tpo_layer_norm_fwd, [0, 0, f, f, f, 4, 8, 1e-5, f, None, None, None], (2, 8))
    refused(lib.tpo_layer_norm_bwd,
            [0, 0, f, f, f, f, f, 4, 8, 1e-5, f, None, None, None, 0, None], (2, 3, 5, 6))
    refused(lib.tpo_attention_fwd,
            [0, f, f, f, f, f, None, None, *sizes, f, None, None, None, 0, None], (1, 2, 3, 4, 5, 22))
    refused(lib.tpo_attention_bwd,
            [0, f, f, f, f, f, f, f, f, f, None, None, *sizes, f, None, None, None, 0, None],
            (1, 2, 3, 4, 5, 7, 8, 9))
    refused(lib.tpo_gated_fwd, [0, f, f, f, 4, 8, 8, 0, f, None, None, 0, None], (1, 2, 3, 8))
    refused(lib.tpo_gated_bwd, [0, f, f, f, f, None, 4, 8, 8, 0, f, f, f, f, 1 << 30, None],
            (1, 2, 3, 4))
