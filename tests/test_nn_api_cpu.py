"""The transformer operators without a GPU: fake shapes (what torch.compile traces), the CPU's
answer, Python's refusals, and the C entries' checks of their arguments."""
import ctypes

import pytest
import torch

P, I, D, C = ctypes.c_void_p, ctypes.c_int64, ctypes.c_double, ctypes.c_int


@pytest.fixture(scope="module")
def lib(tpo):
    from torch_point_ops import _native

    L = ctypes.CDLL(_native.HIP_LIB)
    L.tpo_last_error.restype = ctypes.c_char_p
    L.tpo_layer_norm_fwd.argtypes = [C, C, P, P, P, I, I, D, P, P, P, P]
    L.tpo_layer_norm_bwd.argtypes = [C, C, P, P, P, P, P, I, I, D, P, P, P, P, I, P]
    L.tpo_attention_fwd.argtypes = [C] + [P] * 7 + [I] * 12 + [C, D, P, P, P, P, I, P]
    L.tpo_attention_bwd.argtypes = [C] + [P] * 11 + [I] * 12 + [C, D, P, P, P, P, I, P]
    L.tpo_gated_fwd.argtypes = [C, P, P, P, I, I, I, C, P, P, P, I, P]
    L.tpo_gated_bwd.argtypes = [C, P, P, P, P, P, I, I, I, C, P, P, P, P, I, P]
    L.tpo_layer_norm_bwd_workspace_size.argtypes = [I, I]
    for n in ("attention_fwd", "attention_bwd"):
        getattr(L, f"tpo_{n}_workspace_size").argtypes = [C] + [I] * 6
    for n in ("gated_fwd", "gated_bwd"):
        getattr(L, f"tpo_{n}_workspace_size").argtypes = [C] + [I] * 3
    for n in ("layer_norm_bwd", "attention_fwd", "attention_bwd", "gated_fwd", "gated_bwd"):
        getattr(L, f"tpo_{n}_workspace_size").restype = I
    return L


def test_fake_shapes(tpo):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w = torch.empty(2, 5, 16, dtype=torch.bfloat16), torch.empty(16)
        assert tpo.layer_norm(x, w).shape == x.shape and tpo.layer_norm(x).dtype == x.dtype
        y, m, r = torch.ops.torch_point_ops_norm.layer_norm_forward(x, w, None, 1e-5)
        assert m.shape == r.shape == (10,) and m.dtype == torch.float32
        g = torch.ops.torch_point_ops_norm.layer_norm_backward(y, x, w, None, m, r, 1e-5,
                                                               [True, True, True])
        assert [t.shape for t in g] == [(2, 5, 16), (16,), (0,)] and g[1].dtype == torch.float32
        q, k = torch.empty(7, 4, 32), torch.empty(9, 2, 32)
        o = torch.empty(3, dtype=torch.int64)
        assert tpo.packed_attention(q, k, k, o, o).shape == q.shape
        out, lse, rest = torch.ops.torch_point_ops_attention.packed_attention_forward(
            q, k, k, o, o, None, None, True, 1.0)
        assert lse.shape == (4, 7)
        g = torch.ops.torch_point_ops_attention.packed_attention_backward(
            out, q, k, k, out, lse, rest, o, o, None, None, True, 1.0)
        assert [t.shape for t in g] == [q.shape, k.shape, k.shape]
        x, w = torch.empty(3, 4, 16), torch.empty(24, 16)
        h = tpo.gated_projection(x, w, w)
        assert h.shape == (3, 4, 24)
        g = torch.ops.torch_point_ops_gated.gated_projection_backward(
            h, x, w, w, torch.empty(0), 0, [True, False])
        assert [t.shape for t in g] == [x.shape, (0,), (0,)]


def test_cpu_tensors_are_refused(tpo):
    x, o = torch.ones(4, 8), torch.tensor([0, 4])
    for t in (x, x.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="layer_norm is not implemented for CPU"):
            tpo.layer_norm(t)
        with pytest.raises(RuntimeError, match="gated_projection is not implemented for CPU"):
            tpo.gated_projection(t, x, x)
        with pytest.raises(RuntimeError, match="packed_attention is not implemented for CPU"):
            tpo.packed_attention(t.view(4, 1, 8), x.view(4, 1, 8), x.view(4, 1, 8), o)


def test_python_refusals(tpo):
    x, o = torch.ones(4, 1, 8), torch.tensor([0, 4])
    with pytest.raises(ValueError, match="activation must be one of"):
        tpo.gated_projection(x, x, x, activation="tanh")
    with pytest.raises(ValueError, match="activation must be one of"):
        tpo.GatedFeedForward(8, 16, activation=None)
    with pytest.raises(ValueError, match="width must be positive"):
        tpo.LayerNorm(0)
    with pytest.raises(ValueError, match="lengths_k needs offsets_k"):
        tpo.packed_attention(x, x, x, o, lengths_k=o[1:])


def test_modules_hold_what_they_train(tpo):
    assert [n for n, _ in tpo.LayerNorm(6).named_parameters()] == ["weight", "bias"]
    assert [n for n, _ in tpo.LayerNorm(6, bias=False).named_parameters()] == ["weight"]
    shapes = {n: tuple(p.shape) for n, p in tpo.GatedFeedForward(6, 10).named_parameters()}
    assert shapes == {"gate.weight": (10, 6), "up.weight": (10, 6), "down.weight": (6, 10)}
    assert tpo.PackedAttention(causal=False, scale=0.5).scale == 0.5


def test_layer_norm_entry(lib):
    f = P(4096)  # never dereferenced: the calls fail their checks first
    assert lib.tpo_layer_norm_fwd(0, 0, f, f, f, -1, 8, 1e-5, f, None, None, None) == -1
    assert lib.tpo_layer_norm_fwd(0, 0, f, f, f, 4, 0, 1e-5, f, None, None, None) == -1
    assert b"bad sizes" in lib.tpo_last_error()
    assert lib.tpo_layer_norm_fwd(0, 0, f, f, f, 4, 8, 1e-5, f, f, None, None) == -1
    assert lib.tpo_layer_norm_fwd(1, 1, f, f, f, 4, 8, 1e-5, f, None, None, None) == -2
    assert lib.tpo_layer_norm_fwd(3, 2, f, f, f, 4, 8, 1e-5, f, None, None, None) == -2
    assert lib.tpo_layer_norm_fwd(3, 0, f, f, f, 0, 8, 1e-5, f, None, None, None) == 0  # no rows
    assert lib.tpo_layer_norm_bwd(0, 0, f, f, f, f, f, 4, 8, 1e-5, f, f, f, None, 0, None) == -4
    assert b"workspace" in lib.tpo_last_error()
    assert lib.tpo_layer_norm_bwd_workspace_size(-1, 8) == -1
    need = lib.tpo_layer_norm_bwd_workspace_size(32768, 1024)
    assert 0 < need < 32 << 20 and need % 256 == 0


def _attention(lib, dtype=0, B=1, Tq=4, Tk=4, Hq=2, Hk=2, D=16):
    f = P(4096)
    return lib.tpo_attention_fwd(dtype, f, f, f, f, f, None, None, B, Tq, Tk, Hq, Hk, D,
                                 *[Hq * D, D] * 3, 1, 1.0, f, None, None, None, 0, None)


def test_attention_entry(lib):
    for bad in ({"B": -1}, {"Tq": -1}, {"Tk": 1 << 31}, {"Hq": 3}, {"Hq": 0}, {"Hk": 0}, {"D": 0},
                {"D": 129}):
        assert _attention(lib, **bad) == -1, bad
        assert b"bad sizes" in lib.tpo_last_error()
    assert _attention(lib, dtype=1) == -2
    assert _attention(lib, Tq=0) == 0
    f = P(4096)
    assert lib.tpo_attention_bwd(0, f, f, f, f, f, f, f, f, f, None, None, 1, 4, 4, 2, 2, 16,
                                 *[32, 16] * 3, 1, 1.0, f, f, f, None, 0, None) == -4
    assert lib.tpo_attention_fwd_workspace_size(0, 1, 4, 4, 3, 2, 16) == -1
    assert lib.tpo_attention_bwd_workspace_size(3, 1, 4, 4, 2, 2, 200) == -1


def test_gated_entry(lib):
    f = P(4096)
    for M, K, F in ((-1, 8, 8), (4, 0, 8), (4, 8, -1), (1 << 40, 8, 8)):
        assert lib.tpo_gated_fwd(0, f, f, f, M, K, F, 0, f, None, None, 0, None) == -1
    assert lib.tpo_gated_fwd(0, f, f, f, 4, 8, 8, 4, f, None, None, 0, None) == -1
    assert b"activation" in lib.tpo_last_error()
    assert lib.tpo_gated_fwd(1, f, f, f, 4, 8, 8, 0, f, None, None, 0, None) == -2
    assert lib.tpo_gated_fwd(3, f, f, f, 0, 8, 8, 0, f, None, None, 0, None) == 0
    assert lib.tpo_gated_bwd(3, f, f, f, f, None, 4, 8, 8, 0, f, f, f, None, 0, None) == -4
    assert lib.tpo_gated_fwd(3, f, f, f, 4, 8, 8, 0, f, f, None, 0, None) == -1  # halves: not kept
    assert lib.tpo_gated_bwd(3, f, f, f, f, f, 4, 8, 8, 0, f, f, f, f, 1 << 20, None) == -1
    assert lib.tpo_gated_bwd_workspace_size(3, -1, 8, 8) == -1
