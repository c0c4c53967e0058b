"""Derivatives that the operators do not have are refused, not left out of a result.

On meta tensors: autograd's side of a call is the same without a GPU.
"""
import pytest
import torch
import torch.autograd.forward_ad as fw


def _meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, device="meta", dtype=dtype)


def _calls(tpo):
    """Each operator as a function of its differentiable inputs, and these."""
    o = torch.empty(3, dtype=torch.int64, device="meta")
    idx, n = _meta(2, 5, 4, dtype=torch.int64), _meta(2, dtype=torch.int64)
    return {
        "layer_norm": (tpo.layer_norm, [_meta(6, 16), _meta(16), _meta(16)]),
        "packed_attention": (lambda q, k, v: tpo.packed_attention(q, k, v, o),
                             [_meta(6, 4, 16), _meta(6, 2, 16), _meta(6, 2, 16)]),
        "gated_projection": (tpo.gated_projection, [_meta(6, 16), _meta(24, 16), _meta(24, 16)]),
        "chamfer_distance": (lambda a, b: tpo.chamfer_distance(a, b)[0],
                             [_meta(2, 5, 3), _meta(2, 7, 3)]),
        "knn_gather": (lambda x: torch.ops.torch_point_ops_knn.knn_gather(x, idx, n),
                       [_meta(2, 7, 3)]),
        "gather_points": (lambda x: tpo.gather_points(x, _meta(2, 5, dtype=torch.int32)),
                          [_meta(2, 3, 7)]),
    }


NAMES = ["layer_norm", "packed_attention", "gated_projection", "chamfer_distance", "knn_gather",
         "gather_points"]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(tpo, name):
    f, inputs = _calls(tpo)[name]
    for at, x in enumerate(inputs):
        for grad in (False, True):
            with fw.dual_level():
                dual = [fw.make_dual(t.detach().requires_grad_(grad), torch.empty_like(t))
                        if i == at else t for i, t in enumerate(inputs)]
                with pytest.raises(RuntimeError, match="jvp is not implemented"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="jvp is not implemented"):
                    f(*dual)
                # a tensor without a tangent is none of forward mode's business
                assert f(*inputs) is not None
        with pytest.raises(RuntimeError, match="functorch transforms"):
            torch.func.jvp(lambda t: f(*inputs[:at], t, *inputs[at + 1:]), (x,),
                           (torch.empty_like(x),))


NN = NAMES[:3]


@pytest.mark.parametrize("name", NN)
def test_gradients_of_gradients_are_refused(tpo, name):
    f, inputs = _calls(tpo)[name]
    inputs = [t.requires_grad_(True) for t in inputs]
    y = f(*inputs)
    once = torch.autograd.grad(y.sum(), inputs, create_graph=True)
    assert [g.shape for g in once] == [t.shape for t in inputs]
    for g in once:
        # also where the loss has another way to the inputs
        for loss in (g.sum(), g.sum() + y.sum()):
            with pytest.raises(RuntimeError, match="_backward is not implemented"):
                torch.autograd.grad(loss, inputs, retain_graph=True, allow_unused=True)
    # a result that was only asked to keep its graph has its first derivative
    again = torch.autograd.grad(y.sum(), inputs, create_graph=True)
    assert [g.shape for g in again] == [t.shape for t in inputs]


@pytest.mark.parametrize("name", NN)
def test_inner_operators_have_no_derivative(tpo, name):
    """The operators that the autograd functions call, called alone."""
    f, inputs = _calls(tpo)[name]
    o = torch.empty(3, dtype=torch.int64, device="meta")
    more = {"layer_norm": (1e-5,), "packed_attention": (o, o, None, None, True, 1.0),
            "gated_projection": (0,)}[name]
    ns = {"layer_norm": "norm", "packed_attention": "attention", "gated_projection": "gated"}[name]
    op = getattr(getattr(torch.ops, f"torch_point_ops_{ns}"), f"{name}_forward")
    inputs = [t.requires_grad_(True) for t in inputs]
    with pytest.raises(RuntimeError, match="_forward is not implemented"):
        op(*inputs, *more)[0].sum().backward()
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward AD"):
        op(*[fw.make_dual(t.detach(), torch.empty_like(t)) for t in inputs], *more)
