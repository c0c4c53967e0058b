"""Layer norm over the last axis (no counterpart in the reference).

torch.ops.torch_point_ops_norm.layer_norm runs the gfx950 kernels of
libtpo_hip.so; its autograd is registered in C++ (nn_ops.cpp).
"""
import torch

from .. import _C  # noqa: F401


@torch.library.register_fake("torch_point_ops_norm::layer_norm")
def _layer_norm_fake(x, weight, bias, eps):
    return torch.empty(x.shape, device=x.device, dtype=x.dtype)


@torch.library.register_fake("torch_point_ops_norm::layer_norm_forward")
def _layer_norm_forward_fake(x, weight, bias, eps):
    rows = x.numel() // x.shape[-1]
    mean = torch.empty(rows, device=x.device, dtype=torch.float32)
    return torch.empty(x.shape, device=x.device, dtype=x.dtype), mean, torch.empty_like(mean)


@torch.library.register_fake("torch_point_ops_norm::layer_norm_backward")
def _layer_norm_backward_fake(grad, x, weight, bias, mean, rstd, eps, mask):
    gx = torch.empty(x.shape if mask[0] else (0,), device=x.device, dtype=x.dtype)
    gw, gb = (torch.empty(x.shape[-1], device=x.device, dtype=t.dtype)
              if on and t is not None else x.new_empty(0)
              for on, t in ((mask[1], weight), (mask[2], bias)))
    return gx, gw, gb


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x.

    Args: x (..., C) float32, float16 or bfloat16; weight, bias (C) of x's type
    or float32, or None; eps >= 0.  Sums are taken in float32 whatever x's type.
    Differentiable once, in reverse mode, in x, weight and bias; the weights' gradients
    are summed in a fixed order.  C is at most 2^20.  Returns a tensor of x's shape and type.
    """
    return torch.ops.torch_point_ops_norm.layer_norm(x, weight, bias, eps)


from .norm import LayerNorm  # noqa: E402

__all__ = ["layer_norm", "LayerNorm"]
