"""Gated projection of a feed-forward block (no counterpart in the reference).

torch.ops.torch_point_ops_gated.gated_projection runs the gfx950 kernels of
libtpo_hip.so; its autograd is registered in C++ (nn_ops.cpp).
"""
import torch

from .. import _C  # noqa: F401

# codes of include/tpo.h
_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}


@torch.library.register_fake("torch_point_ops_gated::gated_projection")
def _gated_projection_fake(x, w_gate, w_up, activation):
    return torch.empty(*x.shape[:-1], w_gate.shape[0], device=x.device, dtype=x.dtype)


@torch.library.register_fake("torch_point_ops_gated::gated_projection_forward")
def _gated_projection_forward_fake(x, w_gate, w_up, activation):
    rows = x.numel() // x.shape[-1]
    return (torch.empty(*x.shape[:-1], w_gate.shape[0], device=x.device, dtype=x.dtype),
            x.new_empty(rows, 2 * w_gate.shape[0]) if x.dtype == torch.float32
            else x.new_empty(0))


@torch.library.register_fake("torch_point_ops_gated::gated_projection_backward")
def _gated_projection_backward_fake(grad, x, w_gate, w_up, kept, activation, mask):
    gx = torch.empty(x.shape if mask[0] else (0,), device=x.device, dtype=x.dtype)
    gg, gu = (torch.empty(w_gate.shape if mask[1] else (0,), device=x.device, dtype=x.dtype)
              for _ in range(2))
    return gx, gg, gu


def gated_projection(x, w_gate, w_up, activation="silu"):
    """act(x @ w_gate.T) * (x @ w_up.T) in one kernel.

    Args: x (..., K), w_gate and w_up (F, K), float32, float16 or bfloat16; activation
    "silu", "gelu" (x times the normal distribution function), "relu" or "sigmoid".
    Differentiable once, in reverse mode, in x and the weights.  A float32 forward keeps the two projections for
    the backward; for the half types the backward computes them again, which takes less
    time than unrounded ones take through memory, and rounds the gradients at them to x's
    type between the products.  All sums are float32.  Under torch.autocast the inputs
    are taken in its type, as a linear layer's are.  Returns (..., F).
    """
    code = _ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(
            f"activation must be one of {sorted(_ACTIVATIONS)}, but got {activation!r}")
    return torch.ops.torch_point_ops_gated.gated_projection(x, w_gate, w_up, code)


from .gated import GatedFeedForward  # noqa: E402

__all__ = ["gated_projection", "GatedFeedForward"]
