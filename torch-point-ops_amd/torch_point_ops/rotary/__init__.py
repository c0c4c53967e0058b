"""Rotary positions (no counterpart in the reference).

torch.ops.torch_point_ops_rotary.rotary_positions runs the gfx950 kernels of
libtpo_hip.so; its autograd is registered in C++ (cache_ops.cpp).
"""
import math

import torch

from .. import _C  # noqa: F401


@torch.library.register_fake("torch_point_ops_rotary::rotary_positions")
def _rotary_positions_fake(x, positions, frequencies, interleaved, amplitude):
    return torch.empty(x.shape, device=x.device, dtype=x.dtype)


@torch.library.register_fake("torch_point_ops_rotary::rotary_positions_backward")
def _rotary_positions_backward_fake(grad, positions, frequencies, interleaved, amplitude):
    return torch.empty(grad.shape, device=grad.device, dtype=grad.dtype)


def rotary_frequencies(pairs, base=10000.0, stretch=1.0, trained=None, device=None):
    """The frequencies base ** (-j / pairs) of the pairs j, as rotary_positions takes them.

    stretch > 1 makes room for sequences that many times longer than the trained ones: every
    frequency is divided by it or, where the `trained` length is given, those that turn less than
    once over it are, those that turn 32 times or more stay as they are, and those between go
    from one to the other linearly in their turns.
    """
    if pairs < 0 or base <= 0 or stretch <= 0:
        raise ValueError(f"pairs must not be negative, base and stretch must be positive, but got "
                         f"{pairs}, {base} and {stretch}")
    f = float(base) ** (-torch.arange(pairs, dtype=torch.float64, device=device) / max(pairs, 1))
    if trained is None:
        return f / stretch
    kept = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return f * kept + f / stretch * (1 - kept)


def rotary_positions(x, positions, frequencies, interleaved=False, amplitude=1.0):
    """Queries or keys, each head's first 2 P values turned in pairs by position * frequency.

    Args:
      x (T, H, D) float32, float16 or bfloat16, D at most 512; tokens and heads may be a slice of
        a larger tensor (queries and keys of one projection, say).
      positions (T) or (T, A), int64 or float32: a token's place, or its coordinates: the P
        pairs are shared out evenly among the A axes, the first P / A to the first.
      frequencies (P) float64: angles are taken in 64 bits, whatever x's type.
      interleaved: pair j is values 2 j and 2 j + 1, else values j and j + P.
      amplitude: what the turned values are multiplied by.

    y1 = x1 cos a - x2 sin a, y2 = x2 cos a + x1 sin a.  Values from 2 P on stay as they are.
    Returns (T, H, D) of x's type.  Differentiable once, in reverse mode, in x.
    """
    return torch.ops.torch_point_ops_rotary.rotary_positions(x, positions, frequencies,
                                                             interleaved, amplitude)


from .rotary import RotaryPositions  # noqa: E402

__all__ = ["rotary_positions", "rotary_frequencies", "RotaryPositions"]
