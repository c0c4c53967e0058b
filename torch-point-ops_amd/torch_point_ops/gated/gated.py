"""Gated feed-forward module (no counterpart in the reference)."""
import torch

from . import _ACTIVATIONS, gated_projection


class GatedFeedForward(torch.nn.Module):
    """forward(x (..., width)) -> (act(gate x) * (up x)) projected back to width."""

    def __init__(self, width, hidden, activation="silu", device=None, dtype=None):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(
                f"activation must be one of {sorted(_ACTIVATIONS)}, but got {activation!r}")
        self.activation = activation
        kw = {"bias": False, "device": device, "dtype": dtype}
        self.gate = torch.nn.Linear(width, hidden, **kw)
        self.up = torch.nn.Linear(width, hidden, **kw)
        self.down = torch.nn.Linear(hidden, width, **kw)

    def forward(self, x):
        return self.down(gated_projection(x, self.gate.weight, self.up.weight, self.activation))
