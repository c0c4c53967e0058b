"""Layer norm module (no counterpart in the reference)."""
import torch

from . import layer_norm


class LayerNorm(torch.nn.Module):
    """forward(x (..., width)) -> normalised x, with a learned weight and bias."""

    def __init__(self, width, eps=1e-5, bias=True, device=None, dtype=None):
        super().__init__()
        if width <= 0:
            raise ValueError(f"width must be positive, but got {width}")
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = (torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype))
                     if bias else None)

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
