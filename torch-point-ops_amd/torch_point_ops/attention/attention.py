"""Packed attention module (no counterpart in the reference)."""
import torch

from . import packed_attention


class PackedAttention(torch.nn.Module):
    """forward(q, k, v, offsets_q, offsets_k=None, lengths_q=None, lengths_k=None)."""

    def __init__(self, causal=True, scale=None):
        super().__init__()
        self.causal = causal
        self.scale = scale

    def forward(self, q, k, v, offsets_q, offsets_k=None, lengths_q=None, lengths_k=None):
        return packed_attention(q, k, v, offsets_q, offsets_k, lengths_q, lengths_k,
                                self.causal, self.scale)
