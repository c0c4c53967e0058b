"""Attention over packed sequences of different lengths (no counterpart in the reference).

torch.ops.torch_point_ops_attention.packed_attention runs the gfx950 kernels of
libtpo_hip.so; its autograd is registered in C++ (nn_ops.cpp).
"""
import torch

from .. import _C  # noqa: F401


@torch.library.register_fake("torch_point_ops_attention::packed_attention")
def _packed_attention_fake(q, k, v, offsets_q, offsets_k, lengths_q, lengths_k, causal, scale):
    return torch.empty(q.shape, device=q.device, dtype=q.dtype)


@torch.library.register_fake("torch_point_ops_attention::packed_attention_forward")
def _packed_attention_forward_fake(q, k, v, offsets_q, offsets_k, lengths_q, lengths_k, causal,
                                   scale):
    out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    return (out, torch.empty(q.shape[1], q.shape[0], device=q.device, dtype=torch.float32),
            q.new_empty(0) if q.dtype == torch.float32 else torch.empty_like(out))


@torch.library.register_fake("torch_point_ops_attention::packed_attention_backward")
def _packed_attention_backward_fake(grad, q, k, v, out, lse, rest, offsets_q, offsets_k,
                                    lengths_q, lengths_k, causal, scale,
                                    mask=(True, True, True)):
    return tuple(torch.empty(t.shape if on else (0,), device=t.device, dtype=t.dtype)
                 for t, on in zip((q, k, v), mask))


def packed_attention(q, k, v, offsets_q, offsets_k=None, lengths_q=None, lengths_k=None,
                     causal=True, scale=None):
    """softmax(scale q k^T) v, sequence by sequence of a packed batch.

    Args:
      q (Tq, Hq, D), k and v (Tk, Hk, D), float32, float16 or bfloat16, D at most 128; Hq a
        multiple of Hk: query head h reads key head h // (Hq // Hk).  Rows and heads may be
        slices of a larger tensor (one projection of all three, say).
      offsets_q, offsets_k (B + 1) int64, not decreasing: sequence b has the rows
        offsets[b] .. offsets[b + 1].  offsets_k None: k and v are packed as q is, with the
        same lengths.
      lengths_q, lengths_k (B) int64 or None: how many rows of a sequence, from its first, are
        in use.  The others are not read: a padded batch, or a cache with room to grow.
      causal: a row sees the keys up to its own place, counted from the sequence's end, so
        that the last row sees every key (one new token over a cache, or a whole prompt).
      scale: None for D ** -0.5.

    Returns (Tq, Hq, D) of q's type; rows that are not in use or see no key are 0.
    Differentiable once, in reverse mode, in q, k and v, with sums in a fixed order; only the
    gradients that are asked for are computed (k's and v's by one kernel).  Scores, their
    statistics and all sums are float32; half and bfloat16 probabilities (and the scores'
    gradients, which float16 holds from 6e-8 on: scale the loss) are rounded to the type for
    the products.  Under torch.autocast q, k and v are taken in its
    type.
    """
    if offsets_k is None:
        if lengths_k is not None:
            raise ValueError("lengths_k needs offsets_k")
        offsets_k, lengths_k = offsets_q, lengths_q
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return torch.ops.torch_point_ops_attention.packed_attention(
        q, k, v, offsets_q, offsets_k, lengths_q, lengths_k, causal, scale)


from .attention import PackedAttention  # noqa: E402

__all__ = ["packed_attention", "PackedAttention"]
