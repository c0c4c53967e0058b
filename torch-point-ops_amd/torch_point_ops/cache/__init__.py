"""A cache of keys and values in pages of 8 bits (no counterpart in the reference).

torch.ops.torch_point_ops_cache.append and .attention run the gfx950 kernels of
libtpo_hip.so (registered in cache_ops.cpp).  Neither has a derivative.
"""
import torch

from .. import _C  # noqa: F401


@torch.library.register_fake("torch_point_ops_cache::append")
def _append_fake(k, v, keys, values, key_scales, value_scales, table, lengths, offsets,
                 lengths_new, q, positions, frequencies, interleaved, amplitude):
    return k.new_empty(0) if q is None else torch.empty(q.shape, device=q.device, dtype=q.dtype)


@torch.library.register_fake("torch_point_ops_cache::attention")
def _attention_fake(q, keys, values, key_scales, value_scales, table, lengths, offsets, lengths_q,
                    causal, scale):
    return torch.empty(q.shape, device=q.device, dtype=q.dtype)


from .cache import PagedCache  # noqa: E402


def cache_append(cache, k, v, offsets, q=None, frequencies=None, positions=None,
                 interleaved=False, amplitude=1.0, lengths_new=None):
    """Puts the keys and values of new tokens into a PagedCache, keys turned on the way.

    Args:
      cache: a PagedCache whose lengths count the new tokens already.
      k, v (T, Hk, D) float32, float16 or bfloat16: rows offsets[b] .. offsets[b + 1] are the
        last tokens of sequence b.  Rows and heads may be slices of one projection.
      offsets (B + 1) int64, not decreasing; lengths_new (B) int64 or None: how many of a
        sequence's rows, from its first, are new tokens (a padded batch).
      q (T, Hq, D) of k's type, or None: queries, turned as the keys are.
      frequencies (P) float64 or None (nothing is turned), positions, interleaved, amplitude:
        as rotary_positions takes them; positions None: the tokens' places in their sequences.

    Keys are turned in 64 bits and rounded once.  A page and head has one scale for its keys and
    one for its values, powers of two; it grows where a new token needs it, and the page's older
    codes are rounded to it.  Values that are not finite are kept as NaN.  A page that is
    written to belongs to one sequence; pages that are only read may belong to several.
    Changes the cache in place, and nothing but the new tokens' places and pages in it.
    Returns q turned (rows that are not new tokens 0), or None.
    """
    out = torch.ops.torch_point_ops_cache.append(
        k, v, cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.table,
        cache.lengths, offsets, lengths_new, q, positions, frequencies, interleaved, amplitude)
    return None if q is None else out


def cached_attention(q, cache, offsets, lengths_q=None, causal=True, scale=None):
    """softmax(scale q k^T) v of new tokens over a PagedCache, sequence by sequence.

    Args:
      q (T, Hq, D) float32, float16 or bfloat16, Hq a multiple of the cache's heads: rows
        offsets[b] .. offsets[b + 1] are the last tokens of sequence b.
      cache: a PagedCache that holds the new tokens.
      offsets (B + 1) int64; lengths_q (B) int64 or None: as packed_attention takes them.
      causal: a row sees the tokens up to its own; without it, all of its sequence.
      scale: None for D ** -0.5.

    Returns (T, Hq, D) of q's type; rows that are not in use or see no key are 0.  Scores, their
    statistics and all sums are float32; half and bfloat16 probabilities are rounded to the type
    for the product, half ones by 2^-11 of themselves and 2^-24 of their sum, however far apart
    the scales of pages that cache_append wrote.  Under torch.autocast q is taken in its type.
    Without a derivative.
    """
    if scale is None:
        scale = q.shape[-1] ** -0.5
    return torch.ops.torch_point_ops_cache.attention(
        q, cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.table,
        cache.lengths, offsets, lengths_q, causal, scale)


__all__ = ["PagedCache", "cache_append", "cached_attention"]
