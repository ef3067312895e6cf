"""Attention in one piece, and the paged cache that a model reads while decoding.  With the keyword arguments of the other operators
(`offset`, `approx_bwd`, `use_kernel`); the offset lies between 0.75 and 1.5.
"""
from . import _abi
from .block_ops import _flags
from .pam_ops import _require_kernel

__all__ = ["attention"]


def _scoring(name, dim, scale, window, cap):
    """(scale, window, cap) as the host path takes them."""
    if window is not None and window < 1:
        raise ValueError(f"{name}: the window has at least one key, got {window}")
    if cap is not None and not cap > 0:
        raise ValueError(f"{name}: the cap is positive, got {cap}")
    scale = dim ** -0.5 if scale is None and dim > 0 else scale
    return float(scale if scale is not None else 1.0), int(window or 0), float(cap or 0.0)


def attention(q, k, v, *, scale=None, causal=True, window=None, prefix=None, documents=None, slopes=None, cap=None, offset=None,
              approx_bwd=False, use_kernel=True):
    """Queries [batch, tokens, heads, dim] over keys and values [batch, keys, kv_heads, dim] (any strides but the last; heads / kv_heads
    queries' heads share a key's; dim up to 256), with gradients for the three.  The queries are those of the last `tokens` of the `keys` tokens.

        a = sum over d of (q_d (*) scale) (*) k_d        scale: dim ** -0.5
        a = cap (*) tanh(a (/) cap)                      with a cap; tanh u = (1 - w) (/) (1 + w), w = 2 ** -(u (*) 2 log2 e)
        a = a - slopes[head] (*) |i - j|                 with slopes, float32 [heads]
        e_ij = exp(a),  l_i = sum of e_ij,  y_id = (sum of e_ij (*) v_jd) (/) l_i

    over the keys j that query i sees:
      causal      j <= i
      window      |i - j| < window
      prefix      int64 [batch]: the first keys of a batch entry, which every query sees besides
      documents   int64 [batch, keys]: only keys of the query's own document; a negative number is padding's
    A query that sees no key has the result zero, and no gradient.  The quotient is taken after the sum, and a power of two moves no result, so
    that softmax and bmm (which divide before it and subtract the largest score of all rows) give slightly different values."""
    _require_kernel(q, use_kernel)
    dim = q.shape[-1] if q.dim() else 0
    return _abi.host().attention(q, k, v, *_with_masks(_scoring("attention", dim, scale, window, cap), causal, prefix, documents, slopes), *_flags(offset, approx_bwd))


def _with_masks(scoring, causal, prefix, documents, slopes):
    scale, window, cap = scoring
    return scale, bool(causal), window, prefix, documents, slopes, cap
