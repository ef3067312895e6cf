"""Attention in one piece, and the paged cache that a model reads while decoding.  With the keyword arguments of the other operators
(`offset`, `approx_bwd`, `use_kernel`); the offset lies between 0.75 and 1.5.
"""
from . import _abi
from .block_ops import _flags
from .pam_ops import _require_kernel

__all__ = ["attention", "rotary_append", "cached_attention"]


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
    A query that sees no key has the result zero, and no gradient.  Weights below 2 ** -62 of the largest that came before them are none, and scores of 2 ** 127
    and more are no numbers.  The quotient is taken after the sum, and a power of two moves no result, so
    that softmax and bmm (which divide before it and subtract the largest score of all rows) give slightly different values."""
    _require_kernel(q, use_kernel)
    dim = q.shape[-1] if q.dim() else 0
    return _abi.host().attention(q, k, v, *_with_masks(_scoring("attention", dim, scale, window, cap), causal, prefix, documents, slopes), *_flags(offset, approx_bwd))


def rotary_append(q, k, v, cos, sin, cache_k, cache_v, pages, lengths, counts=None, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
                  offset=None, use_kernel=True):
    """The next tokens of every sequence into a paged cache: queries and keys are normed and rotated as `rotary` does it, keys and values
    written to their places in cache_k and cache_v, and the rotated queries returned.

    q [batch, tokens, heads, dim], k and v [batch, tokens, kv_heads, dim]; cache_k and cache_v [pages, page, kv_heads, dim], both of the same
    strides.  pages: int32 [batch, pages of a sequence], where the places 0 ... page - 1 of a sequence are, then the next ones.  lengths: int64 [batch],
    the tokens that are in the cache already (it is left as it is): token t goes to the place lengths + t and has that row of the tables.  counts:
    int64 [batch], how many of the tokens a sequence has; the others are padding: their queries are zeros, and nothing is written for them.
    A position outside the tables makes a head's rotated values NaN; a token whose place is not in the table of pages, or on a page that is not there,
    is not written.  No two tokens of a call may have one place.  There are no gradients."""
    _require_kernel(q, use_kernel)
    flags = _flags(offset, False)
    return _abi.host().rotary_append(q, k, v, cos, sin, cache_k, cache_v, pages, lengths, counts, q_weight, k_weight, bool(interleaved), float(eps), flags[0])


def cached_attention(q, cache_k, cache_v, pages, lengths, counts=None, *, scale=None, window=None, slopes=None, cap=None, offset=None, use_kernel=True):
    """`attention` of the next tokens of every sequence, q [batch, tokens, heads, dim], over a paged cache that has their keys and values already
    (see rotary_append, whose pages, lengths and counts these are): token t sees the places 0 ... lengths + t, or with a window the last of them.
    Made for one or a few tokens, and tables of up to 2 ** 30 places: the cache is read again for every
    twelve of tokens x heads / kv_heads (every four in heads that are no whole quads).  Weights below 2 ** -62 of the largest that came before them are none.  Padding's results are zeros.  A place that
    the table of pages does not have, or on a page that is not there, makes the results that see it NaN.  There are no gradients."""
    _require_kernel(q, use_kernel)
    scale, window, cap = _scoring("cached_attention", q.shape[-1] if q.dim() else 0, scale, window, cap)
    return _abi.host().cached_attention(q, cache_k, cache_v, pages, lengths, counts, scale, window, slopes, cap, _flags(offset, False)[0])


def _with_masks(scoring, causal, prefix, documents, slopes):
    scale, window, cap = scoring
    return scale, bool(causal), window, prefix, documents, slopes, cap
