"""The operators of a decoder block beside the reference's library: a product with an activation and a residual, the gated layer,
the rotation of queries and keys.  Each is a composition of the primitives in one or two kernels, with their keyword arguments
(`offset`, `approx_bwd`, `use_kernel`) and their gradients.
"""
import math

import torch

from . import _abi
from .cuda_bindings import _both, _is_tracing, _offset_value
from .pam_ops import _require_kernel

__all__ = ["linear_act", "gated_linear", "rotary", "rotary_tables"]

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _activation(name):
    if name not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(map(repr, _ACTIVATIONS))}")
    return _ACTIVATIONS[name]


def _flags(offset, approx_bwd):
    """(offset, approximate for the first operands, for the second, for exp and log); a pair counts as set for the last."""
    if _is_tracing():
        raise RuntimeError("this operator is not recorded by torch.jit.trace")
    a, b = _both(approx_bwd)
    return float(_offset_value(offset)), bool(a), bool(b), bool(approx_bwd)


def linear_act(X, W, bias=None, activation=None, residual=None, *, offset=None, approx_bwd=False, use_kernel=True):
    """activation(X W^T + bias) + residual in one product, X [..., d_in], W [d_out, d_in], residual of the result's shape.

    activation: None, "relu", "silu" (x over 1 + exp(-x), one quotient) or "gelu" (x over 1 + exp(-1.702 x)).  The sigmoid's
    exponent is held below 64, so that no x overflows it."""
    _require_kernel(X, use_kernel)
    return _abi.host().layer(False, X, W, bias, _activation(activation), residual, *_flags(offset, approx_bwd))


def gated_linear(X, W, bias=None, activation="silu", *, offset=None, approx_bwd=False, use_kernel=True):
    """activation(X Wg^T + bg) (*) (X Wu^T + bu): the first half of a gated feed-forward layer.  W [2 hidden, d_in] holds the
    gate's rows and then the other factor's, bias [2 hidden] likewise; the result is [..., hidden].  activation as for linear_act."""
    _require_kernel(X, use_kernel)
    return _abi.host().layer(True, X, W, bias, _activation(activation), None, *_flags(offset, approx_bwd))


def rotary_tables(positions, dim, base=10000.0, *, scaling=None, device=None):
    """(cos, sin), each [positions, dim / 2]: the angles p base^(-2 i / dim) of the positions p = 0 ... positions - 1, taken in
    double precision and rounded once.  dim: how many values of a head are rotated (an even number).

    scaling stretches a model trained on `original` positions to longer ones by `factor`:
      {"type": "linear", "factor"}                 every angle over factor
      {"type": "base", "factor"}                   a larger base: base factor^(dim / (dim - 2)), which divides the slowest angle by
                                                   factor and leaves the fastest
      {"type": "by_parts", "factor", "original"}   angles that turn more than `fast` (32) times over `original` positions as they are,
                                                   those that turn less than `slow` (1) times over factor, a blend between; both tables
                                                   times 0.1 ln(factor) + 1"""
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_tables: an even number of values is rotated, got {dim}")
    if positions < 0:
        raise ValueError("rotary_tables: a negative number of positions")
    index = torch.arange(0, dim, 2, dtype=torch.float64)
    scaling = dict(scaling or {})
    kind, factor, magnitude = scaling.pop("type", None), float(scaling.pop("factor", 1.0)), 1.0
    if factor <= 0:
        raise ValueError("rotary_tables: the factor is positive")
    if kind == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    speed = base ** (-index / dim)
    if kind == "linear":
        speed = speed / factor
    elif kind == "by_parts":
        if "original" not in scaling:
            raise ValueError("rotary_tables: 'by_parts' needs the number of original positions")
        turns = scaling.pop("original") * speed / (2 * math.pi)
        fast, slow = float(scaling.pop("fast", 32.0)), float(scaling.pop("slow", 1.0))
        if not fast > slow:
            raise ValueError("rotary_tables: fast turns more often than slow")
        keep = ((turns - slow) / (fast - slow)).clamp(0.0, 1.0)
        speed = speed * keep + speed / factor * (1.0 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif kind not in (None, "base"):
        raise ValueError(f"rotary_tables: unknown scaling {kind!r}")
    if scaling:
        raise ValueError(f"rotary_tables: unknown scaling arguments {sorted(scaling)}")
    angle = torch.arange(positions, dtype=torch.float64).outer(speed)
    return tuple((t * magnitude).to(torch.float32).to(device or torch.get_default_device()) for t in (angle.cos(), angle.sin()))


def rotary(q, k, cos, sin, positions=None, *, q_weight=None, k_weight=None, eps=1e-6, interleaved=False,
           offset=None, approx_bwd=False, use_kernel=True):
    """Queries and keys [batch, tokens, heads, dim] (any strides but the last; k may be None) rotated by their positions; returns
    both.  cos and sin are tables [table rows, rotated / 2] (see rotary_tables); the first `rotated` values of every head turn in
    pairs i, i + rotated / 2, or 2 i, 2 i + 1 if `interleaved`, the others stay:

        y1 = z1 (*) cos - z2 (*) sin        y2 = z2 (*) cos + z1 (*) sin

    positions: the tables' row of every token, int64 [tokens] or [batch, tokens]; None: token t is at row t.  A position outside the
    tables makes a head's rotated values NaN.  With q_weight / k_weight [dim] every head is normed first, in the same pass:
    z = x (/) sqrt(mean(x (*) x) + eps) (*) weight."""
    _require_kernel(q, use_kernel)
    if k is None and k_weight is not None:
        raise ValueError("rotary: a weight for keys that are not there")
    flags = _flags(offset, approx_bwd)
    out = _abi.host().rotary(q, k, cos, sin, positions, q_weight, k_weight, bool(interleaved), float(eps), *flags)
    return out[0], (out[1] if k is not None else None)
