"""Attention and its gradients in 64 bits with an offset and with the slopes of every kind chosen apart (test infrastructure).

Every quantity is a pair of its value and of how far 32 bits may be off from it.  A piecewise-affine product or quotient (its offset is one more of them)
rounds nothing and changes by at most twice its relative change in an operand; a sum of n terms adds n EPS times the sum of their magnitudes; 2^t changes by
at most 2^t per unit of t; a weight below 2^-58 of the largest is known to 2^-60 of it.  A slope or the power of two below a number is a step: where the number is closer to one than it may be
off, the step's size counts (`moved`).  Below 2^-126 a float32's step is 2^-149 whatever its size (STEP).
"""
import numpy as np

import _block_ref as block
from _attention_ref import EPS, LN2, LOG2E, STEP, TURN, floor_log2, moved, visible


class Known:
    def __init__(self, value, off=0.0):
        self.v = np.asarray(value, float)
        self.o = np.broadcast_to(np.asarray(off, float), self.v.shape)

    def __neg__(self):
        return Known(-self.v, self.o)

    def __add__(self, other):
        v = self.v + other.v
        return Known(v, self.o + other.o + EPS * np.abs(v))

    def times(self, other):
        """An ordinary product."""
        v = self.v * other.v
        return Known(v, np.abs(self.v) * other.o + self.o * np.abs(other.v) + self.o * other.o + EPS * np.abs(v))

    def at(self, index):
        return Known(self.v[index], self.o[index])

    @property
    def T(self):
        return Known(self.v.T, self.o.T)


def total(terms, axis, keepdims=False):
    n = terms.v.shape[axis]
    return Known(terms.v.sum(axis, keepdims=keepdims), terms.o.sum(axis, keepdims=keepdims) + n * EPS * np.abs(terms.v).sum(axis, keepdims=keepdims))


def below(x):
    """The power of two below |x|; 0 for 0."""
    return np.where(x == 0, 0.0, np.ldexp(1.0, floor_log2(np.where(x == 0, 1.0, x)).astype(int)))


def step_of(x, y):
    """What x (*) y grows by per unit of y, which has a value of its own: a power of two."""
    (fx, ex), (fy, _) = np.frexp(np.abs(x)), np.frexp(np.abs(y))
    carry = (2.0 * fx - 1.0) + np.where(y == 0, 0.0, 2.0 * fy - 1.0) >= 1.0
    return np.where(x == 0, 0.0, np.sign(x) * np.ldexp(1.0, (ex - 1 + carry).astype(int)))


def ends(v, o):
    """What is o off: as it is, at both ends, and right below a power of two that lies between."""
    border = below(np.abs(v) + o) * (1.0 - 2.0 ** -40)
    return v, v + o, v - o, np.where(border > np.abs(v) - o, np.sign(v) * border, v)


class Arithmetic:
    def __init__(self, offset, first, second, exponent):
        self.offset = float(np.float32(1.0 if offset is None else offset))
        self.first, self.second, self.exponent = first, second, exponent          # approximate ones

    def mul(self, a, b):
        def plain(x, y):
            return block.mul(block.mul(x, y), self.offset)
        return Known(plain(a.v, b.v), 2.0 * (plain(a.o, np.abs(b.v)) + plain(np.abs(a.v), b.o) + plain(a.o, b.o)))

    def div(self, a, b):
        v = block.div(block.div(a.v, b.v), self.offset)
        return Known(v, 2.0 * (block.div(block.div(a.o, np.abs(b.v)), self.offset) + np.abs(v) * b.o / np.abs(b.v)))

    def slope(self, other, own, with_offset=True):
        """What own (*) other grows by per unit of own."""
        factor = block.mul(other.v, self.offset) if with_offset else other.v
        off = 2.0 * other.o
        here = step_of(factor, own.v)
        # (together they may pass where neither does alone, and a piece may begin and end in between: right below a power of two)
        corners = [np.abs(step_of(f, o) - here) for f in ends(factor, off) for o in ends(own.v, own.o)]
        # (what is known to less than a piece's width may be anywhere in one)
        anywhere = np.where(own.o > 0.2 * np.abs(own.v), np.abs(here), 0.0) + np.where(off > 0.2 * np.abs(factor), np.abs(here) + 2.0 * np.abs(step_of(np.abs(factor) + off, own.v)), 0.0)
        return Known(here, np.maximum.reduce(corners + [anywhere]))

    def of_mul(self, own, other, d, approx):
        return self.mul(d, other) if approx else d.times(self.slope(other, own))

    def of_dividend(self, own, over, d):
        inverse = self.div(Known(np.ones_like(over.v)), over)
        return self.mul(inverse, d) if self.first else d.times(self.slope(inverse, own, False))

    def of_divisor(self, quotient, over, d):
        if self.second:
            return -self.mul(self.div(quotient, over), d)
        power = Known(below(quotient.v) * np.sign(quotient.v), moved(below, np.abs(quotient.v), quotient.o))
        by = Known(1.0 / below(over.v), moved(lambda x: 1.0 / below(x), over.v, over.o))
        return -d.times(power.times(by))


class Head:
    """One batch entry's query head, as _attention_ref.Head."""

    def __init__(self, q, k, v, see, slope=None, cap=None, scale=None, offset=None, flags=(True, True, True)):
        self.ar = ar = Arithmetic(offset, *flags)
        q, k, v = (Known(x) for x in (q, k, v))
        tokens, keys, dim = q.v.shape[0], k.v.shape[0], q.v.shape[1]
        self.scale = Known(float(np.float32(dim ** -0.5 if scale is None else scale)))
        self.q, self.k, self.v, self.see = q, k, v, see
        self.qs = ar.mul(q, self.scale)
        self.a = x = total(ar.mul(self.qs.at((slice(None), None)), k.at((None,))), 2)
        self.cap = cap and Known(float(np.float32(cap)))
        if cap:
            self.u = ar.div(Known(np.abs(x.v), x.o), self.cap)
            power = ar.mul(self.u, Known(TURN))
            self.power = Known(np.minimum(power.v, 64.0), power.o)
            self.w = Known(block.exp2(-self.power.v), self.power.o + EPS)
            self.n_cap, self.m_cap = Known(1.0) + -self.w, Known(1.0) + self.w
            self.th = ar.div(self.n_cap, self.m_cap)
            capped = ar.mul(self.th, self.cap)
            x = Known(np.sign(x.v) * capped.v, capped.o)
        if slope is not None:
            far = np.abs(np.arange(keys - tokens, keys)[:, None] - np.arange(keys)[None]).astype(float)
            x = x + -ar.mul(Known(float(np.float32(slope))), Known(far))
        self.x = x
        t = ar.mul(x, Known(LOG2E))
        self.some = see.any(1, keepdims=True)
        most = np.where(self.some, np.floor(np.where(see, t.v, -np.inf).max(1, keepdims=True, initial=-np.inf)), 0.0)
        lower = np.where(see, t.v - most, -100.0)
        e = np.where(see, block.exp2(lower), 0.0)
        # (a whole t is a power of two to the bit; the whole number taken off it is up to 8 below the largest's, so that the difference is rounded at up to that much more)
        rounded = np.where((t.o == 0) & (t.v == np.rint(t.v)), 0.0, t.o + 2.0 * EPS * (6.0 + np.abs(lower)))
        self.e = Known(e, np.where(see, e * rounded + np.where(e < 2.0 ** -58, 2.0 ** -60, 0.0), 0.0))
        l = total(self.e, 1, True)
        self.l = Known(np.where(self.some, l.v, 1.0), np.where(self.some, l.o, 0.0))
        self.n = total(ar.mul(self.e.at((slice(None), slice(None), None)), v.at((None,))), 1)
        self.y = ar.div(self.n, self.l)

    def grads(self, dy):
        ar, dy = self.ar, Known(dy)
        approx = ar.first
        dn = ar.of_dividend(self.n, self.l, dy)
        dl = total(ar.of_divisor(self.y, self.l, dy), 1, True)
        e, v, dn_at = self.e.at((slice(None), slice(None), None)), self.v.at((None,)), dn.at((slice(None), None))
        de = total(ar.of_mul(e, v, dn_at, ar.first), 2) + dl
        de = Known(de.v, de.o + (self.q.v.shape[1] + 3) * STEP)
        if ar.exponent:
            d = ar.mul(self.e, de)
        else:
            d = Known(below(self.e.v), moved(below, self.e.v, self.e.o)).times(de).times(ar.slope(Known(LOG2E), self.x))
        if self.cap:
            dth = ar.of_mul(self.th, self.cap, d, ar.first)
            dw = ar.of_divisor(self.th, self.m_cap, dth) + -ar.of_dividend(self.n_cap, self.m_cap, dth)
            if ar.exponent:
                dpower = -ar.mul(ar.mul(self.w, Known(LN2)), dw)
            else:
                dpower = -Known(below(self.w.v), moved(below, self.w.v, self.w.o)).times(dw)
            du = ar.of_mul(self.u, Known(TURN), dpower, ar.first)
            d = ar.of_dividend(self.a, self.cap, du)
        da = Known(np.where(self.see, d.v, 0.0), np.where(self.see, d.o, 0.0))
        da_at = da.at((slice(None), slice(None), None))
        dqs = total(ar.of_mul(self.qs.at((slice(None), None)), self.k.at((None,)), da_at, ar.first), 1)
        dq = ar.of_mul(self.q, self.scale, dqs, ar.first)
        dk = total(ar.of_mul(self.k.at((None,)), self.qs.at((slice(None), None)), da_at, ar.second), 0)
        dv = total(ar.of_mul(v, e, dn_at, ar.second), 0)
        return [Known(g.v, g.o + STEP) for g in (dq, dk, dv)]


def attention(q, k, v, dy=None, causal=True, window=None, prefix=None, documents=None, slopes=None, cap=None, scale=None, offset=None, flags=(True, True, True)):
    """[batch, tokens, heads, dim]: y, its bound, the gradients for q, k and v, theirs."""
    batch, tokens, heads, dim = q.shape
    keys, group = k.shape[1], heads // k.shape[2]
    out = [np.zeros(x.shape) for x in (q, q, k, v)]
    off = [np.zeros(x.shape) for x in (q, q, k, v)]
    for b in range(batch):
        see = visible(tokens, keys, causal, window, None if prefix is None else prefix[b], None if documents is None else documents[b])
        for h in range(heads):
            kv = h // group
            head = Head(q[b, :, h], k[b, :, kv], v[b, :, kv], see, None if slopes is None else slopes[h], cap, scale, offset, flags)
            parts = [head.y] + (head.grads(dy[b, :, h]) if dy is not None else [])
            for i, part in enumerate(parts):
                at = (b, slice(None), h if i < 2 else kv)
                out[i][at] += part.v
                off[i][at] += part.o + 2.0 * EPS * group * np.abs(part.v) * (i >= 2)
    return out[0], off[0], out[1:], off[1:]
