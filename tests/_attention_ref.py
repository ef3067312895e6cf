"""Attention from its definition, in 64 bits with numpy, with bounds on what 32 bits may make of it (test infrastructure).

Bounds: half a step of a float32 is EPS = 2^-24.  A piecewise-affine product or quotient changes by at most twice its relative change
in an operand, 2^t by at most 2^t per unit of t, and a sum of n terms in any order by n EPS times the sum of their magnitudes.
Below 2^-126 a float32's step is 2^-149 whatever its size (STEP): each of the dim terms of dl, dl's own sum and de are off by up to one more,
and so is each result.

An exact gradient's slopes are powers of two that step where a factor passes from one piece into the next.  Where a factor is closer to such a border than
it may be off, 32 bits may have the slope of either side: the step's size, what the slope changes by between the factor less and plus its bound, times
what it weighs, is added to the bound (`moved`) where a test asks for it (`borders`); most inputs have no such pair.  One pair in some ten thousand is that close (2^t with t within 1e-6 of a whole number).
"""
import numpy as np

from _block_ref import div, exp2, mul, product

EPS = 2.0 ** -24
STEP = 2.0 ** -149
LOG2E = float(np.float32(1.4426950408889634))
TURN = float(np.float32(2.0 * 1.4426950408889634))
LN2 = float(np.float32(0.6931471805599453))


def visible(tokens, keys, causal=True, window=None, prefix=None, documents=None):
    """[tokens, keys] for one batch entry"""
    i, j = np.arange(keys - tokens, keys)[:, None], np.arange(keys)[None]
    see = np.ones((tokens, keys), bool)
    if causal:
        see &= j <= i
    if window:
        see &= np.abs(i - j) < window
    if prefix is not None:
        see |= j < prefix
    if documents is not None:
        see &= (documents[i] == documents[j]) & (documents[i] >= 0)
    return see


def floor_log2(x):
    return np.frexp(x)[1] - 1.0


def slope(other, own):
    """What own (*) other grows by per unit of own: a power of two."""
    (fo, eo), (fw, ew) = np.frexp(np.abs(other)), np.frexp(np.abs(own))
    carry = (2.0 * fo - 1.0) + np.where(own == 0, 0.0, 2.0 * fw - 1.0) >= 1.0
    return np.where(other == 0, 0.0, np.sign(other) * np.ldexp(1.0, (eo - 1 + carry).astype(int)))


def moved(f, x, off):
    """What a step function changes by within x - off ... x + off."""
    here = f(x)
    return np.maximum(np.abs(f(x + off) - here), np.abs(f(np.maximum(x - off, np.where(x > 0, 0.5 * x, -np.inf))) - here))


def power(x):
    return np.ldexp(1.0, np.where(x == 0, -300, floor_log2(np.where(x == 0, 1.0, x))).astype(int))


class Head:
    """One batch entry's query head: q [tokens, dim], k and v [keys, dim], see [tokens, keys], far the distances."""

    def __init__(self, q, k, v, see, slope=None, cap=None, scale=None):
        q, k, v = (np.asarray(x, float) for x in (q, k, v))
        tokens, keys, dim = q.shape[0], k.shape[0], q.shape[1]
        self.scale = float(np.float32(dim ** -0.5 if scale is None else scale))
        self.k, self.v, self.see, self.cap = k, v, see, cap and float(np.float32(cap))
        self.qs = mul(q, self.scale)
        self.q = q
        self.a, size = product(self.qs, k.T)
        self.a_off = (dim + 3) * EPS * size                                  # how far a may be off
        x, x_off = self.a, self.a_off
        if cap:
            self.u = div(np.abs(x), self.cap)
            self.power = np.minimum(mul(self.u, TURN), 64.0)
            self.w = exp2(-self.power)
            self.th = div(1.0 - self.w, 1.0 + self.w)
            # the cap's slope is below 3: u's by 1 / cap, w's by 2.9, th's by 1 (each up to twice that), and 1 - w is off by EPS
            x, x_off = np.sign(x) * mul(self.th, self.cap), 12.0 * x_off + 16.0 * EPS * self.cap
        if slope is not None:
            far = np.abs(np.arange(keys - tokens, keys)[:, None] - np.arange(keys)[None]).astype(float)
            bias = mul(float(np.float32(slope)), far)
            x, x_off = x - bias, x_off + 2.0 * EPS * (np.abs(x) + np.abs(bias))
        self.x, self.x_off = x, x_off
        t = mul(x, LOG2E)
        t_off = 2.0 * x_off + 2.0 * EPS * np.abs(t)
        self.some = see.any(1, keepdims=True)
        most = np.floor(np.where(see, t, -np.inf).max(1, keepdims=True, initial=-np.inf))
        self.most = np.where(self.some, most, 0.0)
        self.e = np.where(see, exp2(np.where(see, t - self.most, -100.0)), 0.0)
        self.e_off = self.e * (t_off + 2.0 * EPS * (2.0 + np.abs(np.where(see, t - self.most, 0.0)))) + np.where(see, 2.0 ** -60, 0.0)
        self.l = np.where(self.some, self.e.sum(1, keepdims=True), 1.0)
        self.l_off = self.e_off.sum(1, keepdims=True) + keys * EPS * self.l
        self.n, size = product(self.e, v)
        self.n_off = n_off = 2.0 * product(self.e_off, np.abs(v))[0] + (keys + 2) * EPS * size
        self.y = div(self.n, self.l)
        self.y_off = 2.0 * (n_off / self.l + np.abs(self.y) * (self.l_off / self.l + EPS))

    def grads(self, dy, approx=True, borders=False):
        """dq, dk, dv and how far each may be off."""
        dy = np.asarray(dy, float)
        keys, dim = self.k.shape
        rel_l = self.l_off / self.l
        if approx:
            dn = mul(div(1.0, self.l), dy)
            part = mul(div(self.y, self.l), dy)
        else:
            dn = dy * slope(div(1.0, self.l), self.n)
            part = dy * np.ldexp(np.sign(self.y), (floor_log2(self.y) - floor_log2(self.l)).astype(int))
        dn_off = np.abs(dn) * (4.0 * rel_l + 4.0 * EPS)
        borders = borders and not approx
        if borders:
            inverse = div(1.0, self.l)
            dn_off = dn_off + np.abs(dy) * (moved(lambda n: slope(inverse, n), self.n, self.n_off) + moved(lambda i: slope(i, self.n), inverse, 2.0 * inverse * (rel_l + EPS)))
        dl = -part.sum(1, keepdims=True)
        dl_off = (np.abs(part) * (6.0 * rel_l + (dim + 4) * EPS)).sum(1, keepdims=True) + 4.0 * (self.y_off / self.l * np.abs(dy)).sum(1, keepdims=True) + (dim + 1) * STEP
        if borders:
            quotient = moved(power, np.abs(self.y), self.y_off) / power(self.l) + power(self.y) * moved(lambda l: 1.0 / power(l), self.l, self.l_off)
            dl_off = dl_off + 2.0 * (np.abs(dy) * quotient).sum(1, keepdims=True)
        if approx:
            p, size = product(dn, self.v.T)
        else:
            terms = dn[:, None, :] * slope(self.v[None], self.e[:, :, None])
            p, size = terms.sum(2), np.abs(terms).sum(2)
            de_moved = 0.0 if not borders else (np.abs(dn)[:, None, :] * moved(lambda e: slope(self.v[None], e), self.e[:, :, None], self.e_off[:, :, None])).sum(2)
        de = p + dl
        de_off = 2.0 * product(dn_off, np.abs(self.v.T))[0] + (dim + 3) * EPS * size + dl_off + EPS * np.abs(de) + STEP + (0.0 if approx else de_moved)
        if approx:
            da = mul(self.e, de)
        else:
            da = np.ldexp(1.0, np.where(self.see, floor_log2(np.where(self.see, self.e, 1.0)), -300).astype(int)) * de * slope(LOG2E, self.x)
        da_off = 2.0 * (self.e_off * np.abs(de) + self.e * de_off) * 2.0 + 2.0 * EPS * np.abs(da)
        if borders:
            by_score = slope(LOG2E, self.x)
            da_off = da_off + np.abs(de) * (moved(power, self.e, self.e_off) * by_score + power(self.e) * moved(lambda x: slope(LOG2E, x), self.x, self.x_off)) * 2.0
        if self.cap:
            m = 1.0 + self.w
            if approx:
                dth = mul(da, self.cap)
                dw = -(mul(div(self.th, m), dth) + mul(div(1.0, m), dth))
                du = mul(mul(mul(self.w, LN2), -dw), TURN)
                da2 = mul(div(1.0, self.cap), du)
            else:
                dth = da * slope(self.cap, self.th)
                dw = -(dth * np.ldexp(np.where(self.th == 0, 0.0, 1.0), (floor_log2(self.th) - floor_log2(m)).astype(int)) + dth * slope(div(1.0, m), 1.0 - self.w))
                du = np.ldexp(1.0, floor_log2(self.w).astype(int)) * -dw * slope(TURN, self.u)
                da2 = du * slope(div(1.0, self.cap), self.a)
            # |da2| is at most 6 |da|; its own factors change by w's, th's and m's relative change, 12 EPS + 6 a_off / cap
            da_off = 12.0 * da_off + 8.0 * np.abs(da) * (16.0 * EPS + 12.0 * self.a_off / self.cap)
            da = da2
        da, da_off = np.where(self.see, da, 0.0), np.where(self.see, da_off, 0.0)

        def out(weights, off, rows, exact_own):
            """sum over i of weights[i, o] (*) rows[i, d]"""
            if approx:
                total, size = product(weights, rows)
            else:
                terms = weights[:, :, None] * slope(rows[None], exact_own[:, None, :])
                total, size = terms.sum(1), np.abs(terms).sum(1)
            return total, 2.0 * product(off, np.abs(rows))[0] + (weights.shape[1] + 2) * EPS * size
        dqs, dqs_off = out(da, da_off, self.k, self.qs)
        dq = mul(dqs, self.scale) if approx else dqs * slope(self.scale, self.q)
        dq_off = 2.0 * self.scale * dqs_off + EPS * np.abs(dq)
        dk, dk_off = out(da.T, da_off.T, self.qs, self.k)
        if approx:
            dv, size = product(self.e.T, dn)
        else:
            terms = dn[None] * slope(self.e.T[:, :, None], self.v[:, None, :])
            dv, size = terms.sum(1), np.abs(terms).sum(1)
            dv_moved = 0.0 if not borders else (np.abs(dn)[None] * moved(lambda e: slope(e, self.v[:, None, :]), self.e.T[:, :, None], self.e_off.T[:, :, None])).sum(1)
        dv_off = 2.0 * (product(self.e_off.T, np.abs(dn))[0] + product(self.e.T, dn_off)[0]) + (self.e.shape[0] + 2) * EPS * size + (0.0 if approx else dv_moved)
        return (dq, dk, dv), (dq_off + STEP, dk_off + STEP, dv_off + STEP)


def attention(q, k, v, dy=None, approx=True, causal=True, window=None, prefix=None, documents=None, slopes=None, cap=None, scale=None, borders=False):
    """[batch, tokens, heads, dim]: y and its bound, with dy also the gradients for q, k, v and theirs."""
    batch, tokens, heads, dim = q.shape
    keys, group = k.shape[1], heads // k.shape[2]
    y, y_off = np.zeros(q.shape), np.zeros(q.shape)
    grads = [np.zeros(x.shape) for x in (q, k, v)] if dy is not None else None
    offs = [np.zeros(x.shape) for x in (q, k, v)] if dy is not None else None
    for b in range(batch):
        see = visible(tokens, keys, causal, window, None if prefix is None else prefix[b], None if documents is None else documents[b])
        for h in range(heads):
            head = Head(q[b, :, h], k[b, :, h // group], v[b, :, h // group], see, None if slopes is None else slopes[h], cap, scale)
            y[b, :, h], y_off[b, :, h] = head.y, head.y_off
            if dy is not None:
                parts, off = head.grads(dy[b, :, h], approx, borders)
                grads[0][b, :, h], offs[0][b, :, h] = parts[0], off[0]
                for i in (1, 2):
                    grads[i][b, :, h // group] += parts[i]
                    offs[i][b, :, h // group] += off[i] + 2.0 * EPS * group * np.abs(parts[i])
    return (y, y_off, grads, offs) if dy is not None else (y, y_off)
