"""The decoder block's operators from their definitions, in 64 bits with numpy (test infrastructure).

|x| = 2^E (1 + m): a (*) b adds E + m, a (/) b subtracts it; values here are moderate, so that nothing over- or underflows.
"""
import numpy as np

CAP = 64.0
LN2 = float(np.float32(0.6931471805599453))
SCALE = {"silu": float(np.float32(-1.4426950408889634)), "gelu": float(np.float32(-1.702 * 1.4426950408889634))}


def _parts(x):
    m, e = np.frexp(np.abs(x))
    return e - 1.0, 2.0 * m - 1.0                       # E, fraction; a zero has E = -1, fraction -1: masked by the callers


def _join(e, f, sign):
    carry = np.floor(f)                                 # the fractions' sum or difference lies in [-1, 2)
    return sign * np.ldexp(1.0 + (f - carry), (e + carry).astype(int))


def mul(a, b):
    a, b = np.broadcast_arrays(np.asarray(a, float), np.asarray(b, float))
    (ea, fa), (eb, fb) = _parts(a), _parts(b)
    return np.where((a == 0) | (b == 0), 0.0, _join(ea + eb, fa + fb, np.sign(a) * np.sign(b)))


def div(a, b):
    a, b = np.broadcast_arrays(np.asarray(a, float), np.asarray(b, float))
    (ea, fa), (eb, fb) = _parts(a), _parts(b)
    return np.where(a == 0, 0.0, _join(ea - eb, fa - fb, np.sign(a) * np.sign(b)))


def exp2(x):
    f = np.floor(x)
    return np.ldexp(1.0 + (x - f), f.astype(int))


def log2(x):
    e, f = _parts(x)
    return e + f


def sqrt(x):
    return exp2(mul(log2(x), 0.5))


def product(a, b):
    """a[m, k] (x) b[k, n] and the sum of the terms' magnitudes"""
    terms = mul(a[:, :, None], b[None])
    return terms.sum(1), np.abs(terms).sum(1)


def act(z, name):
    if name is None:
        return z
    if name == "relu":
        return np.maximum(z, 0.0)
    return div(z, 1.0 + exp2(np.minimum(mul(z, SCALE[name]), CAP)))


def act_grad(z, d, name):
    """The approximate gradient: the other factor for a product's slope, the primitives' formulas."""
    if name is None:
        return d
    if name == "relu":
        return np.where(z > 0, d, 0.0)
    c = SCALE[name]
    t = mul(z, c)
    e = exp2(np.minimum(t, CAP))
    u = 1.0 + e
    du = -mul(div(div(z, u), u), d)
    dt = np.where(t <= CAP, mul(mul(e, LN2), du), 0.0)
    return mul(div(1.0, u), d) + mul(dt, c)


def linear_act(x, w, bias, name, residual):
    z, _ = product(x, w.T)
    y = act(z + (0.0 if bias is None else bias), name)
    return y if residual is None else y + residual


def gated(x, w, bias, name):
    f = w.shape[0] // 2
    z = product(x, w.T)[0] + (0.0 if bias is None else bias)
    return mul(act(z[:, :f], name), z[:, f:])


def pairs(rotated, interleaved):
    return (slice(0, rotated, 2), slice(1, rotated, 2)) if interleaved else (slice(0, rotated // 2), slice(rotated // 2, rotated))


def norm(x, weight, eps):
    root = sqrt(div(mul(x, x).sum(-1, keepdims=True), float(x.shape[-1])) + eps)
    return mul(div(x, root), weight)


def rotary(x, cos, sin, weight=None, eps=1e-6, interleaved=False):
    """x [..., tokens, heads, dim], cos and sin [..., tokens, rotated / 2]: the rows of the tokens"""
    z = x if weight is None else norm(x, weight, eps)
    i, j = pairs(2 * cos.shape[-1], interleaved)
    c, s = cos[..., None, :], sin[..., None, :]
    y = z.copy()
    y[..., i] = mul(z[..., i], c) - mul(z[..., j], s)
    y[..., j] = mul(z[..., j], c) + mul(z[..., i], s)
    return y


def rotary_grad(x, dy, cos, sin, weight=None, eps=1e-6, interleaved=False):
    """The approximate gradients for x and for the weight."""
    i, j = pairs(2 * cos.shape[-1], interleaved)
    c, s = cos[..., None, :], sin[..., None, :]
    dz = dy.copy()
    dz[..., i] = mul(dy[..., i], c) + mul(dy[..., j], s)
    dz[..., j] = mul(dy[..., j], c) - mul(dy[..., i], s)
    if weight is None:
        return dz, None
    d = float(x.shape[-1])
    v = div(mul(x, x).sum(-1, keepdims=True), d) + eps
    root = sqrt(v)
    n = div(x, root)
    dn = mul(dz, weight)
    droot = -mul(div(n, root), dn).sum(-1, keepdims=True)
    dlog = mul(mul(mul(root, LN2), droot), 0.5)
    dsum = mul(div(1.0, d), div(div(dlog, v), LN2))
    return mul(div(1.0, root), dn) + 2.0 * mul(dsum, x), mul(dz, n).reshape(-1, x.shape[-1]).sum(0)


def clip(grads, bound, eps=1e-6):
    total = sum(mul(g, g).sum() for g in grads)
    length = float(sqrt(np.array(total)))
    scale = min(1.0, float(div(bound, length + eps))) if np.isfinite(bound) else 1.0
    return length, [mul(g, scale) for g in grads]


def slope(f, x, direction, h=2.0 ** -30):
    """The derivative of f along `direction` at x by differences: everything here is affine in pieces, so that within one the
    difference is exact up to rounding."""
    return (f(x + h * direction) - f(x - h * direction)) / (2.0 * h)
