"""The operators of a decoder block and its training step, as a program that trains or serves one calls them, beside their
plain forms.

  linear_act    pam.linear_act: X W^T + bias, an activation and a residual in one product; with gradients where the case trains
  gated         pam.gated_linear: act(X Wg^T + bg) (*) (X Wu^T + bu), both projections in one weight
  rotary        pam.rotary: the rotation of queries and keys by their positions, with or without the norm of every head before it
  clip          pam_amd.optim.clip_grads: the global norm of many gradients, and the gradients scaled down to a bound

(*) and (/) are the piecewise-affine product and quotient: the sum and the difference of two numbers' exponents and mantissa
fractions.  With `own` false `run` computes the operators from elementary torch operations on the bit patterns, in 32 bits;
with `own` true by the package's kernels.  `exact` is the definition in 64 bits.  Gradients are the approximate ones that the
training recipes use (the other factor for a product's slope): the exact ones jump by a factor of two where a mantissa sum
carries, and no two orders of the sums before agree on them.
"""
import math

import torch

own = False

EPS = 1e-6
CAP = 64.0                       # the sigmoid's exponent is held below this: 1 + 2^64 is 2^64, and x (/) 2^64 nothing


# ---------------------------------------------------------------- the cases

def _linear_act(tokens, d_in, d_out, activation="", bias=True, residual=False, train=False, zeros=False):
    return dict(kind="linear_act", tokens=tokens, d_in=d_in, d_out=d_out, activation=activation, bias=bias, residual=residual,
                train=train, zeros=zeros)


def _gated(tokens, width, hidden, activation="silu", bias=False, train=False):
    return dict(kind="gated", tokens=tokens, width=width, hidden=hidden, activation=activation, bias=bias, train=train)


def _rotary(batch, tokens, heads, kv_heads, dim, rotated, norm=False, interleaved=False, table=4096, scattered=False, train=False):
    return dict(kind="rotary", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotated=rotated, norm=norm,
                interleaved=interleaved, table=table, scattered=scattered, train=train)


def _clip(width, hidden, layers, vocabulary, bound):
    return dict(kind="clip", width=width, hidden=hidden, layers=layers, vocabulary=vocabulary, bound=bound)


def listed():
    def named(name, case):
        return dict(case, name=name)
    return [
        # serving one token: the projection behind a 2048-wide feed-forward layer, back onto the residual stream of a 1024-wide model
        named("linear_act_one_token", _linear_act(1, 2048, 1024, residual=True)),
        # a short prompt of odd length through a projection of odd width, with padding tokens whose rows are zero
        named("linear_act_ragged", _linear_act(771, 300, 1001, activation="gelu", residual=True, zeros=True)),
        # a training step of the feed-forward layer of the translation model: 4096 tokens a batch, 512 -> 1024
        named("linear_act_train", _linear_act(4096, 512, 1024, activation="silu", train=True)),
        # serving one token: both projections of a gated layer, whose 33.5 MB of weights are read once
        named("gated_one_token", _gated(1, 1024, 4096)),
        # ... five sequences decoded side by side by a 768-wide model
        named("gated_five_tokens", _gated(5, 768, 2048, bias=True)),
        # the smallest training step: a layer of a 64-wide model on 8 x 12 tokens, all launches and host work
        named("gated_train_small", _gated(96, 64, 128, train=True)),
        # the largest: 4096 tokens of a 1024-wide model
        named("gated_train_large", _gated(4096, 1024, 2048, train=True)),
        # one decoding step of 16 sequences at positions of their own, queries and keys normed
        named("rotary_decode", _rotary(16, 1, 16, 4, 128, 128, norm=True, scattered=True)),
        # a prompt of odd length, half of every 80-wide head rotated, neighbouring pairs
        named("rotary_prompt", _rotary(1, 3001, 12, 12, 80, 40, interleaved=True)),
        # a training step on 4 x 4096 tokens: shared keys' heads, norms with their weights' gradients
        named("rotary_train", _rotary(4, 4096, 16, 4, 128, 128, norm=True, train=True)),
        # gradients of a two-layer, 64-wide model below the bound: the norm is all that is needed
        named("clip_small", _clip(64, 128, 2, 512, 1e3)),
        # gradients of the translation model (253 tensors) scaled down
        named("clip_large", _clip(512, 1024, 6, 10000, 0.1)),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high):
    """Most widths are multiples of 32, some are anything."""
    w = _spread(rng, low, high)
    return max(32, w // 32 * 32) if rng.random() < 0.6 else w


def draw(rng):
    kind = rng.choice(["linear_act", "linear_act", "gated", "gated", "rotary", "rotary", "clip"])
    train = rng.random() < 0.5
    if kind == "linear_act":
        d_in, d_out = _width(rng, 40, 2048), _width(rng, 40, 4096)
        most = 16_000_000_000 // (d_in * d_out)
        few = not train and rng.random() < 0.4
        tokens = _spread(rng, 1, 8) if few else _spread(rng, 8, min(12608, most))
        # (relu's slope jumps at zero, where two orders of a sum fall on either side)
        activation = rng.choice(["", "silu", "gelu"] if train else ["", "relu", "silu", "gelu"])
        return _linear_act(tokens, d_in, d_out, activation=activation, bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=train,
                           zeros=rng.random() < 0.3)
    if kind == "gated":
        width, hidden = _width(rng, 40, 1536), _width(rng, 40, 4096)
        most = 8_000_000_000 // (width * hidden)
        few = not train and rng.random() < 0.4
        tokens = _spread(rng, 1, 8) if few else _spread(rng, 8, min(8192, most))
        return _gated(tokens, width, hidden, activation=rng.choice(["silu", "silu", "gelu"]), bias=rng.random() < 0.3, train=train)
    if kind == "rotary":
        dim = rng.choice([32, 64, 64, 80, 96, 100, 128, 128, 256, 18])
        rotated = dim if rng.random() < 0.6 else max(2, dim // 4 * 2)
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4])
        tokens = 1 if not train and rng.random() < 0.3 else _spread(rng, 2, 4096)
        most = 40_000_000 // (tokens * (heads + kv_heads) * dim)
        return _rotary(_spread(rng, 1, max(1, min(32, most))), tokens, heads, kv_heads, dim, rotated, norm=rng.random() < 0.6,
                       interleaved=rng.random() < 0.3, scattered=rng.random() < 0.4, train=train)
    return _clip(_width(rng, 33, 512), _width(rng, 50, 1024), rng.randint(1, 6), _spread(rng, 100, 10000), 10.0 ** rng.uniform(-2, 3))


# ---------------------------------------------------------------- what a program holds before the call

def _leaf(t, train):
    return t.requires_grad_(True) if train else t


def _clip_shapes(case):
    w, f = case["width"], case["hidden"]
    attention = [(w, w), (w,)] * 4
    ffn = [(f, w), (f,), (w, f), (w,)]
    norm = [(w,), (w,)]
    encoder = attention + norm + ffn + norm
    decoder = attention + norm + attention + norm + ffn + norm
    return [(case["vocabulary"], w)] + case["layers"] * encoder + case["layers"] * decoder


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = {"case": dict(case)}
    kind = case["kind"]
    if kind == "linear_act":
        m, k, n, train = case["tokens"], case["d_in"], case["d_out"], case["train"]
        x = normal(m, k)
        if case["zeros"]:
            x[m - (m + 3) // 4:] = 0.0                                   # padding tokens
        s["x"] = _leaf(x, train)
        s["w"] = _leaf(normal(n, k, std=k ** -0.5), train)
        s["bias"] = _leaf(normal(n, std=0.1), train) if case["bias"] else None
        s["residual"] = _leaf(normal(m, n), train) if case["residual"] else None
        s["dy"] = normal(m, n, std=1e-2) if train else None
    elif kind == "gated":
        m, k, f, train = case["tokens"], case["width"], case["hidden"], case["train"]
        s["x"] = _leaf(normal(m, k), train)
        s["w"] = _leaf(normal(2 * f, k, std=k ** -0.5), train)           # the gate's rows, then the other factor's
        s["bias"] = _leaf(normal(2 * f, std=0.1), train) if case["bias"] else None
        s["dy"] = normal(m, f, std=1e-2) if train else None
    elif kind == "rotary":
        b, t, h, kv, d, r, train = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dim", "rotated", "train"))
        s["q"], s["k"] = _leaf(normal(b, t, h, d), train), _leaf(normal(b, t, kv, d), train)
        s["qw"] = _leaf(normal(d, std=0.1).add_(1.0), train) if case["norm"] else None
        s["kw"] = _leaf(normal(d, std=0.1).add_(1.0), train) if case["norm"] else None
        angle = torch.arange(case["table"], dtype=torch.float64).outer(10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r))
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
        s["positions"] = torch.randint(0, case["table"], (b, t), generator=g, device="cuda") if case["scattered"] else None
        s["dq"], s["dk"] = (normal(b, t, h, d, std=1e-2), normal(b, t, kv, d, std=1e-2)) if train else (None, None)
    else:
        # gradients as a backward pass leaves them, in tensors of their own; the clipped ones go to one flat buffer
        s["grads"] = [normal(*shape, std=1e-3) for shape in _clip_shapes(case)]
        sizes = [t.numel() for t in s["grads"]]
        s["flat"] = torch.empty(sum(sizes), device="cuda")
        s["out"] = [o.view(t.shape) for o, t in zip(s["flat"].split(sizes), s["grads"])]
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import pam_amd as pam
    from pam_amd.optim import clip_grads

    case = s["case"]
    kind = case["kind"]
    if kind == "linear_act":
        y = pam.linear_act(s["x"], s["w"], s["bias"], case["activation"] or None, s["residual"], approx_bwd=True)
        if not case["train"]:
            return y
        wanted = [t for t in (s["x"], s["w"], s["bias"], s["residual"]) if t is not None]
        return y, torch.autograd.grad(y, wanted, s["dy"])
    if kind == "gated":
        y = pam.gated_linear(s["x"], s["w"], s["bias"], case["activation"], approx_bwd=True)
        if not case["train"]:
            return y
        return y, torch.autograd.grad(y, [t for t in (s["x"], s["w"], s["bias"]) if t is not None], s["dy"])
    if kind == "rotary":
        q, k = pam.rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                          interleaved=case["interleaved"], approx_bwd=True)
        if not case["train"]:
            return q, k
        wanted = [t for t in (s["q"], s["k"], s["qw"], s["kw"]) if t is not None]
        return q, k, torch.autograd.grad((q, k), wanted, (s["dq"], s["dk"]))
    norm = clip_grads(s["grads"], case["bound"], out=s["out"])
    return norm, s["flat"]


# ---------------------------------------------------------------- the plain forms, in 32 bits

_BIAS, _SIGN = 0x3F800000, -0x80000000


def _mul(a, b):
    """a (*) b: the magnitudes' bit patterns added less the bias, zero where that underflows."""
    a, b = torch.broadcast_tensors(a, b)
    ai, bi = a.view(torch.int32), b.view(torch.int32)
    magnitude = (ai & 0x7FFFFFFF) - _BIAS + (bi & 0x7FFFFFFF)
    magnitude = torch.where((a == 0) | (b == 0), 0, magnitude.clamp_(min=0))
    return (magnitude | ((ai ^ bi) & _SIGN)).view(torch.float32)


def _div(a, b):
    a, b = torch.broadcast_tensors(a, b)
    ai, bi = a.view(torch.int32), b.view(torch.int32)
    magnitude = (ai & 0x7FFFFFFF) - (bi & 0x7FFFFFFF) + _BIAS
    magnitude = torch.where(a == 0, 0, magnitude.clamp_(min=0))
    return (magnitude | ((ai ^ bi) & _SIGN)).view(torch.float32)


def _exp2(x):
    f = torch.floor(x)
    return torch.ldexp((1.0 + x) - f, f.to(torch.int32))


def _log2(x):
    return (x.view(torch.int32) - _BIAS).to(torch.float32) * 2.0 ** -23


def _sqrt(x):
    return _exp2(_mul(_log2(x), _number(0.5, x)))


def _number(v, like):
    return torch.tensor(v, dtype=torch.float32, device=like.device)


_CHUNK = 1 << 27


def _product(a, b):
    """sum_k a[m, k] (*) b[n, k], some rows of a at a time."""
    m, k, n = a.shape[0], a.shape[1], b.shape[0]
    # (a zero's magnitude is so far below every other that its sums are negative)
    def parts(t):
        bits = t.contiguous().view(torch.int32)
        return torch.where(t == 0, -(1 << 30), (bits & 0x7FFFFFFF) - _BIAS // 2), bits & _SIGN
    am, a_sign = parts(a)
    bm, b_sign = parts(b)
    bm = bm - (_BIAS - 2 * (_BIAS // 2))
    out = torch.empty(m, n, device=a.device)
    rows = max(1, _CHUNK // (n * k))
    for i in range(0, m, rows):
        for j in range(0, n, max(1, _CHUNK // k)):
            e = j + max(1, _CHUNK // k)
            magnitude = (am[i:i + rows, None, :] + bm[None, j:e]).clamp_(min=0)
            magnitude ^= a_sign[i:i + rows, None, :]
            magnitude ^= b_sign[None, j:e]
            out[i:i + rows, j:e] = magnitude.view(torch.float32).sum(-1)
    return out


_SCALE = {"silu": 1.0, "gelu": 1.702}


def _act(z, activation):
    if not activation:
        return z
    if activation == "relu":
        return z.relu()
    c = _number(-_SCALE[activation] * math.log2(math.e), z)
    return _div(z, 1.0 + _exp2(_mul(z, c).clamp(max=CAP)))


def _act_grad(z, dy, activation):
    """The approximate gradient of _act: those of the quotient, of the power of two and of the product with the constant."""
    if not activation:
        return dy
    if activation == "relu":
        return torch.where(z > 0, dy, 0.0)
    c, ln2, one = _number(-_SCALE[activation] * math.log2(math.e), z), _number(math.log(2.0), z), _number(1.0, z)
    t = _mul(z, c)
    e = _exp2(t.clamp(max=CAP))
    u = 1.0 + e
    du = -_mul(_div(_div(z, u), u), dy)
    dt = torch.where(t <= CAP, _mul(_mul(e, ln2), du), 0.0)
    return _mul(_div(one, u), dy) + _mul(dt, c)


def _rotate(x, cos, sin, rotated, interleaved):
    head, rest = x[..., :rotated], x[..., rotated:]
    x1, x2 = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rotated // 2], head[..., rotated // 2:])
    y1, y2 = _mul(x1, cos) - _mul(x2, sin), _mul(x2, cos) + _mul(x1, sin)
    head = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((head, rest), -1)


def _norm(x, weight):
    d = _number(float(x.shape[-1]), x)
    root = _sqrt(_div(_mul(x, x).sum(-1, keepdim=True), d) + EPS)
    n = _div(x, root)
    return _mul(n, weight), n, root, d


def _norm_grad(x, weight, dz):
    _, n, root, d = _norm(x, weight)
    one, half, ln2 = _number(1.0, x), _number(0.5, x), _number(math.log(2.0), x)
    dn = _mul(dz, weight)
    dweight = _mul(dz, n).flatten(0, -2).sum(0)
    droot = -_mul(_div(n, root), dn).sum(-1, keepdim=True)
    variance = _div(_mul(x, x).sum(-1, keepdim=True), d) + EPS
    dlog = _mul(_mul(_mul(root, ln2), droot), half)
    dsum = _mul(_div(one, d), _div(_div(dlog, variance), ln2))
    dx = _mul(_div(one, root), dn) + 2.0 * _mul(dsum, x)
    return dx, dweight


def _run_plain(s):
    with torch.no_grad():
        return _plain(s)


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "linear_act":
        z = _product(s["x"], s["w"])
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, case["activation"])
        if s["residual"] is not None:
            y = y + s["residual"]
        if not case["train"]:
            return y
        dz = _act_grad(z, s["dy"], case["activation"])
        grads = [_product(dz, s["w"].t()), _product(dz.t(), s["x"].t())]
        grads += [dz.sum(0)] if s["bias"] is not None else []
        grads += [s["dy"].clone()] if s["residual"] is not None else []
        return y, grads
    if kind == "gated":
        f = case["hidden"]
        z = _product(s["x"], s["w"])
        if s["bias"] is not None:
            z = z + s["bias"]
        gate, up = z[:, :f].contiguous(), z[:, f:].contiguous()
        a = _act(gate, case["activation"])
        y = _mul(a, up)
        if not case["train"]:
            return y
        dz = torch.cat((_act_grad(gate, _mul(s["dy"], up), case["activation"]), _mul(s["dy"], a)), 1)
        grads = [_product(dz, s["w"].t()), _product(dz.t(), s["x"].t())]
        return y, grads + ([dz.sum(0)] if s["bias"] is not None else [])
    if kind == "rotary":
        t, r, il = case["tokens"], case["rotated"], case["interleaved"]
        at = s["positions"] if s["positions"] is not None else torch.arange(t, device=s["cos"].device)
        cos, sin = s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2)
        ys, dxs, dws = [], [], []
        for x, w, dy in ((s["q"], s["qw"], s["dq"]), (s["k"], s["kw"], s["dk"])):
            ys.append(_rotate(_norm(x, w)[0] if w is not None else x, cos, sin, r, il))
            if case["train"]:
                dz = _rotate(dy, cos, -sin, r, il)
                dx, dw = _norm_grad(x, w, dz) if w is not None else (dz, None)
                dxs.append(dx)
                dws += [dw] if w is not None else []
        return (*ys, dxs + dws) if case["train"] else tuple(ys)
    total = torch.stack([_mul(t, t).sum() for t in s["grads"]]).sum()
    norm = _sqrt(total)
    scale = _div(_number(case["bound"], norm), norm + EPS).clamp(max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(_mul(t, scale))
    return norm, s["flat"]


# ---------------------------------------------------------------- the definition, in 64 bits

class _Def:
    """The arithmetic on real numbers, as doubles: |x| = 2^E (1 + m) and (E, m) added as E + m is."""

    BIAS, MAGNITUDE, SIGN = 1023 << 52, (1 << 63) - 1, -(1 << 63)

    @staticmethod
    def bits(x):
        # (a zero stands as 2^-900: its products vanish beside anything fp32 holds)
        return torch.where(x == 0, 2.0 ** -900, x.double()).view(torch.int64)

    @classmethod
    def join(cls, magnitude, sign):
        x = (magnitude.clamp(min=0) | (sign & cls.SIGN)).view(torch.float64)
        return torch.where(x.abs() < 2.0 ** -700, 0.0, x)

    @classmethod
    def mul(cls, a, b):
        i, j = cls.bits(a), cls.bits(b)
        return cls.join((i & cls.MAGNITUDE) - cls.BIAS + (j & cls.MAGNITUDE), i ^ j)

    @classmethod
    def div(cls, a, b):
        i, j = cls.bits(a), cls.bits(b)
        return cls.join((i & cls.MAGNITUDE) - (j & cls.MAGNITUDE) + cls.BIAS, i ^ j)

    @staticmethod
    def exp2(x):
        whole = x.floor()
        return torch.ldexp(1.0 + (x - whole), whole.to(torch.int32))

    @staticmethod
    def log2(x):
        mantissa, exponent = torch.frexp(x)
        return (exponent - 1).double() + (2.0 * mantissa - 1.0)

    @classmethod
    def power(cls, x, p):
        return cls.exp2(cls.mul(cls.log2(x), p))

    @classmethod
    def product(cls, a, b):
        """sum_k a[m, k] (*) b[k, n]"""
        i, j = cls.bits(a), cls.bits(b).t().contiguous() - cls.BIAS
        out = torch.empty(a.shape[0], b.shape[1], dtype=torch.float64, device=a.device)
        most = 1 << 26
        columns = max(1, min(out.shape[1], most // a.shape[1]))
        rows = max(1, most // (columns * a.shape[1]))
        for r in range(0, out.shape[0], rows):
            for c in range(0, out.shape[1], columns):
                out[r:r + rows, c:c + columns] = (i[r:r + rows].unsqueeze(1) + j[c:c + columns].unsqueeze(0)).view(torch.float64).sum(2)
        return out


def _f32(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda").double()      # a constant as the definition has it


def _sigmoid_parts(z, activation):
    c = _f32(-(1.702 if activation == "gelu" else 1.0) * math.log2(math.e))
    t = _Def.mul(z, c)
    e = _Def.exp2(t.clamp(max=CAP))
    return c, t, e, 1.0 + e


def exact(case, seed):
    with torch.no_grad():
        return _exact(case, prepare(case, seed))


def _exact(case, s):
    D, kind = _Def, case["kind"]
    if kind in ("linear_act", "gated"):
        x, w, activation = s["x"].double(), s["w"].double(), case["activation"]
        z = D.product(x, w.t())
        if s["bias"] is not None:
            z = z + s["bias"].double()
        gate = z[:, :case["hidden"]] if kind == "gated" else z
        if activation in ("silu", "gelu"):
            c, t, e, u = _sigmoid_parts(gate, activation)
            a = D.div(gate, u)
        else:
            a = gate.clamp(min=0.0) if activation == "relu" else gate
        y = D.mul(a, z[:, case["hidden"]:]) if kind == "gated" else a
        if s.get("residual") is not None:
            y = y + s["residual"].double()
        if not case["train"]:
            return y
        dy = s["dy"].double()
        da = D.mul(dy, z[:, case["hidden"]:]) if kind == "gated" else dy
        if activation in ("silu", "gelu"):
            through_u = -D.mul(D.div(a, u), da)
            through_t = torch.where(t <= CAP, D.mul(D.mul(e, _f32(math.log(2.0))), through_u), 0.0)
            dz = D.mul(D.div(torch.ones_like(u), u), da) + D.mul(through_t, c)
        else:
            dz = torch.where(gate > 0, da, 0.0) if activation == "relu" else da
        if kind == "gated":
            dz = torch.cat((dz, D.mul(dy, a)), 1)
        grads = [D.product(dz, w), D.product(dz.t(), x)]
        grads += [dz.sum(0)] if s["bias"] is not None else []
        grads += [dy] if s.get("residual") is not None else []
        return y, grads
    if kind == "rotary":
        r = case["rotated"]
        at = s["positions"] if s["positions"] is not None else torch.arange(case["tokens"], device="cuda").expand(case["batch"], -1)
        cos, sin = (s[key].double()[at][:, :, None, :] for key in ("cos", "sin"))
        first = torch.arange(0, r, 2, device="cuda") if case["interleaved"] else torch.arange(r // 2, device="cuda")
        second = first + (1 if case["interleaved"] else r // 2)
        outs, grads, weights = [], [], []
        for name in ("q", "k"):
            x = s[name].double()
            z = x
            if case["norm"]:
                w = s[name + "w"].double()
                v = D.div(D.mul(x, x).sum(-1, keepdim=True), torch.full((), float(case["dim"]), dtype=torch.float64, device="cuda")) + EPS
                root = D.power(v, _f32(0.5))
                n = D.div(x, root)
                z = D.mul(n, w)
            y = z.clone()
            y[..., first] = D.mul(z[..., first], cos) - D.mul(z[..., second], sin)
            y[..., second] = D.mul(z[..., second], cos) + D.mul(z[..., first], sin)
            outs.append(y)
            if case["train"]:
                dy = s["d" + name].double()
                dz = dy.clone()
                dz[..., first] = D.mul(dy[..., first], cos) + D.mul(dy[..., second], sin)
                dz[..., second] = D.mul(dy[..., second], cos) - D.mul(dy[..., first], sin)
                if case["norm"]:
                    dn = D.mul(dz, w)
                    weights.append(D.mul(dz, n).sum((0, 1, 2)))
                    droot = -D.mul(D.div(n, root), dn).sum(-1, keepdim=True)
                    dpower = D.mul(D.mul(root, _f32(math.log(2.0))), droot)
                    dv = D.div(D.div(D.mul(dpower, _f32(0.5)), v), _f32(math.log(2.0)))
                    dsquare = D.mul(D.div(torch.ones_like(v), torch.full_like(v, float(case["dim"]))), dv)
                    dz = D.mul(D.div(torch.ones_like(root), root), dn) + 2.0 * D.mul(dsquare, x)
                grads.append(dz)
        return (*outs, grads + weights) if case["train"] else tuple(outs)
    total = sum(D.mul(t.double(), t.double()).sum() for t in s["grads"])
    norm = D.power(total, _f32(0.5))
    scale = D.div(_f32(case["bound"]), norm + EPS).clamp(max=1.0)
    return norm, torch.cat([D.mul(t, scale).flatten() for t in s["grads"]])


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    """Bytes: every input read once and every output written once.  Operations: two per PAM multiply-accumulate (an integer and a
    float add), a few per value elsewhere."""
    kind, train = case["kind"], case.get("train", False)
    if kind == "linear_act":
        m, k, n = case["tokens"], case["d_in"], case["d_out"]
        values = m * k + n * k + (n if case["bias"] else 0) + m * n * (2 if case["residual"] else 1)
        each = 10 if case["activation"] in ("silu", "gelu") else 2
        return {"bytes": 4 * values * (2 if train else 1), "flops": (6 if train else 2) * m * k * n + each * (4 if train else 1) * m * n}
    if kind == "gated":
        m, k, f = case["tokens"], case["width"], case["hidden"]
        values = m * k + 2 * f * k + (2 * f if case["bias"] else 0) + m * f
        return {"bytes": 4 * values * (2 if train else 1), "flops": (12 if train else 4) * m * k * f + 14 * (4 if train else 1) * m * f}
    if kind == "rotary":
        rows = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        tables = min(case["table"], case["batch"] * case["tokens"]) * case["rotated"]
        n = rows * case["dim"]
        return {"bytes": 4 * (n * (4 if train else 2) + tables) + (8 * case["batch"] * case["tokens"] if case["scattered"] else 0),
                "flops": n * (6 + (6 if case["norm"] else 0)) * (3 if train else 1)}
    n = sum(math.prod(shape) for shape in _clip_shapes(case))
    return {"bytes": 8 * n, "flops": 4 * n}
