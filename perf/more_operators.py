"""Attention in one piece and the cache that it reads while decoding, as a program that trains or serves a model calls them, beside
their plain forms.

  attention     pam.attention: every query over the keys that it may see (causal, a window, a prefix, documents), its scores
                with a bias by distance or capped; with gradients where the case trains
  append        pam.rotary_append: queries and keys normed and rotated by their positions, keys and values put into the pages of a cache
  cached        pam.cached_attention: one or a few new tokens of every sequence over its pages

(*) and (/) are the piecewise-affine product and quotient: the sum and the difference of two numbers' exponents and mantissa
fractions, 2^x the inverse of such a number's logarithm.  With the scores a_ij = sum_d (q_id (*) scale) (*) k_jd, capped to
x = cap (*) tanh(a (/) cap), tanh u = (1 - w) (/) (1 + w) with w = 2^-(u (*) 2 log2 e), and less slope (*) distance,

  e_ij = 2^(x_ij (*) log2 e),   l_i = sum_j e_ij,   y_id = (sum_j e_ij (*) v_jd) (/) l_i

over the keys j that query i sees; a query that sees none has the result zero.  A row's e and l may be scaled by a power of
two, which moves no result.  With `own` false `run` computes this from elementary torch operations on the bit patterns, in 32
bits; with `own` true by the package's kernels.  `exact` is the definition in 64 bits.  Gradients are the approximate ones that
the training recipes use (the other factor for a product's slope, e itself for the slope of e^x).
"""
import math

import torch

own = False

EPS = 1e-6
LOG2E = math.log2(math.e)


# ---------------------------------------------------------------- the cases

def _attention(batch, tokens, keys, heads, kv_heads, dim, causal=True, window=0, prefix=0, documents=0, slopes=False, cap=0.0, train=False):
    return dict(kind="attention", batch=batch, tokens=tokens, keys=keys, heads=heads, kv_heads=kv_heads, dim=dim, causal=causal, window=window,
                prefix=prefix, documents=documents, slopes=slopes, cap=cap, train=train)


def _append(batch, tokens, heads, kv_heads, dim, rotated, page, seen, norm=False, interleaved=False, ragged=False):
    return dict(kind="append", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotated=rotated, page=page, seen=seen,
                norm=norm, interleaved=interleaved, ragged=ragged)


def _cached(batch, tokens, heads, kv_heads, dim, page, seen, window=0, slopes=False, cap=0.0, ragged=False):
    return dict(kind="cached", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, page=page, seen=seen, window=window,
                slopes=slopes, cap=cap, ragged=ragged)


def listed():
    def named(name, case):
        return dict(case, name=name)
    return [
        # the smallest training step: a 64-wide model's heads on 8 sequences of 12 tokens
        named("attention_small", _attention(8, 12, 12, 4, 2, 16, train=True)),
        # a vision model of 64 images of 197 patches, every patch over all of them
        named("attention_patches", _attention(64, 197, 197, 3, 3, 64, causal=False)),
        # a prompt's last 333 tokens over 1500, shared keys' heads, wide heads
        named("attention_prompt", _attention(2, 333, 1500, 16, 4, 128)),
        # training on documents packed into rows of 2048 tokens, the last ones padding
        named("attention_documents", _attention(2, 2048, 2048, 8, 2, 128, documents=7, train=True)),
        # training with a prefix that all tokens see and a bias by distance, an odd length, heads of 80
        named("attention_prefix", _attention(2, 1001, 1001, 6, 3, 80, prefix=129, slopes=True, train=True)),
        # training a layer with a sliding window and capped scores
        named("attention_window", _attention(4, 1024, 1024, 8, 8, 64, window=256, cap=30.0, train=True)),
        # the largest training step: 4096 tokens, causal
        named("attention_large", _attention(1, 4096, 4096, 8, 2, 64, train=True)),
        # one decoding step of 16 sequences, keys and queries normed
        named("append_one_token", _append(16, 1, 16, 4, 128, 128, 64, 200, norm=True, ragged=True)),
        # prompts of different lengths, padded, half of every head rotated in neighbouring pairs
        named("append_prompts", _append(5, 1777, 12, 4, 80, 40, 16, 30, interleaved=True, ragged=True)),
        # the smallest: one sequence early in its life
        named("cached_early", _cached(1, 1, 4, 2, 64, 16, 37)),
        # 16 sequences of different lengths, up to 4000 tokens
        named("cached_batch", _cached(16, 1, 16, 4, 128, 64, 4000, ragged=True)),
        # one sequence with a long past, five tokens at once to be checked
        named("cached_long", _cached(1, 5, 8, 2, 128, 64, 100000, slopes=True)),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly spread over its logarithm."""
    high = max(low, high)
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "append", "append", "cached", "cached", "cached"])
    dim = rng.choice([16, 32, 64, 64, 80, 96, 100, 128, 128, 256, 18])
    kv_heads = rng.choice([1, 2, 3, 4])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    if kind == "attention":
        train = rng.random() < 0.5
        keys = _spread(rng, 1, 4096)
        tokens = keys if train or rng.random() < 0.5 else _spread(rng, 1, keys)
        most = int((2e10 if train else 4e10) / (3 if train else 1) // (tokens * keys * heads * dim))
        while most < 1:
            keys, tokens = (keys + 1) // 2, (tokens + 1) // 2
            most = int((2e10 if train else 4e10) / (3 if train else 1) // (tokens * keys * heads * dim))
        return _attention(_spread(rng, 1, min(16, most)), tokens, keys, heads, kv_heads, dim, causal=rng.random() < 0.8,
                          window=_spread(rng, 1, keys) if rng.random() < 0.25 else 0, prefix=_spread(rng, 1, keys) if rng.random() < 0.2 else 0,
                          documents=rng.randint(2, 9) if rng.random() < 0.3 and keys >= 32 else 0, slopes=rng.random() < 0.25,
                          cap=rng.choice([20.0, 30.0, 50.0]) if rng.random() < 0.25 else 0.0, train=train)
    if kind == "append":
        rotated = dim if rng.random() < 0.6 else max(2, dim // 4 * 2)
        tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
        batch = _spread(rng, 1, max(1, min(32, 12_000_000 // (tokens * (heads + kv_heads) * dim))))
        return _append(batch, tokens, heads, kv_heads, dim, rotated, rng.choice([1, 16, 17, 64, 256]), _spread(rng, 1, 1000), norm=rng.random() < 0.6,
                       interleaved=rng.random() < 0.3, ragged=rng.random() < 0.6)
    tokens = 1 if rng.random() < 0.6 else rng.randint(2, 9)
    batch = _spread(rng, 1, 32)
    seen = _spread(rng, 1, max(1, min(100000, 50_000_000 // (batch * kv_heads * dim))))
    return _cached(batch, tokens, heads, kv_heads, dim, rng.choice([1, 16, 17, 64, 256]), seen, window=_spread(rng, 1, seen) if rng.random() < 0.25 else 0,
                   slopes=rng.random() < 0.25, cap=rng.choice([20.0, 30.0, 50.0]) if rng.random() < 0.2 else 0.0, ragged=rng.random() < 0.6)


def _uneven(count, most):
    """`count` whole numbers up to `most`, the first one `most`, the others spread by the golden ratio."""
    return [most] + [max(1, round(most * (i * 0.6180339887 % 1.0))) for i in range(1, count)]


def _document_of(case):
    """The document of every key: their lengths are uneven, the last one is padding."""
    n, keys = case["documents"], case["keys"]
    weights = [0.3 + i * 0.6180339887 % 1.0 for i in range(n)]
    ids, at = [], 0
    for i, w in enumerate(weights):
        end = keys if i == n - 1 else min(keys, at + max(1, int(keys * w / sum(weights))))
        ids += [i if i < n - 1 else -1] * (end - at)
        at = end
    return ids


# ---------------------------------------------------------------- what a program holds before the call

def _leaf(t, train):
    return t.requires_grad_(True) if train else t


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = {"case": dict(case)}
    kind, b, t, h, kv, d = (case[key] for key in ("kind", "batch", "tokens", "heads", "kv_heads", "dim"))
    if case.get("slopes"):
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda")
    else:
        s["slopes"] = None
    if kind == "attention":
        keys, train = case["keys"], case["train"]
        s["q"], s["k"], s["v"] = (_leaf(normal(*shape), train) for shape in ((b, t, h, d), (b, keys, kv, d), (b, keys, kv, d)))
        s["dy"] = normal(b, t, h, d, std=1e-2) if train else None
        s["documents"] = torch.tensor(_document_of(case), device="cuda").expand(b, -1).contiguous() if case["documents"] else None
        s["prefix"] = torch.tensor(_uneven(b, case["prefix"]), device="cuda") if case["prefix"] else None
        return s
    # a cache whose pages belong to the sequences in any order; some belong to none
    page, seen = case["page"], case["seen"]
    lengths = _uneven(b, seen) if case["ragged"] else [seen] * b
    each = (seen + t + page - 1) // page
    total = b * each + 3
    s["pages"] = torch.randperm(total, generator=g, device="cuda")[:b * each].view(b, each).to(torch.int32).contiguous()
    s["lengths"] = torch.tensor(lengths, device="cuda")
    s["counts"] = torch.tensor(_uneven(b, t), device="cuda") if case["ragged"] and t > 1 else None
    s["cache_k"], s["cache_v"] = normal(total, page, kv, d), normal(total, page, kv, d)
    s["q"] = normal(b, t, h, d)
    if kind == "append":
        r = case["rotated"]
        s["k"], s["v"] = normal(b, t, kv, d), normal(b, t, kv, d)
        s["qw"] = normal(d, std=0.1).add_(1.0) if case["norm"] else None
        s["kw"] = normal(d, std=0.1).add_(1.0) if case["norm"] else None
        angle = torch.arange(seen + t, dtype=torch.float64).outer(10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r))
        s["cos"], s["sin"] = angle.cos().float().cuda(), angle.sin().float().cuda()
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    import pam_amd as pam

    case = s["case"]
    if case["kind"] == "attention":
        y = pam.attention(s["q"], s["k"], s["v"], causal=case["causal"], window=case["window"] or None, prefix=s["prefix"], documents=s["documents"],
                          slopes=s["slopes"], cap=case["cap"] or None, approx_bwd=True)
        return (y, torch.autograd.grad(y, (s["q"], s["k"], s["v"]), s["dy"])) if case["train"] else y
    if case["kind"] == "append":
        q = pam.rotary_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["cache_k"], s["cache_v"], s["pages"], s["lengths"], s["counts"],
                              q_weight=s["qw"], k_weight=s["kw"], eps=EPS, interleaved=case["interleaved"])
        return q, s["cache_k"], s["cache_v"]
    return pam.cached_attention(s["q"], s["cache_k"], s["cache_v"], s["pages"], s["lengths"], s["counts"], window=case["window"] or None,
                                slopes=s["slopes"], cap=case["cap"] or None)


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
    columns = max(1, min(n, _CHUNK // k))
    rows = max(1, _CHUNK // (columns * k))
    for i in range(0, m, rows):
        for j in range(0, n, columns):
            magnitude = (am[i:i + rows, None, :] + bm[None, j:j + columns]).clamp_(min=0)
            magnitude ^= a_sign[i:i + rows, None, :]
            magnitude ^= b_sign[None, j:j + columns]
            out[i:i + rows, j:j + columns] = magnitude.view(torch.float32).sum(-1)
    return out


def _capped(a, cap):
    """cap (*) tanh(a (/) cap), and what its gradient reads."""
    c = _number(cap, a)
    w = _exp2(-_mul(_div(a.abs(), c), _number(2.0 * LOG2E, a)).clamp(max=64.0))
    th = _div(1.0 - w, 1.0 + w)
    return torch.copysign(_mul(th, c), a), w, th


def _capped_grad(w, th, dx, cap):
    c, one = _number(cap, w), _number(1.0, w)
    dth = _mul(dx, c)
    dw = -_mul(_div(th, 1.0 + w), dth) - _mul(_div(one, 1.0 + w), dth)
    du = -_mul(_mul(_mul(w, _number(math.log(2.0), w)), dw), _number(2.0 * LOG2E, w))
    return _mul(_div(one, c), du)


def _seen(at_q, at_k, causal, window, prefix=None, documents=None):
    """Which keys a query sees; at_q, at_k: their positions."""
    far = at_q[:, None] - at_k[None, :]
    see = torch.ones_like(far, dtype=torch.bool)
    if causal:
        see &= far >= 0
    if window:
        see &= far.abs() < window
    if prefix is not None:
        see |= at_k[None, :] < prefix
    if documents is not None:
        of_q = documents[at_q]
        see &= (of_q[:, None] == documents[None, :]) & (of_q[:, None] >= 0)
    return see, far


def _rows(t):
    """One key head's queries [tokens, heads, dim] as rows, a token's heads behind each other."""
    return t.reshape(-1, t.shape[-1])


def _attend(q, k, v, see, far, slopes, cap, scale, dy=None):
    """One batch entry and key head: q [tokens, group, dim], k and v [keys, dim], see and far [tokens, keys], slopes [group] or None."""
    tokens, group, dim = q.shape
    see, far = (x.repeat_interleave(group, 0) for x in (see, far))
    scale, log2e = _number(scale, q), _number(LOG2E, q)
    qs = _mul(_rows(q), scale)
    a = _product(qs, k)
    x, w, th = _capped(a, cap) if cap else (a, None, None)
    if slopes is not None:
        x = x - _mul(slopes.repeat(tokens)[:, None], far.abs().to(torch.float32))
    t = _mul(x, log2e)
    most = torch.where(see, t, -math.inf).amax(1, keepdim=True).floor()
    e = torch.where(see, _exp2(t - torch.where(most == -math.inf, 0.0, most)), 0.0)
    some = see.any(1, keepdim=True)
    total = torch.where(some, e.sum(1, keepdim=True), 1.0)
    y = _div(_product(e, v.t()), total)
    if dy is None:
        return y.view(tokens, group, dim)
    dy, one = _rows(dy), _number(1.0, q)
    dn = _mul(_div(one, total), dy)
    dl = -_mul(_div(y, total), dy).sum(1, keepdim=True)
    de = _product(dn, v) + dl
    da = _mul(e, de)
    if cap:
        da = torch.where(see, _capped_grad(w, th, da, cap), 0.0)
    dq = _mul(_product(da, k.t()), scale)
    return y.view(tokens, group, dim), dq.view(tokens, group, dim), _product(da.t(), qs.t()), _product(e.t(), dn.t())


def _rotate(x, cos, sin, rotated, interleaved):
    head, rest = x[..., :rotated], x[..., rotated:]
    x1, x2 = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :rotated // 2], head[..., rotated // 2:])
    y1, y2 = _mul(x1, cos) - _mul(x2, sin), _mul(x2, cos) + _mul(x1, sin)
    head = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((head, rest), -1)


def _norm(x, weight):
    variance = _div(_mul(x, x).sum(-1, keepdim=True), _number(float(x.shape[-1]), x)) + EPS
    root = _exp2(_mul(_log2(variance), _number(0.5, x)))
    return _mul(_div(x, root), weight)


def _slots(s):
    """The page and the place in it of every new token, [batch, tokens], and which tokens there are."""
    t, page = s["case"]["tokens"], s["case"]["page"]
    new = torch.arange(t, device="cuda")
    at = s["lengths"][:, None] + new
    there = new < s["counts"][:, None] if s["counts"] is not None else torch.ones_like(at, dtype=torch.bool)
    return s["pages"].gather(1, at // page).long(), at % page, at, there


def _gathered(cache, s, i, end, kv):
    page = s["case"]["page"]
    at = torch.arange(end, device="cuda")
    return cache[s["pages"][i].long()[at // page], at % page, kv]


def _run_plain(s):
    with torch.no_grad():
        return _plain(s)


def _plain(s):
    case = s["case"]
    kind, batch, tokens, heads, kv_heads, dim = (case[key] for key in ("kind", "batch", "tokens", "heads", "kv_heads", "dim"))
    group, scale = heads // kv_heads, dim ** -0.5
    if kind == "append":
        page_of, place, at, there = _slots(s)
        cos, sin = s["cos"][at].unsqueeze(-2), s["sin"][at].unsqueeze(-2)
        q, k = (_rotate(_norm(x, w) if w is not None else x, cos, sin, case["rotated"], case["interleaved"])
                for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])))
        s["cache_k"][page_of[there], place[there]] = k[there]
        s["cache_v"][page_of[there], place[there]] = s["v"][there]
        return torch.where(there[..., None, None], q, 0.0), s["cache_k"], s["cache_v"]
    y = torch.empty_like(s["q"])
    grads = [torch.empty_like(s[name]) for name in "qkv"] if case.get("train") else None
    lengths = s["lengths"].tolist() if kind == "cached" else None
    counts = s["counts"].tolist() if kind == "cached" and s["counts"] is not None else [tokens] * batch
    for i in range(batch):
        if kind == "attention":
            at_q, at_k = torch.arange(case["keys"] - tokens, case["keys"], device="cuda"), torch.arange(case["keys"], device="cuda")
            see, far = _seen(at_q, at_k, case["causal"], case["window"], None if s["prefix"] is None else s["prefix"][i],
                             None if s["documents"] is None else s["documents"][i])
        else:
            end = lengths[i] + counts[i]
            at_q, at_k = torch.arange(lengths[i], end, device="cuda"), torch.arange(end, device="cuda")
            see, far = _seen(at_q, at_k, True, case["window"])
            y[i, counts[i]:] = 0.0
        for j in range(kv_heads):
            mine = slice(j * group, (j + 1) * group)
            slopes = s["slopes"][mine] if s["slopes"] is not None else None
            if kind == "cached":
                k, v = (_gathered(s[name], s, i, end, j) for name in ("cache_k", "cache_v"))
                y[i, :counts[i], mine] = _attend(s["q"][i, :counts[i], mine], k, v, see, far, slopes, case["cap"], scale)
            elif not case["train"]:
                y[i, :, mine] = _attend(s["q"][i, :, mine], s["k"][i, :, j], s["v"][i, :, j], see, far, slopes, case["cap"], scale)
            else:
                y[i, :, mine], grads[0][i, :, mine], grads[1][i, :, j], grads[2][i, :, j] = _attend(
                    s["q"][i, :, mine], s["k"][i, :, j], s["v"][i, :, j], see, far, slopes, case["cap"], scale, s["dy"][i, :, mine])
    return (y, grads) if grads else y


# ---------------------------------------------------------------- the definition, in 64 bits

class _Def:
    """The arithmetic on real numbers, as doubles: |x| = 2^E (1 + m) and (E, m) added as E + m is."""

    BIAS, MAGNITUDE, SIGN = 1023 << 52, (1 << 63) - 1, -(1 << 63)

    @staticmethod
    def bits(x):
        # (a zero stands as 2^-480: its products, with another zero too, are numbers and vanish beside anything fp32 holds)
        return torch.where(x == 0, 2.0 ** -480, x.double()).view(torch.int64)

    @classmethod
    def join(cls, magnitude, sign):
        x = (magnitude.clamp(min=0) | (sign & cls.SIGN)).view(torch.float64)
        return torch.where(x.abs() < 2.0 ** -330, 0.0, x)

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


def exact(case, seed):
    with torch.no_grad():
        return _exact(case, prepare(case, seed))


def _exact_head(case, s, i, head, k, v, positions):
    """One query head over its keys in 64 bits; returns the result and, where the case trains, dq and the head's part of dk and dv."""
    D = _Def
    first, last = positions
    q = s["q"][i, :last - first, head].double()
    mine, keys = torch.arange(first, last, device="cuda").unsqueeze(1), torch.arange(k.shape[0], device="cuda").unsqueeze(0)
    hidden = mine < keys if case.get("causal", True) else torch.zeros_like(mine < keys)
    if case["window"]:
        hidden = hidden | ((mine - keys).abs() >= case["window"])
    if case.get("prefix"):
        hidden = hidden & (keys >= s["prefix"][i])
    if case.get("documents"):
        of = s["documents"][i]
        hidden = hidden | (of[mine] != of[keys]) | (of[mine] < 0)
    scaled = D.mul(q, _f32(case["dim"] ** -0.5))
    score = D.product(scaled, k.t())
    if case["cap"]:
        c, turn = _f32(case["cap"]), _f32(2.0 * LOG2E)
        w = D.exp2(-D.mul(D.div(score.abs(), c), turn).clamp(max=64.0))
        th = D.div(1.0 - w, 1.0 + w)
        x = D.mul(th, c) * score.sign()
    else:
        x = score
    if s["slopes"] is not None:
        x = x - D.mul(s["slopes"][head].double(), (mine - keys).abs().double())
    t = D.mul(x, _f32(LOG2E)).masked_fill(hidden, -math.inf)
    top = t.amax(1, keepdim=True).clamp(min=-1e30).floor()
    e = D.exp2((t - top).clamp(min=-300.0)).masked_fill(hidden, 0.0)
    l = e.sum(1, keepdim=True)
    l = torch.where(l == 0, 1.0, l)
    y = D.div(D.product(e, v), l)
    if not case.get("train"):
        return (y,)
    dy = s["dy"][i, :, head].double()
    through_n = D.mul(D.div(torch.ones_like(l), l), dy)
    through_l = -D.mul(D.div(y, l), dy).sum(1, keepdim=True)
    through_e = D.product(through_n, v.t()) + through_l
    through_x = D.mul(e, through_e)
    if case["cap"]:
        through_th = D.mul(through_x, c)
        through_w = -(D.mul(D.div(torch.ones_like(w), 1.0 + w), through_th) + D.mul(D.div(th, 1.0 + w), through_th))
        through_x = D.mul(D.div(torch.ones_like(c), c), -D.mul(D.mul(D.mul(w, _f32(math.log(2.0))), through_w), turn)).masked_fill(hidden, 0.0)
    return (y, D.mul(D.product(through_x, k), _f32(case["dim"] ** -0.5)), D.product(through_x.t().contiguous(), scaled),
            D.product(e.t().contiguous(), through_n))


def _exact(case, s):
    D, kind, batch, tokens = _Def, case["kind"], case["batch"], case["tokens"]
    if kind == "append":
        r = case["rotated"]
        first = torch.arange(0, r, 2, device="cuda") if case["interleaved"] else torch.arange(r // 2, device="cuda")
        second = first + (1 if case["interleaved"] else r // 2)
        q_out = torch.zeros_like(s["q"], dtype=torch.float64)
        caches = [s["cache_k"].double(), s["cache_v"].double()]
        lengths = s["lengths"].tolist()
        counts = s["counts"].tolist() if s["counts"] is not None else [tokens] * batch
        for i in range(batch):
            n = counts[i]
            at = torch.arange(lengths[i], lengths[i] + n, device="cuda")
            cos, sin = (s[key].double()[at][:, None, :] for key in ("cos", "sin"))
            slot = s["pages"][i].long()[at // case["page"]] * case["page"] + at % case["page"]
            for name, weight in (("q", "qw"), ("k", "kw")):
                z = s[name][i, :n].double()
                if case["norm"]:
                    v = D.div(D.mul(z, z).sum(-1, keepdim=True), torch.full((), float(case["dim"]), dtype=torch.float64, device="cuda")) + EPS
                    z = D.mul(D.div(z, D.exp2(D.mul(D.log2(v), _f32(0.5)))), s[weight].double())
                y = z.clone()
                y[..., first] = D.mul(z[..., first], cos) - D.mul(z[..., second], sin)
                y[..., second] = D.mul(z[..., second], cos) + D.mul(z[..., first], sin)
                if name == "q":
                    q_out[i, :n] = y
                else:
                    caches[0].view(-1, *caches[0].shape[2:])[slot] = y
            caches[1].view(-1, *caches[1].shape[2:])[slot] = s["v"][i, :n].double()
        return q_out, caches[0], caches[1]
    group = case["heads"] // case["kv_heads"]
    y = torch.zeros_like(s["q"], dtype=torch.float64)
    grads = [torch.zeros_like(s[name], dtype=torch.float64) for name in "qkv"] if case.get("train") else None
    for i in range(batch):
        if kind == "cached":
            n = tokens if s["counts"] is None else int(s["counts"][i])
            first = int(s["lengths"][i])
            order = (s["pages"][i].long()[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).flatten()[:first + n]
        else:
            n, first = tokens, case["keys"] - tokens
        for h in range(case["heads"]):
            if kind == "cached":
                k, v = (s[name].flatten(0, 1)[order, h // group].double() for name in ("cache_k", "cache_v"))
            else:
                k, v = s["k"][i, :, h // group].double(), s["v"][i, :, h // group].double()
            out = _exact_head(case, s, i, h, k, v, (first, first + n))
            y[i, :n, h] = out[0]
            if grads:
                grads[0][i, :, h] = out[1]
                grads[1][i, :, h // group] += out[2]
                grads[2][i, :, h // group] += out[3]
    return (y, grads) if grads else y


# ---------------------------------------------------------------- what a pass cannot do without

def _pairs(case, i):
    """How many pairs of a query and a key of batch entry i there are to look at."""
    tokens, keys, window = case["tokens"], case["keys"], case["window"]
    prefix = _uneven(case["batch"], case["prefix"])[i] if case["prefix"] else 0
    document = _document_of(case) if case["documents"] else None
    begin, end = {}, {}
    if document:
        for j, of in enumerate(document):
            begin.setdefault(of, j)
            end[of] = j + 1
    total = 0
    for at in range(keys - tokens, keys):
        low, high = 0, at + 1 if case["causal"] else keys
        if window:
            low, high = max(low, at - window + 1), min(high, at + window)
        first, last = (begin[document[at]], end[document[at]]) if document and document[at] >= 0 else (0, 0) if document else (0, keys)
        body = max(0, min(high, last) - max(low, first))
        head = max(0, min(prefix, last) - first)
        both = max(0, min(high, last, prefix) - max(low, first))
        total += body + head - both
    return total


def work(case):
    """Bytes: every input read once and every output written once.  Operations: two per PAM multiply-accumulate (an integer and a
    float add), ten per weight; a training step's gradients have five products where the result has two, and compute the scores again."""
    b, t, h, kv, d = (case[key] for key in ("batch", "tokens", "heads", "kv_heads", "dim"))
    if case["kind"] == "attention":
        train = case["train"]
        values = 2 * b * t * h * d + 2 * b * case["keys"] * kv * d
        pairs = h * sum(_pairs(case, i) for i in range(b))
        extra = 8 * b * case["keys"] if case["documents"] else 0
        return {"bytes": 4 * values * (2 if train else 1) + extra, "flops": pairs * ((14 if train else 4) * d + (40 if train else 10))}
    lengths = _uneven(b, case["seen"]) if case["ragged"] else [case["seen"]] * b
    counts = _uneven(b, t) if case["ragged"] and t > 1 else [t] * b
    new = sum(counts)
    if case["kind"] == "append":
        rows = new * (h + kv)
        return {"bytes": 4 * (2 * rows * d + 2 * new * kv * d + min(new, case["seen"] + t) * case["rotated"]) + 4 * new,
                "flops": rows * d * (6 + (6 if case["norm"] else 0))}
    keys = sum(min(n + c, case["window"] + c - 1 if case["window"] else n + c) for n, c in zip(lengths, counts))
    pairs = h * sum(sum(min(n + i + 1, case["window"] or n + i + 1) for i in range(c)) for n, c in zip(lengths, counts))
    return {"bytes": 4 * (2 * keys * kv * d + 2 * b * t * h * d), "flops": pairs * (4 * d + 10)}
