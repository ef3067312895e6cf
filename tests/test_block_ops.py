"""The decoder block's operators: product with activation and residual, gated layer, rotation of queries and keys, clipping.

Two references.  The chain of the package's own primitives, bit for bit where the order of the sums is the same (products of
more than 24 rows with sums of at most 1024 terms, rotations without a norm).  And the definition in 64 bits (tests/_block_ref.py), with these bounds, fixed
before the first run:
  * a sum of K PAM terms in float32, in any order: off by at most K 2^-23 times the sum of the terms' magnitudes (the terms
    themselves are exact);
  * a PAM product or quotient passes on at most twice the relative error of an operand, silu and gelu (slopes below 1.3 in
    magnitude) at most 2.6 times the absolute one; 2^t of this arithmetic rounds 1 + t, which is 2^-24 |t| relative;
  * what is elementwise behind a sum of squares (a head's norm): 2^-17 relative to the largest value of the result.
Exact gradients are held to the 64-bit function's differences, as these are its slopes.
"""
import math

import numpy as np
import pytest
import torch

import pam_amd as pam
from pam_amd import optim
import _block_ref as ref
from _util import assert_same_bits

EPS23 = 2.0 ** -23
OFF = 1.0552
FLAGS = [True, False, (True, False), (False, True)]


def normal(rng, *shape, std=1.0):
    return (rng.standard_normal(shape) * std).astype(np.float32)


def gpu(a, grad=False):
    return None if a is None else torch.from_numpy(np.array(a)).cuda().requires_grad_(grad)


def host(t):
    return t.detach().cpu().numpy()


def wide(a):
    return None if a is None else a.astype(np.float64)


# ---------------------------------------------------------------- tables and refusals

def test_tables_are_the_angles_rounded_once():
    cos, sin = pam.rotary_tables(50, 12, base=10000.0, device="cpu")
    angle = np.arange(50)[:, None] * 10000.0 ** (-np.arange(0, 12, 2) / 12)
    assert cos.shape == sin.shape == (50, 6) and cos.dtype is torch.float32
    assert np.abs(cos.numpy() - np.cos(angle)).max() <= 2.0 ** -24 and np.abs(sin.numpy() - np.sin(angle)).max() <= 2.0 ** -24


def test_scaled_tables():
    speed = 10000.0 ** (-np.arange(0, 16, 2) / 16)
    p = np.arange(40)[:, None]
    cos, _ = pam.rotary_tables(40, 16, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert np.allclose(cos.numpy(), np.cos(p * speed / 4.0), rtol=0, atol=1e-7)
    cos, _ = pam.rotary_tables(40, 16, scaling={"type": "base", "factor": 4.0}, device="cpu")
    longer = (10000.0 * 4.0 ** (16 / 14)) ** (-np.arange(0, 16, 2) / 16)
    assert np.allclose(cos.numpy(), np.cos(p * longer), rtol=0, atol=1e-7) and np.isclose(longer[-1], speed[-1] / 4.0)
    cos, sin = pam.rotary_tables(40, 16, scaling={"type": "by_parts", "factor": 8.0, "original": 1024}, device="cpu")
    turns = 1024 * speed / (2 * np.pi)
    keep = np.clip((turns - 1.0) / 31.0, 0, 1)
    assert keep[0] == 1.0 and keep[-1] == 0.0
    scale = 0.1 * math.log(8.0) + 1.0
    assert np.allclose(cos.numpy(), scale * np.cos(p * (speed * keep + speed / 8.0 * (1 - keep))), rtol=0, atol=2e-7)
    for bad in ({"type": "other"}, {"type": "by_parts", "factor": 2.0}, {"type": "linear", "factor": 0.0}, {"type": "linear", "factor": 2.0, "more": 1},
                {"type": "by_parts", "factor": 2.0, "original": 10, "fast": 1.0, "slow": 1.0}):
        with pytest.raises(ValueError):
            pam.rotary_tables(4, 8, scaling=bad, device="cpu")
    for positions, dim in ((4, 7), (4, 0), (-1, 4)):
        with pytest.raises(ValueError):
            pam.rotary_tables(positions, dim, device="cpu")


def test_no_fallback_on_the_cpu():
    x, w = torch.ones(2, 4), torch.ones(6, 4)
    cos, sin = pam.rotary_tables(2, 4, device="cpu")
    for call in (lambda: pam.linear_act(x, w), lambda: pam.gated_linear(x, w), lambda: pam.rotary(x.view(1, 2, 1, 4), None, cos, sin),
                 lambda: optim.clip_grads([x], 1.0), lambda: optim.grad_norm([x])):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(NotImplementedError):
        pam.linear_act(x, w, use_kernel=False)


def test_clip_arguments():
    for call in (lambda: optim.clip_grads([torch.ones(2)], -1.0), lambda: optim.clip_grads([torch.ones(2)], float("nan")),
                 lambda: optim.clip_grads([torch.ones(2)], 1.0, out=[]), lambda: optim.clip_grad_norm_([torch.ones(2)], 1.0, norm_type=1.0)):
        with pytest.raises(ValueError):
            call()
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0          # no gradients


@pytest.mark.gpu
def test_refusals():
    x, w = torch.ones(2, 4, device="cuda"), torch.ones(6, 4, device="cuda")
    q = torch.ones(1, 3, 2, 8, device="cuda")
    cos, sin = pam.rotary_tables(4, 8, device="cuda")
    value = [lambda: pam.linear_act(x, w[:, :3]), lambda: pam.linear_act(x, w, activation="tanh"), lambda: pam.linear_act(x, w[0]),
             lambda: pam.linear_act(x, w, torch.ones(5, device="cuda")), lambda: pam.linear_act(x, w, None, None, torch.ones(2, 5, device="cuda")),
             lambda: pam.gated_linear(x, w[:5]), lambda: pam.gated_linear(x, w, torch.ones(3, device="cuda")),
             lambda: pam.rotary(q[0], None, cos, sin), lambda: pam.rotary(q, q[:, :2], cos, sin), lambda: pam.rotary(q[..., :6], None, cos, sin),
             lambda: pam.rotary(q, None, cos[:2], sin[:2]), lambda: pam.rotary(q, None, cos, sin[:3]),
             lambda: pam.rotary(q, q, cos, sin, q_weight=torch.ones(7, device="cuda")), lambda: pam.rotary(q, None, cos, sin, k_weight=torch.ones(8, device="cuda")),
             lambda: pam.rotary(q, None, cos, sin, torch.zeros(2, device="cuda", dtype=torch.int64)), lambda: pam.rotary(q, None, cos, sin, torch.zeros(3, dtype=torch.int64)),
             lambda: optim.clip_grads([], 1.0), lambda: optim.clip_grads([x], 1.0, out=[w])]
    for call in value:
        with pytest.raises(ValueError):
            call()
    wrong_type = [lambda: pam.linear_act(x.double(), w.double()), lambda: pam.gated_linear(x.half(), w.half()), lambda: pam.rotary(q.bfloat16(), None, cos, sin),
                  lambda: pam.rotary(q, None, cos, sin, torch.zeros(3, device="cuda", dtype=torch.int32)), lambda: optim.clip_grads([x.double()], 1.0)]
    for call in wrong_type:
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError):
        pam.rotary(q, None, cos.clone().requires_grad_(True), sin)
    with pytest.raises(RuntimeError):
        optim.clip_grad_norm_([_with_grad(torch.full((3,), math.nan))], 1.0, error_if_nonfinite=True)


def _with_grad(g):
    p = torch.nn.Parameter(torch.zeros_like(g, device="cuda"))
    p.grad = g.cuda()
    return p


# ---------------------------------------------------------------- the chains of primitives

def chain_act(z, name, kw):
    if name is None:
        return z
    if name == "relu":
        return z.relu()
    t = pam.mul(z, -math.log2(math.e) if name == "silu" else -1.702 * math.log2(math.e), **kw)
    return pam.div(z, 1.0 + pam.exp2(torch.clamp(t, max=64.0), **kw), **kw)


def chain_gated(x, w, bias, name, kw):
    z = pam.linear(x, w, bias, **kw)
    f = w.shape[0] // 2
    return pam.mul(chain_act(z[..., :f].contiguous(), name, kw), z[..., f:].contiguous(), **kw)


def same_with_grads(ours, chain, tensors, dy, what):
    assert_same_bits(host(ours), host(chain), what)
    got = torch.autograd.grad(ours, tensors, dy, retain_graph=True)
    want = torch.autograd.grad(chain, tensors, dy)
    for i, (g, c) in enumerate(zip(got, want)):
        assert_same_bits(host(g), host(c), f"{what}, gradient {i}")


SHAPES = [(29, 4, 4), (27, 33, 20), (64, 64, 64), (70, 130, 132), (100, 515, 66), (300, 96, 8), (33, 40, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
def test_linear_act_is_the_chain(m, k, n, activation):
    rng = np.random.default_rng(m * 7 + n)
    for approx, offset, with_bias, with_residual in [(FLAGS[m % 4], None, True, True), (True, OFF, True, False), (False, None, False, True)]:
        kw = dict(offset=offset, approx_bwd=approx)
        x, w, b, r = gpu(normal(rng, m, k), True), gpu(normal(rng, n, k, std=k ** -0.5), True), gpu(normal(rng, n), True), gpu(normal(rng, m, n), True)
        with torch.no_grad():
            x[m // 2] = 0.0
        dy = gpu(normal(rng, m, n, std=0.1))
        z = pam.linear(x, w, b if with_bias else None, **kw)
        want = chain_act(z, activation, kw)
        if with_residual:
            want = want + r
        got = pam.linear_act(x, w, b if with_bias else None, activation, r if with_residual else None, **kw)
        tensors = [x, w] + ([b] if with_bias else []) + ([r] if with_residual else [])
        same_with_grads(got, want, tensors, dy, f"{kw}")
        with torch.no_grad():
            assert_same_bits(host(pam.linear_act(x, w, b if with_bias else None, activation, r if with_residual else None, **kw)), host(want), "without a graph")


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
def test_gated_linear_is_the_chain(m, k, n, activation):
    """An even number of hidden values; with an odd one the halves may be summed in other pieces."""
    f = n // 2 * 2
    rng = np.random.default_rng(m * 5 + f)
    for approx, offset, with_bias in [(FLAGS[m % 4], None, True), (True, OFF, False), (False, None, False)]:
        kw = dict(offset=offset, approx_bwd=approx)
        x, w, b = gpu(normal(rng, m, k), True), gpu(normal(rng, 2 * f, k, std=k ** -0.5), True), gpu(normal(rng, 2 * f), True)
        with torch.no_grad():
            x[m // 3] = 0.0
        bias = b if with_bias else None
        same_with_grads(pam.gated_linear(x, w, bias, activation, **kw), chain_gated(x, w, bias, activation, kw), [x, w] + ([b] if with_bias else []),
                        gpu(normal(rng, m, f, std=0.1)), f"{kw}")
        with torch.no_grad():
            assert_same_bits(host(pam.gated_linear(x, w, bias, activation, **kw)), host(chain_gated(x, w, bias, activation, kw)), "without a graph")


EDGES = np.array([0.0, -0.0, 1e-40, -1e-42, 1.2e-38, 3e38, -3e38, np.inf, -np.inf, np.nan, 1.0, -1.0, 50.0, -50.0, -200.0, 200.0, 1e-20, -1e30, 64.0, -88.8], dtype=np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("offset", [None, OFF])
def test_activations_of_any_value(activation, offset):
    """A product with 1 hands every value to the activation as it is (as its class)."""
    n = len(EDGES)
    for approx in FLAGS:
        kw = dict(offset=None, approx_bwd=approx)
        x = gpu(np.tile(EDGES[:, None], (1, 1)), True)
        ones = gpu(np.ones((12, 1), np.float32), True)
        dy = gpu(np.resize(EDGES, (n, 12)) + np.float32(0.25))
        kw["offset"] = offset
        z = pam.linear(x, ones, **kw)
        same_with_grads(pam.linear_act(x, ones, None, activation, **kw), chain_act(z, activation, kw), [x, ones], dy, f"{kw}")
        w = gpu(np.concatenate([np.ones((n, 1), np.float32), EDGES[:, None]]), True)
        one = gpu(np.ones((12, 1), np.float32), True)
        same_with_grads(pam.gated_linear(one, w, None, activation, **kw), chain_gated(one, w, None, activation, kw), [one, w], gpu(np.ones((12, n), np.float32)), f"gated {kw}")


@pytest.mark.gpu
def test_activation_is_finite_for_every_finite_value():
    x = gpu(np.array([[-1e4], [-100.0], [-89.0], [-1e-30], [0.0], [100.0], [1e4]] * 2, np.float32))
    one = torch.ones(1, 1, device="cuda")
    for name in ("silu", "gelu"):
        y = pam.linear_act(x, one, None, name).flatten()
        assert y.isfinite().all() and (y[:3].abs() < 1e-14).all() and y[5] == 100.0 and y[6] == 1e4


# ---------------------------------------------------------------- products against 64 bits

def act_slack(z, name):
    """Rounding of the activation itself, relative to its result: 2^t and the quotient."""
    return 0.0 if name in (None, "relu") else (np.abs(ref.mul(z, ref.SCALE[name])) + 4.0) * EPS23 * np.abs(ref.act(z, name)) * 2


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 24, 25, 65])
@pytest.mark.parametrize("k,n", [(1, 1), (3, 5), (64, 7), (129, 30), (257, 66), (1030, 12), (4096, 3)])
def test_products_against_64_bits(m, k, n):
    rng = np.random.default_rng(m * 1000 + k + n)
    for activation, zeros in ((None, False), ("silu", True), ("gelu", False)):
        x, w, b, r = normal(rng, m, k), normal(rng, n, k, std=k ** -0.5), normal(rng, n, std=0.1), normal(rng, m, n)
        if zeros:
            x[:, ::2] = np.maximum(x[:, ::2], 0.0)
            w[n // 2] = 0.0
        z, size = ref.product(wide(x), wide(w).T)
        z, slack = z + wide(b), size * (k + 2) * EPS23 + np.abs(z) * EPS23
        want = ref.act(z, activation) + wide(r)
        got = host(pam.linear_act(gpu(x), gpu(w), gpu(b), activation, gpu(r)))
        bound = 2.6 * slack + act_slack(z, activation) + (np.abs(want) + np.abs(r)) * EPS23 + 1e-30
        assert (np.abs(got - want) <= bound).all(), (activation, np.max(np.abs(got - want) / bound))
        w2, b2 = normal(rng, 2 * n, k, std=k ** -0.5), normal(rng, 2 * n, std=0.1)
        z, size = ref.product(wide(x), wide(w2).T)
        z, slack = z + wide(b2), size * (k + 2) * EPS23 + np.abs(z) * EPS23
        g, u = z[:, :n], z[:, n:]
        a = ref.act(g, activation)
        want = ref.mul(a, u)
        got = host(pam.gated_linear(gpu(x), gpu(w2), gpu(b2), activation))
        bound = 2.0 * ((2.6 * slack[:, :n] + act_slack(g, activation)) * np.abs(u) + slack[:, n:] * np.abs(a)) + np.abs(want) * EPS23 + 1e-30
        assert (np.abs(got - want) <= 1.05 * bound).all(), (activation, np.max(np.abs(got - want) / bound))


def views(rng, rows, cols, how):
    """A matrix of the values of a contiguous one, in other strides or at another alignment."""
    a = normal(rng, rows, cols)
    if how == "row gap":
        t = torch.zeros(rows, cols + 5, device="cuda")[:, 3:3 + cols]
    elif how == "columns":
        t = torch.zeros(cols, rows, device="cuda").t()
    elif how == "odd address":
        t = torch.zeros(rows * cols + 1, device="cuda")[1:].view(rows, cols)
    else:
        t = torch.zeros(rows, 2 * cols, device="cuda")[:, ::2]
    return a, t.copy_(gpu(a))


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["row gap", "columns", "odd address", "every second"])
@pytest.mark.parametrize("m,k,n", [(1, 72, 10), (4, 300, 64), (40, 72, 36), (130, 260, 70)])
def test_other_layouts(how, m, k, n):
    rng = np.random.default_rng(m + k)
    x, xt = views(rng, m, k, how)
    w, wt = views(rng, n, k, how)
    r, rt = views(rng, m, n, how)
    plain = [pam.linear_act(gpu(x), gpu(w), None, "silu", gpu(r)), pam.gated_linear(gpu(x), gpu(w))]
    other = [pam.linear_act(xt, wt, None, "silu", rt), pam.gated_linear(xt, wt)]
    size = np.abs(ref.mul(wide(x)[:, :, None], wide(w).T[None])).sum(1).max()
    for p, o in zip(plain, other):                       # (another loader may take another order of the sums)
        assert np.abs(host(p) - host(o)).max() <= 8 * k * EPS23 * (size + np.abs(r).max())


@pytest.mark.gpu
def test_leading_dimensions_and_empty_ones():
    rng = np.random.default_rng(0)
    x, w, r = gpu(normal(rng, 2, 3, 8)), gpu(normal(rng, 6, 8)), gpu(normal(rng, 2, 3, 6))
    assert_same_bits(host(pam.linear_act(x, w, None, "silu", r)).reshape(6, 6), host(pam.linear_act(x.view(6, 8), w, None, "silu", r.view(6, 6))))
    assert pam.gated_linear(x, w).shape == (2, 3, 3)
    assert pam.linear_act(x[0, 0], w).shape == (6,) and pam.gated_linear(x[0, 0], w).shape == (3,)
    assert pam.linear_act(x[:0], w).shape == (0, 3, 6) and pam.gated_linear(x[:, :0], w).shape == (2, 0, 3)
    b = gpu(normal(rng, 6))
    none = torch.zeros(4, 0, device="cuda")
    empty = torch.zeros(6, 0, device="cuda")
    assert_same_bits(host(pam.linear_act(none, empty, b, "relu")), host(b.relu().expand(4, 6)))        # sums over nothing
    assert pam.gated_linear(none, empty).eq(0).all()
    # gradients of nothing
    x0, w0 = torch.zeros(0, 8, device="cuda", requires_grad=True), gpu(normal(rng, 6, 8), True)
    for y in (pam.linear_act(x0, w0, None, "silu"), pam.gated_linear(x0, w0)):
        gx, gw = torch.autograd.grad(y, (x0, w0), torch.zeros_like(y))
        assert gx.shape == (0, 8) and gw.eq(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(9, 7, 6), (33, 40, 10)])
@pytest.mark.parametrize("activation", [None, "silu", "gelu"])
def test_layer_gradients(m, k, n, activation):
    """Approximate gradients against the formulas in 64 bits; exact ones against the function's differences."""
    rng = np.random.default_rng(m + n)
    x, w, b = normal(rng, m, k), normal(rng, 2 * n, k, std=k ** -0.5), normal(rng, 2 * n, std=0.1)
    dy = normal(rng, m, 2 * n), normal(rng, m, n)
    for gated in (False, True):
        ours = pam.gated_linear if gated else pam.linear_act
        name, d = activation, dy[gated]
        t = [gpu(v, True) for v in (x, w, b)]
        got = [host(g) for g in torch.autograd.grad(ours(*t, name, approx_bwd=True), t, gpu(d))]
        z = ref.product(wide(x), wide(w).T)[0] + wide(b)
        if gated:
            a, u = ref.act(z[:, :n], name), z[:, n:]
            dz = np.concatenate([ref.act_grad(z[:, :n], ref.mul(wide(d), u), name), ref.mul(wide(d), a)], 1)
        else:
            dz = ref.act_grad(z, wide(d), name)
        want = [ref.product(dz, wide(w)), ref.product(dz.T, wide(x)), (dz.sum(0), np.abs(dz).sum(0))]
        for g, (v, size) in zip(got, want):
            # (two levels of sums; dz in turn moves with z: slopes of the gradient below 4)
            assert (np.abs(g - v) <= 16 * (k + m + 2 * n) * EPS23 * size.max()).all()
        got = [host(g) for g in torch.autograd.grad(ours(*t, name, approx_bwd=False), t, gpu(d))]
        f = ref.gated if gated else (lambda *a: ref.linear_act(*a, None))
        at = [wide(v) for v in (x, w, b)]
        for i, g in enumerate(got):
            direction = rng.standard_normal(at[i].shape)
            def along(v):
                return (f(*at[:i], v, *at[i + 1:], name) * d).sum()
            want = ref.slope(along, at[i], direction)
            assert abs((g * direction).sum() - want) <= 1e-4 * np.abs(g * direction).sum() + 1e-5


# ---------------------------------------------------------------- rotation

def chain_rotary(x, cos, sin, interleaved, kw):
    rotated = 2 * cos.shape[-1]
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    x1, x2 = (x[..., 0:rotated:2], x[..., 1:rotated:2]) if interleaved else (x[..., :rotated // 2], x[..., rotated // 2:rotated])
    c, s = c.expand_as(x1).contiguous(), s.expand_as(x1).contiguous()
    x1, x2 = x1.contiguous(), x2.contiguous()
    y1, y2 = pam.mul(x1, c, **kw) - pam.mul(x2, s, **kw), pam.mul(x2, c, **kw) + pam.mul(x1, s, **kw)
    head = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((head, x[..., rotated:]), -1)


HEADS = [(2, 5, 3, 1, 64, 64), (1, 70, 4, 2, 128, 128), (3, 1, 2, 2, 80, 40), (2, 9, 1, 1, 18, 18), (1, 3, 5, 2, 7, 2), (2, 4, 2, 1, 256, 64), (1, 2, 1, 1, 600, 600),
         (2, 3, 2, 2, 100, 26), (1, 4, 1, 3, 12, 8), (1, 2, 2, 1, 5, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,rotated", HEADS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_the_chain(batch, tokens, heads, kv, dim, rotated, interleaved):
    rng = np.random.default_rng(dim + tokens)
    angle = rng.uniform(-4, 4, (tokens + 3, rotated // 2))
    cos, sin = gpu(np.cos(angle).astype(np.float32)), gpu(np.sin(angle).astype(np.float32))
    for i, (approx, offset) in enumerate([(True, None), (False, OFF), ((True, False), None)]):
        kw = dict(offset=offset, approx_bwd=approx)
        q, k = gpu(normal(rng, batch, tokens, heads, dim), True), gpu(normal(rng, batch, tokens, kv, dim), True)
        positions = [None, torch.from_numpy(rng.integers(0, tokens + 3, (batch, tokens))).cuda(), torch.from_numpy(rng.integers(0, tokens + 3, tokens)).cuda()][i]
        at = torch.arange(tokens, device="cuda") if positions is None else positions
        yq, yk = pam.rotary(q, k, cos, sin, positions, interleaved=interleaved, **kw)
        for y, x in ((yq, q), (yk, k)):
            same_with_grads(y, chain_rotary(x, cos[at], sin[at], interleaved, kw), [x], gpu(normal(rng, *x.shape)), f"{kw}")


@pytest.mark.gpu
@pytest.mark.parametrize("batch,tokens,heads,kv,dim,rotated", HEADS)
@pytest.mark.parametrize("interleaved", [False, True])
def test_normed_rotation_against_64_bits(batch, tokens, heads, kv, dim, rotated, interleaved):
    rng = np.random.default_rng(dim * 3 + tokens)
    angle = rng.uniform(-4, 4, (tokens, rotated // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    x = [normal(rng, batch, tokens, h, dim, std=s) for h, s in ((heads, 1.0), (kv, 20.0))]
    w = [normal(rng, dim, std=0.1) + np.float32(1.0) for _ in x]
    dy = [normal(rng, *v.shape, std=0.1) for v in x]
    qk, ws = [gpu(v, True) for v in x], [gpu(v, True) for v in w]
    y = pam.rotary(*qk, gpu(cos), gpu(sin), q_weight=ws[0], k_weight=ws[1], interleaved=interleaved, approx_bwd=True)
    grads = torch.autograd.grad(y, qk + ws, [gpu(d) for d in dy])
    exact = torch.autograd.grad(pam.rotary(*qk, gpu(cos), gpu(sin), q_weight=ws[0], k_weight=ws[1], interleaved=interleaved, approx_bwd=False), qk + ws, [gpu(d) for d in dy])
    for i in range(2):
        args = (wide(cos), wide(sin), wide(w[i]), 1e-6, interleaved)
        want = ref.rotary(wide(x[i]), *args)
        dx, dw = ref.rotary_grad(wide(x[i]), wide(dy[i]), *args)
        for got, v in ((y[i], want), (grads[i], dx), (grads[2 + i], dw)):
            assert np.abs(host(got) - v).max() <= 2.0 ** -17 * np.abs(v).max()
        for got, at, f in ((exact[i], wide(x[i]), lambda v: ref.rotary(v, *args)), (exact[2 + i], wide(w[i]), lambda v: ref.rotary(wide(x[i]), wide(cos), wide(sin), v, 1e-6, interleaved))):
            direction = rng.standard_normal(at.shape)
            slope = ref.slope(lambda v: (f(v) * dy[i]).sum(), at, direction * np.abs(at).max())
            terms = host(got) * direction * np.abs(at).max()
            assert abs(terms.sum() - slope) <= 1e-4 * np.abs(terms).sum() + 1e-5


def chain_norm(x, weight, eps, kw):
    """By primitives, the row's sum by torch."""
    d = x.shape[-1]
    total = pam.mul(x, x, **kw).sum(-1, keepdim=True)
    root = pam.pow(pam.div(total, float(d), **kw) + eps, 0.5, **kw)
    return pam.mul(pam.div(x, root.expand_as(x).contiguous(), **kw), weight.expand_as(x).contiguous(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotated", [(64, 64), (80, 40), (18, 10), (256, 64)])
@pytest.mark.parametrize("offset", [None, OFF, 1.4])
def test_normed_rotation_is_the_chain(dim, rotated, offset):
    """Up to the order of the head's sums: 2^-17 of the largest value, approximate gradients."""
    rng = np.random.default_rng(dim)
    kw = dict(offset=offset, approx_bwd=True)
    angle = rng.uniform(-4, 4, (6, rotated // 2))
    cos, sin = gpu(np.cos(angle).astype(np.float32)), gpu(np.sin(angle).astype(np.float32))
    x, w = gpu(normal(rng, 2, 6, 3, dim), True), gpu(normal(rng, dim, std=0.1) + np.float32(1.0), True)
    d = normal(rng, 2, 6, 3, dim, std=0.1)
    d[0, 2], d[1, 4, 1] = 0.0, 0.0                       # a token and a head that the loss leaves out
    y, _ = pam.rotary(x, None, cos, sin, q_weight=w, **kw)
    want = chain_rotary(chain_norm(x, w, 1e-6, kw), cos, sin, False, kw)
    got, expected = [y, *torch.autograd.grad(y, (x, w), gpu(d))], [want, *torch.autograd.grad(want, (x, w), gpu(d))]
    for a, b in zip(got, expected):
        a, b = host(a), host(b)
        assert np.abs(a - b).max() <= 2.0 ** -17 * np.abs(b).max()
    assert not host(got[1])[0, 2].any() and not host(got[1])[1, 4, 1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rotated", [(64, 64), (80, 40), (18, 10), (256, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("approx", [True, False])
def test_heads_do_not_depend_on_each_other(dim, rotated, interleaved, approx):
    """A head with values that take the full definitions changes no bit of its neighbours."""
    rng = np.random.default_rng(dim + rotated)
    angle = rng.uniform(-4, 4, (5, rotated // 2))
    cos, sin = gpu(np.cos(angle).astype(np.float32)), gpu(np.sin(angle).astype(np.float32))
    usual, w, d = normal(rng, 1, 5, 3, dim), gpu(normal(rng, dim, std=0.1) + np.float32(1.0)), gpu(normal(rng, 1, 5, 3, dim, std=0.1))
    odd = usual.copy()
    odd[0, ::2, 1, 0], odd[0, ::2, 1, 1], odd[0, ::2, 1, -1] = 0.0, 1e-39, -3e20
    results = []
    for values in (usual, odd):
        x = gpu(values, True)
        y, _ = pam.rotary(x, None, cos, sin, q_weight=w, interleaved=interleaved, approx_bwd=approx)
        results.append([host(y), host(torch.autograd.grad(y, x, d)[0])])
    for a, b in zip(*results):
        assert_same_bits(a[:, :, ::2], b[:, :, ::2])
        assert_same_bits(a[:, 1::2], b[:, 1::2])


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 260, 20), (8, 1030, 40), (70, 260, 70)])
def test_rows_do_not_depend_on_each_other(m, k, n):
    rng = np.random.default_rng(m)
    usual, w = normal(rng, m, k), gpu(normal(rng, 2 * n, k, std=0.1))
    odd = usual.copy()
    odd[1, 0], odd[1, 5], odd[1, k // 2], odd[1, -1] = 0.0, 1e-39, -3e30, 1e-25
    for call in (lambda x: pam.linear_act(x, w, None, "silu"), lambda x: pam.gated_linear(x, w)):
        a, b = host(call(gpu(usual))), host(call(gpu(odd)))
        assert_same_bits(np.delete(a, 1, 0), np.delete(b, 1, 0))


@pytest.mark.gpu
def test_rotation_of_one_tensor_and_norm_of_the_other():
    rng = np.random.default_rng(4)
    q, k, w = gpu(normal(rng, 2, 3, 2, 16)), gpu(normal(rng, 2, 3, 1, 16)), gpu(normal(rng, 16))
    cos, sin = pam.rotary_tables(8, 16, device="cuda")
    both, kk = pam.rotary(q, k, cos, sin, q_weight=w)
    alone, none = pam.rotary(q, None, cos, sin, q_weight=w)
    assert none is None
    assert_same_bits(host(both), host(alone))
    assert_same_bits(host(kk), host(pam.rotary(k, None, cos, sin)[0]))
    # a head of zeros: its norm is that of eps, its values stay zero
    y, _ = pam.rotary(torch.zeros_like(q), None, cos, sin, q_weight=w)
    assert y.eq(0).all()


@pytest.mark.gpu
def test_positions_outside_the_tables():
    rng = np.random.default_rng(5)
    q = gpu(normal(rng, 1, 4, 2, 20))
    cos, sin = pam.rotary_tables(6, 16, device="cuda")
    y, _ = pam.rotary(q, None, cos, sin, torch.tensor([5, 6, -1, 1 << 40], device="cuda"))
    assert y[0, 0].isfinite().all() and y[0, 1:, :, :16].isnan().all()
    assert_same_bits(host(y[..., 16:]), host(q[..., 16:]))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_rotation_of_views(norm):
    """Heads cut from one projection, heads before tokens, columns that are not contiguous, odd addresses: the values of copies."""
    rng = np.random.default_rng(6)
    cos, sin = pam.rotary_tables(9, 64, device="cuda")
    w = gpu(normal(rng, 64)) if norm else None
    qkv = gpu(normal(rng, 2, 7, 8, 64))
    cases = [qkv[:, :, :5], qkv.transpose(1, 2)[:, :7].clone().transpose(1, 2), gpu(normal(rng, 2, 7, 4, 128))[..., ::2], gpu(normal(rng, 2 * 7 * 3 * 64 + 1))[1:].view(2, 7, 3, 64),
             gpu(normal(rng, 1, 7, 3, 64)).expand(2, 7, 3, 64)]
    for x in cases:
        x = x.detach().requires_grad_(True)
        c = x.detach().clone().contiguous().requires_grad_(True)
        d = gpu(normal(rng, 2, x.shape[2], 7, 64)).transpose(1, 2)
        yx, yc = (pam.rotary(t, None, cos, sin, q_weight=w, approx_bwd=True)[0] for t in (x, c))
        assert_same_bits(host(yx), host(yc))
        assert_same_bits(host(torch.autograd.grad(yx, x, d)[0]), host(torch.autograd.grad(yc, c, d.contiguous())[0]))


@pytest.mark.gpu
def test_rotation_of_nothing():
    cos, sin = pam.rotary_tables(4, 8, device="cuda")
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        y, _ = pam.rotary(q, None, cos, sin, q_weight=w)
        assert y.shape == shape
        dq, dw = torch.autograd.grad(y, (q, w), torch.zeros_like(y))
        assert dq.shape == shape and dw.eq(0).all()


# ---------------------------------------------------------------- clipping

@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [5, 0, 3], [4096, 1, 2047, 2049, 100000], [7] * 200, [300001], [64 * 64] * 97])
@pytest.mark.parametrize("bound", [1e-3, 1.0, 1e6, math.inf, 0.0])
def test_clip_against_64_bits(sizes, bound):
    rng = np.random.default_rng(len(sizes))
    grads = [normal(rng, n, std=0.3) for n in sizes]
    length, want = ref.clip([wide(g) for g in grads], bound)
    n = max(sum(sizes), 1)
    slack = (math.log2(n) + 16) * EPS23              # (sums of at most 16 and a tree of the rest; the root passes on as much)
    tensors = [gpu(g) for g in grads]
    assert abs(float(optim.grad_norm(tensors)) - length) <= 2 * slack * length
    out = [torch.full_like(t, 7.0) for t in tensors]
    kept = [t.clone() for t in tensors]
    norm = optim.clip_grads(tensors, bound, out=out)
    assert norm.shape == () and abs(float(norm) - length) <= 2 * slack * length
    for t, k, o, v in zip(tensors, kept, out, want):
        assert torch.equal(t, k)
        assert (np.abs(host(o) - v) <= 8 * slack * np.abs(v) + 1e-37).all()
    params = [_with_grad(t.cpu()) for t in tensors]
    assert torch.equal(optim.clip_grad_norm_(params, bound), norm)
    for p, o in zip(params, out):
        assert torch.equal(p.grad, o)


@pytest.mark.gpu
def test_clip_is_the_chain():
    """The products are those of pam.mul with the scale, bit for bit, zeros and infinite values among them."""
    rng = np.random.default_rng(9)
    g = normal(rng, 1000)
    g[:3] = [0.0, 1e-40, 1e-30]
    for offset in (None, OFF):
        t = gpu(g)
        out = torch.empty_like(t)
        norm = optim.clip_grads([t], 0.5, out=[out], offset=offset)
        scale = pam.div(torch.full((1,), 0.5, device="cuda"), norm.view(1) + 1e-6, offset=offset).clamp(max=1.0)
        assert_same_bits(host(out), host(pam.mul(t, scale.expand_as(t).contiguous(), offset=offset)))
    for bad in (math.inf, math.nan):
        g[7] = bad
        t = gpu(g)
        assert optim.clip_grads([t], 0.5).isnan() and t.isnan().all()


@pytest.mark.gpu
def test_clip_of_views():
    rng = np.random.default_rng(10)
    flat = gpu(normal(rng, 1001))
    parts = [flat[1:301], flat[301:302], flat[302:1001].view(3, 233)]                 # one buffer, odd addresses
    transposed, gaps = gpu(normal(rng, 6, 10)).t(), gpu(normal(rng, 8, 8))[:, :5]
    tensors = parts + [transposed, gaps]
    copies = [t.clone().contiguous() for t in tensors]
    rest = flat[:1].clone()
    length, want = ref.clip([wide(host(c)) for c in copies], 0.1)
    slack = (math.log2(1100) + 16) * EPS23
    assert abs(float(optim.clip_grads(tensors, 0.1)) - length) <= 2 * slack * length
    for t, v in zip(tensors, want):
        assert (np.abs(host(t) - v) <= 8 * slack * np.abs(v)).all()
    assert torch.equal(flat[:1], rest)
    same = gpu(normal(rng, 6, 10))
    turned = same.t().clone(memory_format=torch.preserve_format)                      # another order in memory
    into = torch.empty(10, 6, device="cuda")
    optim.clip_grads([turned], 0.1, out=[into])
    optim.clip_grads([same], 0.1)
    assert torch.equal(into, same.t())


@pytest.mark.gpu
def test_clip_refuses_shared_outputs():
    flat = torch.ones(100, device="cuda")
    for ins, outs in (([flat, flat], None), ([flat[:60], flat[50:]], None), ([flat[:50]], [flat[10:60]]), ([flat[:10], flat[10:20]], [flat[10:20], flat[30:40]]),
                      ([flat[:10], flat[20:30]], [flat[40:50], flat[45:55]])):
        with pytest.raises(ValueError):
            optim.clip_grads(ins, 1.0, out=outs)
    assert flat.eq(1.0).all()
    assert float(optim.grad_norm([flat, flat])) > 10.0           # (only read)


# ---------------------------------------------------------------- streams, graphs, repeats

def _pass(seed):
    rng = np.random.default_rng(seed)
    x, w, b, r = gpu(normal(rng, 48, 64), True), gpu(normal(rng, 96, 64, std=0.1), True), gpu(normal(rng, 96)), gpu(normal(rng, 48, 96))
    one = gpu(normal(rng, 1, 64))
    cos, sin = pam.rotary_tables(16, 32, device="cuda")
    nw = gpu(normal(rng, 32), True)
    d = gpu(normal(rng, 48, 96))

    def run():
        y = pam.linear_act(x, w, b, "silu", r, approx_bwd=True)
        gx, gw = torch.autograd.grad(y, (x, w), d)
        h = pam.gated_linear(x, w, b, approx_bwd=True)
        hx, hw = torch.autograd.grad(h, (x, w), d[:, :48])
        q, _ = pam.rotary(h.detach().view(3, 16, 1, 48)[..., :32], None, cos, sin, q_weight=nw, approx_bwd=True)
        qw, = torch.autograd.grad(q, nw, q.detach())
        norm = optim.clip_grads([gx, gw, hx, hw, qw], 0.5)
        return [y, h, pam.linear_act(one, w.detach(), b, "gelu"), pam.gated_linear(one, w.detach(), b), q, gx, gw, hx, hw, qw, norm]
    return run


@pytest.mark.gpu
def test_another_stream_and_repeats():
    run = _pass(1)
    want = [t.detach().clone() for t in run()]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = run()
    stream.synchronize()
    for again in (other, run(), run()):
        for a, b in zip(again, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_graph_replays():
    run = _pass(2)
    want = [t.detach().clone() for t in run()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(4):
        for t in out:
            t.detach().fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)
        run()                                            # the program's own work between replays
        torch.cuda.synchronize()
