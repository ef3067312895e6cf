"""The decoder block's operators where a call could go wrong without a word: derivatives that no kernel computes, shared memory,
positions that no table has.
"""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import pam_amd as pam
import _block_ref as ref
from pam_amd import optim
from pam_amd.blocks import Attention


def ones(*shape):
    return torch.ones(*shape, device="cuda")


# ---------------------------------------------------------------- derivatives

@pytest.mark.gpu
@pytest.mark.parametrize("recording", [True, False])
def test_forward_mode_is_refused(recording):
    """Not answered by a result without a tangent, in any argument; calls beside it are not concerned."""
    x, w, b, r, q, n = ones(3, 4), ones(6, 4), ones(6), ones(3, 6), ones(1, 3, 2, 8), ones(8)
    cos, sin = pam.rotary_tables(4, 8, device="cuda")
    with forward_ad.dual_level(), torch.set_grad_enabled(recording):
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: pam.linear_act(dual(x), w), lambda: pam.linear_act(x, dual(w), b, "silu", r), lambda: pam.linear_act(x, w, dual(b)),
                     lambda: pam.linear_act(x, w, None, None, dual(r)), lambda: pam.linear_act(dual(ones(2, 3, 4)), w), lambda: pam.gated_linear(dual(x), w),
                     lambda: pam.gated_linear(x, dual(w)), lambda: pam.gated_linear(x, w, dual(b)), lambda: pam.rotary(dual(q), None, cos, sin),
                     lambda: pam.rotary(q, dual(q), cos, sin), lambda: pam.rotary(q, None, dual(cos), sin), lambda: pam.rotary(q, None, cos, sin, q_weight=dual(n)),
                     lambda: pam.rotary(q, q, cos, sin, k_weight=dual(n))):
            with pytest.raises(NotImplementedError):
                call()
        assert pam.linear_act(x, w).shape == (3, 6) and pam.rotary(q, None, cos, sin)[0].shape == q.shape


def test_clipping_is_not_traced():
    for call in (lambda x: optim.grad_norm([x]), lambda x: optim.clip_grads([x], 1.0), lambda x: optim.clip_grad_norm_([_with_grad(x)], 1.0)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(call, (torch.ones(3),), check_trace=False)


def _with_grad(g):
    p = torch.nn.Parameter(torch.zeros_like(g))
    p.grad = g.detach()
    return p


@pytest.mark.gpu
def test_the_norm_is_no_constant_of_a_graph():
    """The norm of gradients that carry a graph is refused where it would silently leave that graph; clipping such gradients records
    nothing, as torch.nn.utils.clip_grad_norm_ does not."""
    w = ones(5).requires_grad_()
    grad, = torch.autograd.grad((w ** 3).sum(), w, create_graph=True)
    assert grad.requires_grad
    for t in (grad, w):
        with pytest.raises(RuntimeError, match="no gradient"):
            optim.grad_norm([ones(2), t])
        with torch.no_grad():
            assert float(optim.grad_norm([t])) > 0.0
        assert not optim.grad_norm(t.detach()).requires_grad
    out = torch.empty_like(grad, requires_grad=False)
    assert not optim.clip_grads([grad], 0.5, out=[out]).requires_grad and float(out[0]) < 3.0
    w.grad = grad
    assert not optim.clip_grad_norm_([w], 0.5, error_if_nonfinite=True).requires_grad
    with forward_ad.dual_level():
        g = forward_ad.make_dual(ones(3), ones(3))
        for call in (lambda: optim.grad_norm([ones(3), g]), lambda: optim.clip_grads([g], 1.0, out=[ones(3)])):
            with pytest.raises(NotImplementedError):
                call()


@pytest.mark.gpu
def test_clipped_tensors_count_as_modified():
    """A graph that has saved a tensor is not run on the clipped values of it."""
    def graph(saved):
        return (saved * ones(4).requires_grad_()).sum()
    g, out, kept = 3 * ones(4), ones(4), 3 * ones(4)
    sums = [graph(t) for t in (g, out, kept)]
    optim.clip_grads([g], 0.5)
    optim.clip_grads([kept], 0.5, out=[out])
    for y in sums[:2]:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    optim.grad_norm([kept])
    sums[2].backward()                                   # only read
    with torch.inference_mode():
        t = 3 * ones(4)
        optim.clip_grads([t], 0.5)
        assert float(t[0]) < 3.0


# ---------------------------------------------------------------- memory that outputs share

@pytest.mark.gpu
def test_clip_refuses_shared_outputs_of_other_strides():
    """Outputs that are written by a copy are looked at where they are, not where the copy comes from."""
    a, b, o = ones(10, 10), ones(10, 10), torch.full((10, 10), 7.0, device="cuda")
    wide = torch.full((4, 12), 7.0, device="cuda")
    for ins, outs in (([a, b], [o.t(), o.t()]), ([a, b], [o.t(), o]), ([a, b], [o, o.t()]), ([a[:4, :5], b[:4, :5]], [wide[:, :5], wide[:, 4:9]]),
                      ([a[0, :4]], [o[0, :1].expand(4)]), ([a[:3, :3]], [torch.as_strided(o, (3, 3), (2, 1))])):
        with pytest.raises(ValueError):
            optim.clip_grads(ins, 1.0, out=outs)
    row = torch.full((1, 4), 3.0, device="cuda")
    with pytest.raises(ValueError):
        optim.clip_grads([b, row.expand(5, 4)], 1.0)                 # in place, all rows one
    assert o.eq(7.0).all() and wide.eq(7.0).all() and b.eq(1.0).all() and row.eq(3.0).all()          # and nothing written
    # columns and halves of one buffer share its span, not its values
    optim.clip_grads([a[:4, :6], b[:4, :6]], 1.0, out=[wide[:, ::2], wide[:, 1::2]])
    assert wide.eq(wide[0, 0]).all() and float(wide[0, 0]) < 1.0
    wide.fill_(1.0)
    optim.clip_grads([wide[:, :6], wide[:, 6:]], 1.0)
    assert wide.eq(wide[0, 0]).all() and float(wide[0, 0]) < 1.0


@pytest.mark.gpu
def test_shared_values_are_found_exactly():
    """Drawn views of one buffer, their addresses written out: refused if and only if one address is there twice."""
    rng = np.random.default_rng(11)
    flat, refused = torch.zeros(400, device="cuda"), 0
    for _ in range(400):
        views, addresses = [], []
        for _ in range(2):
            sizes, strides = rng.integers(1, 5, 2), rng.integers(1, 13, 2)
            start = int(rng.integers(0, 60))
            views.append(torch.as_strided(flat, tuple(int(n) for n in sizes), tuple(int(n) for n in strides), start))
            addresses += [start + i * int(strides[0]) + j * int(strides[1]) for i in range(sizes[0]) for j in range(sizes[1])]
        grads = [ones(*v.shape) for v in views]
        if len(set(addresses)) < len(addresses):
            refused += 1
            with pytest.raises(ValueError):
                optim.clip_grads(grads, 0.5, out=views)
        else:
            flat.zero_()
            optim.clip_grads(grads, 0.5, out=views)
            assert all(v.eq(views[0].flatten()[0]).all() for v in views) and int(flat.ne(0).sum()) == len(addresses)
    assert 50 < refused < 350


# ---------------------------------------------------------------- positions that no table has

@pytest.mark.gpu
def test_decoding_past_the_tables_is_refused():
    """The rotation makes such positions NaN; the module knows how many tokens its cache has, and says so."""
    attention = Attention(16, 2, 1, 8).cuda()
    cos, sin = pam.rotary_tables(6, 8, device="cuda")
    with torch.no_grad():
        cache = {}
        for tokens in (4, 1, 1):
            assert attention(ones(2, tokens, 16), cos, sin, cache).isfinite().all()
        for tokens, kept in ((1, cache), (7, None), (3, {k: v[:, :4] for k, v in cache.items()})):
            with pytest.raises(ValueError):
                attention(ones(2, tokens, 16), cos, sin, kept)
    assert cache["k"].shape[1] == 6


# ---------------------------------------------------------------- more work than one launch counts

@pytest.mark.gpu
@pytest.mark.parametrize("dim", [2, 18])
def test_rotation_of_more_heads_than_one_launch_takes(dim):
    """2^26 heads of a size that takes a wavefront each are 2^32 work-items.  The input is one token, expanded."""
    tokens, heads = (1 << 20) + 1, 64
    cos, sin = pam.rotary_tables(4, dim, device="cuda")
    generator = torch.Generator("cuda").manual_seed(1)
    one, d = (torch.randn(1, 1, heads, dim, device="cuda", generator=generator) for _ in range(2))
    x = one.clone().requires_grad_()
    k = torch.randn(1, 1, 2, dim, device="cuda", generator=generator)
    first = torch.full((1,), 3, device="cuda")
    want, want_k = pam.rotary(x, k, cos, sin, first, approx_bwd=True)
    dx, = torch.autograd.grad(want, x, d)
    many = one.expand(1, tokens, heads, dim).requires_grad_()
    y, yk = pam.rotary(many, k.expand(1, tokens, 2, dim), cos, sin, first.expand(tokens), approx_bwd=True)
    assert y.eq(want).all() and yk.eq(want_k).all()
    g, = torch.autograd.grad(y, many, d.expand(1, tokens, heads, dim))
    assert g.eq(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1 << 27, (1 << 27) + 8, (1 << 28) + 5])
def test_one_row_through_more_weights_than_one_launch_takes(rows):
    x, w = torch.full((1, 1), 1.5, device="cuda"), torch.full((1, 1), 1.25, device="cuda")
    want = float(pam.mul(x, w))
    y = pam.linear_act(x, w.expand(rows, 1))
    assert y.shape == (1, rows) and y.eq(want).all()
    h = pam.gated_linear(x, w.expand(rows // 2 * 2, 1), activation=None)
    assert h.shape == (1, rows // 2) and h.eq(float(pam.mul(y[:, :1], y[:, :1]))).all()


@pytest.mark.gpu
def test_norm_of_more_values_than_one_launch_takes():
    """33 times 2^31 values in one table, read from one tensor."""
    t = torch.full((1 << 31,), 2.0 ** -10, device="cuda")
    total = 33 * 2.0 ** 31 * 2.0 ** -20                  # (sums of equal powers of two, added in pairs: exact)
    assert float(optim.grad_norm([t] * 33)) == float(ref.sqrt(np.array(total)))
