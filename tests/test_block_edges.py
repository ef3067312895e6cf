"""The decoder block's operators where a call could go wrong without a word: derivatives that no kernel computes, shared memory,
positions that no table has.
"""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import pam_amd as pam
from pam_amd import optim


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
