"""The decoder block's operators where a call could go wrong without a word: derivatives that no kernel computes, shared memory,
positions that no table has.
"""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import pam_amd as pam


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
