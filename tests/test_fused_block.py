"""The decoder block with attention in one piece: the operators as a model runs them together."""
import pytest
import torch

from pam_amd.blocks import Attention, DecoderBlock


def _pam():
    import pam_amd as pam
    return pam


def test_the_chain_is_what_a_block_has_by_itself():
    assert not DecoderBlock(32, 4, 2, 8, 48).attention.fused and DecoderBlock(32, 4, 2, 8, 48, fused=True).attention.fused


@pytest.mark.gpu
@pytest.mark.parametrize("approx", [True, False])
def test_the_block_is_its_operators(approx):
    """The module's result and gradients are those of the operators called one by one, bit for bit."""
    pam = _pam()
    torch.manual_seed(0)
    layer = Attention(32, 4, 2, 16, fused=True, approx_bwd=approx).cuda()
    cos, sin = pam.rotary_tables(30, 16, device="cuda")
    x = torch.randn(2, 30, 32, device="cuda", requires_grad=True)
    got = layer(x, cos, sin)

    def by_hand():
        kw = dict(approx_bwd=approx)
        qkv = pam.linear_act(layer.norm(x), layer.qkv, **kw).view(2, 30, -1, 16)
        q, k, v = qkv.split((4, 2, 2), 2)
        q, k = pam.rotary(q, k, cos, sin, q_weight=layer.q_weight, k_weight=layer.k_weight, **kw)
        return pam.linear_act(pam.attention(q, k, v, **kw).reshape(2, 30, -1), layer.out, None, None, x, **kw)
    want = by_hand()
    assert torch.equal(got, want)
    dy = torch.randn_like(got)
    leaves = [x, layer.qkv, layer.q_weight, layer.k_weight, layer.out]
    for g, w in zip(torch.autograd.grad(got, leaves, dy), torch.autograd.grad(want, leaves, dy)):
        assert torch.equal(g, w) and g.isfinite().all() and g.abs().max() > 0


@pytest.mark.gpu
def test_a_cached_block_continues():
    pam = _pam()
    torch.manual_seed(1)
    block = DecoderBlock(32, 4, 2, 16, 48, fused=True).cuda()
    cos, sin = pam.rotary_tables(40, 16, device="cuda")
    x = torch.randn(3, 40, 32, device="cuda")
    with torch.no_grad():
        whole, cache = block(x, cos, sin), {}
        parts = [block(x[:, a:b], cos, sin, cache) for a, b in [(0, 17), (17, 20)] + [(i, i + 1) for i in range(20, 40)]]
    # the same values in other orders of sums of at most 64 terms, through two residual products each twice as sensitive
    assert (torch.cat(parts, 1) - whole).abs().max() <= 2.0 ** -24 * 64 * 16 * whole.abs().max()
