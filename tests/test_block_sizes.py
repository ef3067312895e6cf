"""The decoder block's operators at the sizes of real models, which other ways through the kernels serve than small ones: many rows of
weights for few tokens, heads in many turns of the resident work-groups, gradients in many tables.

Bounds as in test_block_ops: a sum of K PAM terms in float32 is off by at most K 2^-23 times the sum of the terms' magnitudes; sums of whole
numbers are exact.
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


def product64(x, w):
    """sum over k of x[m, k] (*) w[n, k] in double precision, on the bit patterns, and the sum of the terms' magnitudes."""
    bias, magnitude, sign = 1023 << 52, (1 << 63) - 1, -(1 << 63)
    xb, wb = x.double().view(torch.int64), w.double().view(torch.int64)
    sums, sizes = [], []
    for i in range(x.shape[0]):
        bits = (xb[i] & magnitude) - bias + (wb & magnitude)
        terms = torch.where((x[i] == 0) | (w == 0), 0, bits | ((xb[i] ^ wb) & sign)).view(torch.float64)
        sums.append(terms.sum(1)); sizes.append(terms.abs().sum(1))
    return torch.stack(sums), torch.stack(sizes)


# ---------------------------------------------------------------- few rows through many weights

@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 17, 24])
@pytest.mark.parametrize("rows,k", [(16390, 70), (8198, 300), (8194, 1100), (4098, 2052)])
def test_few_rows_through_many_weights(m, rows, k):
    """Every number of a wavefront's rows of weights and of wavefronts along k; rows past whole groups; zeros and values beyond the window."""
    generator = torch.Generator("cuda").manual_seed(m + rows)
    x = torch.randn(m, k, device="cuda", generator=generator)
    w = torch.randn(rows, k, device="cuda", generator=generator) * k ** -0.5
    bias, residual = torch.randn(rows, device="cuda", generator=generator), torch.randn(m, rows, device="cuda", generator=generator)
    x[m // 2, k // 3], x[0, 5] = 0.0, 1e-39
    w[7, 2], w[rows - 1, k - 1], w[rows // 2, 64:66] = 0.0, 1e-42, torch.tensor([1e25, -0.0], device="cuda")
    z, size = product64(x, w)
    z = z + bias.double()
    slack = size * (k + 2) * EPS23 + z.abs() * EPS23 + 1e-30
    want = z + residual.double()
    got = pam.linear_act(x, w, bias, None, residual).double()
    assert ((got - want).abs() <= slack + want.abs() * EPS23).all()
    f = rows // 2
    got = pam.gated_linear(x, w, bias, "relu").double()
    a, u = z[:, :f].clamp(min=0.0), z[:, f:]
    want = torch.from_numpy(ref.mul(a.cpu().numpy(), u.cpu().numpy())).cuda()
    assert ((got - want).abs() <= 1.05 * 2.0 * (slack[:, :f] * u.abs() + slack[:, f:] * a) + want.abs() * EPS23 + 1e-30).all()


# ---------------------------------------------------------------- heads in many turns

def tables(positions, half):
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * 0.37 ** torch.arange(half, dtype=torch.float64)
    return angle.cos().float().cuda(), angle.sin().float().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("dim,tokens,heads", [(64, 7001, 15), (128, 40001, 14), (80, 9001, 9)])
def test_heads_of_many_turns(approx, dim, tokens, heads):
    """A head's gradient is what it is in a call of one turn, whichever turn it falls into, heads that take the full definitions among them."""
    generator = torch.Generator("cuda").manual_seed(dim)
    cos, sin = tables(50, dim // 4)
    positions = torch.randint(0, 50, (tokens,), device="cuda", generator=generator)
    q, k, dq, dk = (torch.randn(1, tokens, n, dim, device="cuda", generator=generator) for n in (heads, 2, heads, 2))
    for t in (q, dq):                                    # odd ones in a few turns, and tokens that a loss leaves out
        for at in (3, tokens // 3, 2 * tokens // 3 + 1, tokens - 1):
            t[0, at, at % heads, 1] = 1e-39
    q[0, tokens // 2, 0, 0], dq[0, tokens // 4] = 0.0, 0.0
    wq, wk = (1.0 + 0.1 * torch.randn(dim, device="cuda", generator=generator) for _ in range(2))

    def gradients(a, b):
        leaves = [t[:, a:b].clone().requires_grad_() for t in (q, k)] + [w.clone().requires_grad_() for w in (wq, wk)]
        y = pam.rotary(leaves[0], leaves[1], cos, sin, positions[a:b], q_weight=leaves[2], k_weight=leaves[3], approx_bwd=approx)
        return torch.autograd.grad(y, leaves, (dq[:, a:b], dk[:, a:b]))
    whole = gradients(0, tokens)
    step = 1000
    for a in list(range(0, tokens, step))[::max(1, tokens // step // 9)] + [tokens - step]:
        part = gradients(a, min(a + step, tokens))
        for g, p in zip(whole, part[:2]):
            assert torch.equal(g[:, a:a + step].view(torch.int32), p.view(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("tokens,heads", [(7001, 15), (70003, 16)])
def test_weights_gradients_of_many_turns(approx, tokens, heads):
    """Heads of ones and minus ones are their own norm, and without a rotation the weight's gradient is a sum of whole numbers: exact, so that
    a head left out or counted twice shows."""
    dim = 64
    generator = torch.Generator("cuda").manual_seed(tokens)
    cos, sin = torch.ones(1, dim // 2, device="cuda"), torch.zeros(1, dim // 2, device="cuda")
    at = torch.zeros(1, dtype=torch.int64, device="cuda").expand(tokens)
    q, k = (torch.randint(0, 2, (1, tokens, n, dim), device="cuda", generator=generator).float() * 2.0 - 1.0 for n in (heads, 3))
    dq, dk = (torch.randint(1, 9, t.shape, device="cuda", generator=generator).float() for t in (q, k))
    for d in (dq, dk):                                   # (these heads go by the checked functions)
        for token in (0, 11, tokens // 2, tokens // 2 + 1, tokens - 1):
            d[0, token, token % d.shape[2], 5] = 1e-39
    leaves = [q.requires_grad_(), k.requires_grad_()] + [torch.ones(dim, device="cuda", requires_grad=True) for _ in range(2)]
    y = pam.rotary(*leaves[:2], cos, sin, at, q_weight=leaves[2], k_weight=leaves[3], eps=0.0, approx_bwd=approx)
    assert torch.equal(y[0], q) and torch.equal(y[1], k)
    grads = torch.autograd.grad(y, leaves, (dq, dk))
    for x, d, g in ((q, dq, grads[2]), (k, dk, grads[3])):
        want = (x.detach().double() * d.double()).sum((0, 1, 2))
        assert ((g.double() - want).abs() <= 1e-30).all()


# ---------------------------------------------------------------- gradients in many tables

@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[5_000_001], [4096 * 700, 1, 4096 * 700 - 1], [1 + 37 * (i % 200) for i in range(520)], [30_000 + i for i in range(180)]])
@pytest.mark.parametrize("bound", [0.5, 1e9])
def test_clip_of_many(sizes, bound):
    """More than 1024 work-groups' sums, more tensors than one table of either pass holds."""
    rng = np.random.default_rng(len(sizes))
    flat = (rng.standard_normal(sum(sizes)) * 0.01).astype(np.float32)
    flat[::1009] = 0.0
    flat[5::100003] = 1e-39
    length, (want,) = ref.clip([flat.astype(np.float64)], bound)
    slack = (math.log2(flat.size) + 16) * EPS23
    tensors = list(torch.from_numpy(flat).cuda().split(sizes))
    assert abs(float(optim.grad_norm(tensors)) - length) <= 2 * slack * length
    out = torch.full((flat.size,), 7.0, device="cuda")
    norm = optim.clip_grads(tensors, bound, out=list(out.split(sizes)))
    assert abs(float(norm) - length) <= 2 * slack * length
    assert (np.abs(out.cpu().numpy() - want) <= 8 * slack * np.abs(want) + 1e-37).all()
    assert torch.equal(optim.clip_grads(tensors, bound), norm)                         # in place
    assert_same_bits(torch.cat(tensors).cpu().numpy(), out.cpu().numpy())
