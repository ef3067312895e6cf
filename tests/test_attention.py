"""pam.attention against its definition in 64 bits, its masks, its gradients and its refusals."""
import numpy as np
import pytest
import torch

import _attention_ref as ref

gpu = pytest.mark.gpu


def _host():
    import pam_amd as pam
    return pam


def _inputs(seed, batch, tokens, keys, heads, kv_heads, dim, spread=1.0):
    rng = np.random.RandomState(seed)
    q, k, v, dy = (rng.standard_normal(s).astype(np.float32) for s in ((batch, tokens, heads, dim), (batch, keys, kv_heads, dim), (batch, keys, kv_heads, dim),
                                                                       (batch, tokens, heads, dim)))
    return q * np.float32(spread), k, v, dy * np.float32(1e-2)


def _check(got, want, off, what):
    got = got.detach().cpu().double().numpy()
    assert np.isfinite(got).all(), f"{what}: {np.count_nonzero(~np.isfinite(got))} values that are none"
    bad = np.abs(got - want) > off
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / np.maximum(off, 1e-300)):.2f} times the bound"


def _cuda(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _run(q, k, v, dy, masks, approx=True):
    pam = _host()
    leaves = [_cuda(x).requires_grad_(dy is not None) for x in (q, k, v)]
    on = {n: _cuda(x) if isinstance(x, np.ndarray) else x for n, x in masks.items()}
    y = pam.attention(*leaves, **on, approx_bwd=approx)
    return (y, torch.autograd.grad(y, leaves, _cuda(dy))) if dy is not None else (y, None)


def _compare(shape, masks, seed=0, approx=True, train=True, spread=1.0, change=None, borders=False):
    q, k, v, dy = _inputs(seed, *shape, spread=spread)
    if change:
        change(q, k, v, dy)
    y, grads = _run(q, k, v, dy if train else None, masks, approx)
    want = ref.attention(q, k, v, dy if train else None, approx, borders=borders, **masks)
    _check(y, want[0], want[1], "y")
    for name, got, w, off in zip("qkv", grads or (), *(want[2:] if train else ((), ()))):
        _check(got, w, off, "d" + name)
    return y, grads, want


SHAPES = [  # batch, tokens, keys, heads, kv heads, dim
    (1, 1, 1, 1, 1, 4), (2, 3, 3, 2, 1, 18), (1, 70, 70, 3, 3, 64), (2, 33, 65, 4, 2, 16), (1, 129, 200, 2, 2, 100), (1, 5, 130, 6, 2, 80), (1, 64, 64, 2, 1, 128),
    (1, 4, 4, 2, 2, 256), (1, 3, 5, 2, 1, 130), (1, 5, 5, 2, 2, 192), (1, 70, 300, 1, 1, 112), (3, 300, 300, 4, 1, 20), (1, 40, 40, 1, 1, 96), (1, 67, 67, 2, 2, 256), (1, 50, 50, 2, 1, 130), (1, 17, 17, 1, 1, 1), (1, 33, 70, 3, 1, 48), (1, 20, 9, 2, 2, 32),
]


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_result_and_gradients(shape, causal):
    _compare(shape, dict(causal=causal), seed=sum(shape))


MASKS = {
    "window": dict(window=7), "window_both_ways": dict(window=5, causal=False), "window_of_one": dict(window=1), "prefix": dict(prefix=np.array([11, 0])),
    "prefix_and_window": dict(prefix=np.array([3, 200]), window=4), "slopes": dict(slopes=np.array([0.5, 0.03, 0.0, 1.7], np.float32)),
    "cap": dict(cap=3.0), "cap_and_slopes": dict(cap=30.0, slopes=np.array([0.5, 0.25, 0.1, 0.02], np.float32), causal=False),
    "scale": dict(scale=0.031), "negative_slopes": dict(slopes=np.array([-0.1, 0.1, -1.0, 0.0], np.float32)),
}


@gpu
@pytest.mark.parametrize("name", MASKS)
@pytest.mark.parametrize("shape", [(2, 77, 90, 4, 2, 32), (2, 130, 130, 4, 1, 80)], ids=["prompt", "whole"])
def test_masks_and_scores(shape, name):
    _compare(shape, MASKS[name], seed=5)


def _documents(batch, keys, seed):
    rng = np.random.RandomState(seed)
    out = np.zeros((batch, keys), np.int64)
    for b in range(batch):
        cuts = np.sort(rng.choice(np.arange(1, keys), 4, replace=False))
        out[b] = np.array([7, 3, 1 << 40, -1, 3])[np.searchsorted(cuts, np.arange(keys), side="right")]
    return out


@gpu
@pytest.mark.parametrize("more", [{}, dict(causal=False), dict(prefix=np.array([40, 90])), dict(window=9)], ids=["causal", "all", "prefix", "window"])
def test_documents(more):
    shape = (2, 150, 190, 4, 2, 48)
    documents = _documents(2, 190, 3)
    y, grads, _ = _compare(shape, dict(documents=documents, **more), seed=8)
    padding = torch.from_numpy(documents < 0).cuda()
    assert (documents < 0).any()
    assert (y[padding[:, 40:]] == 0).all() and (grads[0][padding[:, 40:]] == 0).all()
    assert (grads[1][padding] == 0).all() and (grads[2][padding] == 0).all()


@gpu
def test_rows_that_see_nothing():
    """More queries than keys: the first ones stand before all keys."""
    y, grads, _ = _compare((1, 90, 30, 2, 1, 64), {}, seed=2)
    assert (y[:, :60] == 0).all() and (grads[0][:, :60] == 0).all()
    pam = _host()
    q, k = torch.randn(1, 3, 2, 8, device="cuda", requires_grad=True), torch.randn(1, 0, 1, 8, device="cuda", requires_grad=True)
    y = pam.attention(q, k, k, approx_bwd=True)
    assert (y == 0).all()
    dq, dk = torch.autograd.grad(y, (q, k), torch.ones_like(y))
    assert (dq == 0).all() and dk.shape == k.shape
    empty = torch.randn(2, 0, 4, 8, device="cuda", requires_grad=True)
    k = torch.randn(2, 5, 2, 8, device="cuda", requires_grad=True)
    y = pam.attention(empty, k, k, approx_bwd=True)
    assert y.shape == empty.shape
    assert (torch.autograd.grad(y, k, torch.ones_like(y))[0] == 0).all()


@gpu
@pytest.mark.parametrize("dim", [1, 16, 18, 64, 100, 128, 130, 256])
def test_rows_of_a_single_key_give_no_gradient(dim):
    """Their weight is one whatever the score is: nothing for queries and keys, to the bit, and dy for the value."""
    for seed, shape, more in ((1, (2, 1, 1, 4, 2, dim), {}), (2, (1, 70, 70, 4, 2, dim), dict(window=1)), (3, (1, 1, 33, 2, 1, dim), dict(window=1, cap=9.0))):
        q, k, v, dy = _inputs(seed, *shape)
        y, (dq, dk, dv) = _run(q, k, v, dy, more)
        assert (dq == 0).all() and (dk == 0).all() and (dv[:, -1] != 0).all()
        assert torch.equal(y, _cuda(v)[:, -shape[1]:].repeat_interleave(shape[3] // shape[4], 2))


@gpu
@pytest.mark.parametrize("what", ["zero_row", "zero_values", "zero_queries", "small", "large", "one_zero"])
def test_values_out_of_the_ordinary(what):
    def change(q, k, v, dy):
        if what == "zero_row":
            k[:, 5] = 0; v[:, 9] = 0; q[:, 7] = 0; dy[:, 11] = 0
        elif what == "zero_values":
            for i, x in enumerate((q, k, v, dy)):
                x.reshape(-1)[i::37] = 0
        elif what == "zero_queries":
            q[:, 20:40] = 0; dy[:, 33:] = 0
        elif what == "small":
            v *= np.float32(1e-25); dy[:, :20] *= np.float32(1e-18)
        elif what == "large":
            v[:, 3] *= np.float32(1e14); k[:, 8] *= np.float32(1e-20); dy *= np.float32(1e12)
        else:
            q.reshape(-1)[100] = 0; k.reshape(-1)[200] = 0; v.reshape(-1)[300] = 0; dy.reshape(-1)[400] = 0
    _compare((1, 70, 70, 2, 1, 64), {}, seed=3, change=change)


def _odd(what):
    def change(q, k, v, dy):
        rng = np.random.RandomState(8)
        if what == "zeros_in_keys":
            k[rng.random_sample(k.shape) < 0.05] = 0
        elif what == "zeros_in_values":
            v[rng.random_sample(v.shape) < 0.3] = 0
        elif what == "zeros_everywhere":
            for x in (q, k, v, dy):
                x[rng.random_sample(x.shape) < 0.1] = 0
        elif what == "zero_queries_large_keys":                       # (a zero times anything is zero)
            q[..., : q.shape[3] // 2] = 0; k[..., : k.shape[3] // 2] *= np.float32(2.0 ** 100)
        elif what == "no_gradient_for_some":
            dy[:, ::3] = 0
        elif what == "powers":                                        # (2^-86 stands for zero in a lane)
            q[:] = np.float32(2.0 ** -86) * np.sign(q); k[:] = np.float32(2.0 ** 85) * np.sign(k)
    return change


@gpu
@pytest.mark.parametrize("approx", [True, False])
@pytest.mark.parametrize("what", ["zeros_in_keys", "zeros_in_values", "zeros_everywhere", "zero_queries_large_keys", "no_gradient_for_some", "powers"])
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_zeros_and_powers_in_either_side(dim, what, approx):
    _compare((1, 45, 70, 2, 1, dim), {}, seed=dim, approx=approx, change=_odd(what), borders=True, train=what not in ("zero_queries_large_keys", "powers"))


@gpu
def test_sizes_of_nothing():
    pam = _host()
    def t(*shape):
        return torch.randn(*shape, device="cuda")
    assert pam.attention(t(0, 3, 2, 8), t(0, 3, 1, 8), t(0, 3, 1, 8)).shape == (0, 3, 2, 8)
    assert pam.attention(t(2, 0, 2, 8), t(2, 3, 1, 8), t(2, 3, 1, 8)).shape == (2, 0, 2, 8)
    assert (pam.attention(t(2, 3, 2, 8), t(2, 0, 1, 8), t(2, 0, 1, 8)) == 0).all()
    assert pam.attention(t(2, 3, 0, 8), t(2, 3, 0, 8), t(2, 3, 0, 8)).shape == (2, 3, 0, 8)
    for q, k in (((2, 3, 2, 8), (2, 0, 1, 8)), ((2, 0, 2, 8), (2, 3, 1, 8)), ((0, 3, 2, 8), (0, 3, 1, 8))):
        leaves = [t(*s).requires_grad_() for s in (q, k, k)]
        y = pam.attention(*leaves, approx_bwd=True)
        for g, leaf in zip(torch.autograd.grad(y, leaves, torch.ones_like(y)), leaves):
            assert g.shape == leaf.shape and (g == 0).all()


@gpu
def test_shared_and_broadcast_inputs():
    """One tensor as keys and values, one batch entry for all, and odd numbers of heads that share a key's."""
    pam = _host()
    q, k = torch.randn(3, 20, 7, 36, device="cuda", requires_grad=True), torch.randn(1, 20, 1, 36, device="cuda", requires_grad=True)
    dy = torch.randn(3, 20, 7, 36, device="cuda")
    kb = k.expand(3, -1, -1, -1)
    got = torch.autograd.grad(pam.attention(q, kb, kb, approx_bwd=True), (q, k), dy)
    kc, vc = (k.detach().repeat(3, 1, 1, 1).requires_grad_() for _ in range(2))
    want = torch.autograd.grad(pam.attention(q, kc, vc, approx_bwd=True), (q, kc, vc), dy)
    assert torch.equal(got[0], want[0]) and got[1].shape == k.shape
    sum_of = (want[1].double() + want[2].double()).sum(0, keepdim=True)
    size = (want[1].abs() + want[2].abs()).sum(0, keepdim=True).double()
    assert ((got[1] - sum_of).abs() <= 6 * 2.0 ** -24 * size).all()       # (a sum of six)


@gpu
def test_scores_far_apart():
    """Weights below 2^-62 of the largest, and a maximum that rises along the keys."""
    def change(q, k, v, dy):
        q[:] = np.abs(q); k[:] = np.abs(k) * np.linspace(-40, 40, k.shape[1], dtype=np.float32)[None, :, None, None]
    _compare((1, 300, 300, 1, 1, 32), dict(causal=False), seed=4, change=change)


@gpu
@pytest.mark.parametrize("where", ["q", "k", "v", "k_unseen", "v_unseen"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_no_numbers(where, value):
    """A value that is no number reaches the queries that see it and no others, and nothing at all from masked places."""
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(1, 1, 40, 40, 2, 1, 32))
    clean = pam.attention(q, k, v)
    documents = torch.zeros(1, 40, dtype=torch.int64, device="cuda")
    if where.endswith("unseen"):
        documents[:, 20] = -1
        clean = pam.attention(q, k, v, documents=documents)
    t = dict(q=q, k=k, v=v)[where[0]]
    t[0, 20, 0, 3] = value
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    y = pam.attention(*leaves, documents=documents, approx_bwd=True)
    grads = torch.autograd.grad(y, leaves, dy)
    if where.endswith("unseen"):
        assert torch.equal(y, clean) and all(torch.isfinite(g).all() for g in grads)
    elif where == "v":
        assert y[0, 20:, :, 3].isnan().all() and torch.equal(y[0, :20], clean[0, :20])
        assert torch.isfinite(y[..., 4:]).all() and grads[0][0, 20:].isnan().all()
    else:
        bad = y[0, 20, 0].isnan() if where == "q" else y[0, 20:].isnan()
        assert bad.all() and torch.equal(y[0, :20], clean[0, :20])
        assert (grads[0][0, 20, 0] if where == "q" else grads[0][0, 20:]).isnan().all()
        assert grads[1][0, :20].isnan().all() and grads[2][0, :20].isnan().all()


@gpu
def test_strides_and_parts_of_a_product():
    """Queries, keys and values as views of one projection, and transposed heads: the same numbers as copies."""
    pam = _host()
    qkv = torch.randn(2, 50, 8, 24, device="cuda")
    q, k, v = qkv.split((4, 2, 2), 2)
    want = pam.attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(pam.attention(q, k, v), want)
    by_head = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(pam.attention(*by_head), want)
    odd = torch.empty(2 * 50 * 8 * 24 + 1, device="cuda")[1:].view(2, 50, 8, 24)
    odd.copy_(qkv)
    assert torch.equal(pam.attention(*odd.split((4, 2, 2), 2)), want)
    strided = torch.empty(2, 50, 8, 24, 2, device="cuda")[..., 0]
    strided.copy_(qkv)
    assert torch.equal(pam.attention(*strided.split((4, 2, 2), 2)), want)


@gpu
def test_a_long_row_of_keys():
    """Chains of sums end after 1024 terms and are added up in memory, and the work on few queries is cut along the keys."""
    _compare((1, 3, 5000, 2, 1, 20), {}, seed=6)
    _compare((1, 700, 2300, 8, 8, 16), dict(causal=False), seed=7, train=False)


@gpu
def test_offset_moves_every_product():
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(2, 1, 20, 20, 2, 2, 16))
    off = 1.0552

    def product(a, b):
        return pam.mul(a.unsqueeze(-2), b.unsqueeze(-3), offset=off).double().sum(-1)
    scores = product(pam.mul(q, 0.25, offset=off).transpose(1, 2).contiguous(), k.transpose(1, 2).contiguous())
    later = torch.ones(20, 20, dtype=torch.bool, device="cuda").triu(1)
    e = pam.exp(scores.float(), offset=off).masked_fill(later, 0.0)
    n = pam.mul(e.unsqueeze(-1), v.transpose(1, 2).unsqueeze(2).contiguous(), offset=off).double().masked_fill(later[..., None], 0.0).sum(3)
    want = pam.div(n.float(), e.sum(-1, keepdim=True).expand_as(n).contiguous(), offset=off).transpose(1, 2)
    got = pam.attention(q, k, v, offset=off)
    # (products above: 16 + 20 terms, at most twice as sensitive in each of four steps)
    bound = 2.0 ** -24 * (16 + 20 + 8) * 16 * v.abs().max()
    assert (got - want).abs().max() <= bound


@gpu
@pytest.mark.parametrize("more", [{}, dict(cap=4.0), dict(slopes=np.array([0.25, 0.5], np.float32))], ids=["plain", "cap", "slopes"])
def test_exact_gradients(more):
    """The slopes of the pieces that the values are in; the inputs keep every sum of fractions away from a whole number, where the slope jumps."""
    for seed in range(3):
        _compare((1, 9, 9, 2, 1, 8), dict(causal=True, **more), seed=20 + seed, approx=False)


def test_exact_gradients_are_differences():
    """The definition's exact gradients (64 bits, no GPU) against differences of its result."""
    q, k, v, dy = (x[0, :, 0].astype(float) for x in _inputs(11, 1, 6, 6, 1, 1, 5))
    for more in ({}, dict(cap=2.0), dict(slope=0.25)):
        see = ref.visible(6, 6)
        grads, _ = ref.Head(q, k, v, see, **more).grads(dy, approx=False)
        rng = np.random.RandomState(0)
        for i, x in enumerate((q, k, v)):
            direction = rng.standard_normal(x.shape)
            h = 2.0 ** -30

            def at(step):
                moved = [q, k, v]
                moved[i] = x + step * direction
                return (ref.Head(*moved, see, **more).y * dy).sum()
            assert abs((at(h) - at(-h)) / (2 * h) - (grads[i] * direction).sum()) < 1e-5, (more, i)


@gpu
def test_approximate_gradients_pairwise():
    """approx_bwd as a pair: which factors' slopes are approximate."""
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(30, 1, 9, 9, 2, 1, 8))
    out = {}
    for flags in ((True, True), (False, False), (True, False), (False, True)):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        out[flags] = torch.autograd.grad(pam.attention(*leaves, approx_bwd=flags), leaves, dy)
    for flags, grads in out.items():
        assert all(torch.isfinite(g).all() for g in grads), flags
    # dv: an approximate slope of second operands; of first ones only through dn
    assert not torch.equal(out[True, True][2], out[True, False][2])
    assert not torch.equal(out[True, True][0], out[False, True][0])


@gpu
def test_graph_replays_and_streams():
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(3, 2, 90, 90, 4, 2, 64))
    want = pam.attention(q, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        for _ in range(2):
            eager = torch.autograd.grad(pam.attention(*leaves, approx_bwd=True), leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pam.attention(*leaves, approx_bwd=True)
        grads = torch.autograd.grad(y, leaves, dy)
    for turn in range(3):
        with torch.no_grad():
            for leaf, x in zip(leaves, (q, k, v)):
                leaf.copy_(x if turn != 1 else x.flip(1))
        graph.replay()
        torch.cuda.synchronize()
        if turn != 1:
            assert torch.equal(y, want) and all(torch.equal(a, b) for a, b in zip(grads, eager))
        else:
            assert torch.equal(y, pam.attention(q.flip(1).contiguous(), k.flip(1).contiguous(), v.flip(1).contiguous()))


@gpu
def test_gradients_repeat_bit_for_bit():
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(9, 2, 300, 300, 4, 2, 32))
    first = None
    for _ in range(3):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        grads = torch.autograd.grad(pam.attention(*leaves, approx_bwd=True), leaves, dy)
        first = first or grads
        assert all(torch.equal(a, b) for a, b in zip(first, grads))


@gpu
def test_some_gradients_only():
    pam = _host()
    q, k, v, dy = (_cuda(x) for x in _inputs(10, 1, 30, 30, 2, 2, 16))
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    all_three = torch.autograd.grad(pam.attention(*leaves, approx_bwd=True), leaves, dy)
    for i in range(3):
        mine = [x.clone().requires_grad_(i == j) for j, x in enumerate((q, k, v))]
        got, = torch.autograd.grad(pam.attention(*mine, approx_bwd=True), mine[i], dy)
        assert torch.equal(got, all_three[i])


def _refusals(device):
    pam = _host()

    def t(*s, **kw):
        return torch.zeros(*s, device=device, **kw)
    q, k = t(2, 5, 4, 8), t(2, 6, 2, 8)
    cases = [
        (ValueError, (q, k, t(2, 6, 2, 4)), {}), (ValueError, (q, t(2, 6, 3, 8), t(2, 6, 3, 8)), {}), (ValueError, (q, t(1, 6, 2, 8), t(1, 6, 2, 8)), {}),
        (ValueError, (t(2, 5, 8), k, k), {}), (ValueError, (t(1, 2, 1, 260), t(1, 2, 1, 260), t(1, 2, 1, 260)), {}),
        (TypeError, (q.double(), k, k), {}), (ValueError, (q, k, k), dict(window=0)), (ValueError, (q, k, k), dict(cap=-1.0)),
        (TypeError, (q, k, k), dict(prefix=t(2))), (ValueError, (q, k, k), dict(prefix=t(3, dtype=torch.int64))),
        (ValueError, (q, k, k), dict(documents=t(2, 5, dtype=torch.int64))), (ValueError, (q, k, k), dict(slopes=t(3))),
        (TypeError, (q, k, k), dict(slopes=t(4, dtype=torch.float64))), (RuntimeError, (q, k, k), dict(slopes=t(4).requires_grad_())),
        (ValueError, (q, k, k), dict(scale=0.0)), (ValueError, (q, k, k), dict(scale=float("nan"))), (ValueError, (q, k, k), dict(cap=1e9)),
        (ValueError, (q, k, k), dict(offset=0.5)), (ValueError, (t(2, 7, 4, 8), k, k), dict(documents=t(2, 6, dtype=torch.int64))),
    ]
    return pam, cases


def test_refuses_cpu_tensors():
    pam, cases = _refusals("cpu")
    q = torch.zeros(1, 2, 2, 8)
    with pytest.raises(RuntimeError):
        pam.attention(q, q, q)
    with pytest.raises((RuntimeError, NotImplementedError, ValueError)):
        pam.attention(q, q, q, use_kernel=False)
    for _, args, kw in cases:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            pam.attention(*args, **kw)


@gpu
def test_refusals():
    pam, cases = _refusals("cuda")
    for error, args, kw in cases:
        with pytest.raises(error):
            pam.attention(*args, **kw)
    with pytest.raises(ValueError):
        pam.attention(torch.zeros(1, 2, 2, 8, device="cuda"), torch.zeros(1, 2, 2, 8, device="cuda"), torch.zeros(1, 2, 2, 8, device="cuda"),
                      documents=torch.zeros(1, 2, dtype=torch.int64))
