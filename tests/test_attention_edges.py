"""pam.attention where its usual loops' windows end: gradients of very different sizes in a row, exact zeros beside tiny and large values, weights and gradients
far below the largest, scores near the end of the range, numbers that are none beside an offset, and the scratch of long windows."""
import ctypes

import numpy as np
import pytest
import torch

import _attention_general as general
import test_attention
from test_attention import _check, _cuda, _inputs, _run

gpu = pytest.mark.gpu
APPROX = pytest.mark.parametrize("approx", [True, False], ids=["approximate", "exact"])


def _compare(shape, masks, seed=0, approx=True, train=True, change=None, offset=None, tight=0.0):
    """approx: as approx_bwd, a pair of it for first and second operands counts as set for the exponential.  tight: what part of the gradients' values the bounds hold to 5 % at least."""
    pam = __import__("pam_amd")
    q, k, v, dy = _inputs(seed, *shape)
    if change:
        change(q, k, v, dy)
    flags = (*approx, True) if isinstance(approx, tuple) else (approx,) * 3
    want, off, grads, offs = general.attention(q, k, v, dy if train else None, flags=flags, offset=offset, **masks)
    leaves = [_cuda(x).requires_grad_(train) for x in (q, k, v)]
    on = {n: _cuda(x) if isinstance(x, np.ndarray) else x for n, x in masks.items()}
    y = pam.attention(*leaves, **on, approx_bwd=approx, offset=offset)
    _check(y, want, off, "y")
    if not train:
        return
    assert np.concatenate([(o < 0.05 * np.abs(w))[w != 0] for w, o in zip(grads, offs)]).mean() >= tight
    for name, got, w, o in zip("qkv", torch.autograd.grad(y, leaves, _cuda(dy)), grads, offs):
        _check(got, w, o, "d" + name)


# ---------------------------------------------------------------- gradients that span more than an integer addition may

@gpu
@APPROX
@pytest.mark.parametrize("large,small", [(2.0 ** 12, 1e-40), (2.0 ** 9, 1e-39), (2.0 ** 60, 2.0 ** -118), (2.0 ** 40, 2.0 ** -100), (1e-20, 1e-41)])
@pytest.mark.parametrize("dim", [16, 64, 130])
def test_a_gradient_of_very_different_sizes(dim, large, small, approx):
    """A query's gradient is scaled by its largest value: what is far below that may neither wrap nor be read for another number."""
    def change(q, k, v, dy):
        dy[:, 11] = np.float32(small) * np.sign(dy[:, 11])
        dy[:, 11, :, 0] = large
        dy[:, 30, :, 5] = large
        dy[:, 30, :, 7] = small
    _compare((1, 45, 45, 2, 1, dim), {}, seed=dim, approx=approx, change=change)


@gpu
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@APPROX
def test_a_gradient_that_is_no_number(value, approx):
    """It reaches its query's gradient, and those of the keys that the query sees, whatever else is in the row."""
    q, k, v, dy = _inputs(4, 1, 40, 40, 2, 1, 32)
    v[..., 7] = 0                                        # (y is zero there, too)
    dy[0, 20, 0, 7] = value
    y, (dq, dk, dv) = _run(q, k, v, dy, {}, approx)
    assert torch.isfinite(y).all()
    assert dq[0, 20, 0].isnan().all() and torch.isfinite(dq[0, :20]).all() and torch.isfinite(dq[0, 21:]).all() and torch.isfinite(dq[0, 20, 1]).all()
    assert dk[0, :21].isnan().all() and torch.isfinite(dk[0, 21:]).all()


# ---------------------------------------------------------------- a number that stands for zero

@gpu
@pytest.mark.parametrize("dim", [16, 64, 100])
@pytest.mark.parametrize("large", [2.0 ** 85, 2.0 ** 39, 1.0])
def test_the_power_of_two_that_zeros_stand_as(dim, large):
    """Scaled queries, and keys, of just 2^-86 of either sign are numbers."""
    def queries(q, k, v, dy):
        q[:] = np.float32(2.0 ** -86) * np.sign(q); k[:] = np.float32(large) * np.sign(k)
        q[:, 7, :, 1] = 2.0 ** -100                       # (a value out of the range sends the whole unit through the full definition)

    def keys(q, k, v, dy):
        k[:] = np.float32(2.0 ** -86) * np.sign(k); q[:] = np.float32(large) * np.sign(q)
    for change in (queries, keys):
        _compare((1, 45, 70, 2, 1, dim), dict(scale=1.0), seed=dim, change=change, train=False)


@gpu
@APPROX
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_values_that_are_that_power(dim, approx):
    def change(q, k, v, dy):
        v[:, ::3] = np.float32(2.0 ** -86) * np.sign(v[:, ::3])
        v[:, 1::3] *= np.float32(2.0 ** -80)
    _compare((1, 45, 45, 2, 1, dim), {}, seed=dim + 1, approx=approx, change=change)


@gpu
@APPROX
@pytest.mark.parametrize("what", ["values", "gradients"])
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_zeros_beside_tiny_and_large_values(dim, what, approx):
    """A zero's product is zero, not a small number that others are smaller than."""
    def change(q, k, v, dy):
        if what == "values":
            v *= np.float32(2.0 ** -80); v[..., : dim // 2] = 0; dy[..., : dim // 2] = np.abs(dy[..., : dim // 2]) * np.float32(32.0)
        else:
            dy[..., :-1] = 0; v[..., :-1] = np.float32(2.0 ** 39) * (1.0 + np.abs(v[..., :-1]) % 0.9)
            v[..., -1] = np.float32(2.0 ** -39) * (1.0 + np.abs(v[..., -1]) % 0.5) * np.sign(v[..., -1])
    for tokens, keys in ((7, 9), (45, 70)):
        _compare((1, tokens, keys, 2, 1, dim), {}, seed=dim, approx=approx, change=change)


@gpu
@APPROX
@pytest.mark.parametrize("more", [{}, dict(cap=4.0), dict(slopes=np.array([0.25, 0.5], np.float32))], ids=["plain", "cap", "slopes"])
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_rows_of_zeros(dim, more, approx):
    """Queries and keys that are all zeros, as a layer's are that begins with them, or padding's: every score is zero, and so is its fraction."""
    def change(q, k, v, dy):
        q[:, 20:30] = 0; k[:, 5:12] = 0; q[:, 40, :, 1:] = 0; q[:, 40, :, 0] = np.float32(2.0 ** -60)
    _compare((1, 45, 70, 2, 1, dim), more, seed=dim, approx=approx, change=change)


# ---------------------------------------------------------------- weights and gradients far below the largest

@gpu
@APPROX
@pytest.mark.parametrize("dim", [16, 32, 100])
def test_zeros_and_tiny_values_of_small_weight(dim, approx):
    """Weights down to 2^-60 with values that are zero, or small: their products are far below one."""
    def change(q, k, v, dy):
        rng = np.random.RandomState(dim)
        q[:] = np.abs(q); k[:] = np.abs(k) * np.linspace(-4.0, 4.0, k.shape[1], dtype=np.float32)[None, :, None, None] * np.float32(16.0 / dim ** 0.5)
        v[rng.random_sample(v.shape) < 0.2] = 0
        v[:, ::5] *= np.float32(2.0 ** -70)
    _compare((1, 60, 130, 1, 1, dim), dict(causal=False), seed=4, approx=approx, change=change)


@gpu
@APPROX
@pytest.mark.parametrize("dim", [16, 64, 100])
def test_a_small_gradient_at_a_small_weight(dim, approx):
    """The last key is seen by the last query alone, at a weight of 2^-50, and that query's gradient is 2^-34 of the others'."""
    def change(q, k, v, dy):
        for x in (v, dy):
            x[:] = (1.0 + np.abs(x) % 1.0) * np.sign(x)
        v *= np.float32(2.0 ** -10)
        k[:, -1] = -q[:, -1, :1] * np.float32(50.0 * np.log(2.0) * dim ** 0.5 / np.square(q[0, -1, 0]).sum())
        dy[:, -1] *= np.float32(2.0 ** -32)
    _compare((1, 70, 70, 1, 1, dim), {}, seed=dim, approx=approx, change=change, tight=0.2)


# ---------------------------------------------------------------- the ends of the range

@gpu
@pytest.mark.parametrize("offset", [None, 1.45])
@pytest.mark.parametrize("keys", [3, 200])
def test_scores_at_both_ends(keys, offset):
    """Scores of 2^126 and more beside others as far below zero: all of the weight is the largest one's.  From 2^127 on they are no numbers."""
    pam = __import__("pam_amd")
    q = torch.zeros(1, 1, 1, 4, device="cuda")
    q[..., 0] = 2.0 ** 63
    top = 2.0 ** (63 if offset is None else 62)
    k = torch.zeros(1, keys, 1, 4, device="cuda")
    k[..., 0] = -1.4 * top
    k[:, keys // 2, :, 0] = 1.2 * top
    v = torch.randn(1, keys, 1, 4, device="cuda")
    y = pam.attention(q, k, v, scale=1.0, causal=False, offset=offset)
    assert torch.equal(y[0, 0, 0], v[0, keys // 2, 0])
    k[:, keys // 2, :, 0] = -1.39 * top            # (none is above zero)
    assert torch.equal(pam.attention(q, k, v, scale=1.0, causal=False, offset=offset)[0, 0, 0], v[0, keys // 2, 0])
    for sign in (1.0, -1.0):
        k[:, keys // 2, :, 0] = sign * 2.5 * top
        assert pam.attention(q, k, v, scale=1.0, causal=False, offset=offset).isnan().all()


@gpu
@pytest.mark.parametrize("offset", [0.7501, 0.76, 0.78, 1.0552, 1.45])
@pytest.mark.parametrize("value", [float("nan"), -float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("where", ["q", "k"])
def test_no_numbers_beside_an_offset(where, value, offset):
    pam = __import__("pam_amd")
    q, k, v, dy = (_cuda(x) for x in _inputs(1, 1, 40, 40, 2, 1, 32))
    clean = pam.attention(q, k, v, offset=offset)
    (q if where == "q" else k)[0, 20, 0, 3] = np.float32(value).item()
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    y = pam.attention(*leaves, offset=offset, approx_bwd=True)
    bad = y[0, 20, 0] if where == "q" else y[0, 20:]
    assert bad.isnan().all() and torch.equal(y[0, :20], clean[0, :20])
    dq = torch.autograd.grad(y, leaves, dy)[0]
    assert (dq[0, 20, 0] if where == "q" else dq[0, 20:]).isnan().all() and torch.isfinite(dq[0, :20]).all()


# ---------------------------------------------------------------- offsets, slopes of each kind, masks over several spans

MASKS = {
    "causal": {}, "all": dict(causal=False), "window": dict(window=70), "window_both_ways": dict(window=30, causal=False), "prefix": dict(prefix=np.array([100])),
    "documents": dict(documents=np.repeat(np.array([[0, 1 << 40, 0, -1, 2]]), 29, axis=1)[:, :144]), "slopes": dict(slopes=np.array([0.5, 0.03], np.float32)),
    "cap": dict(cap=3.0), "cap_and_window": dict(cap=10.0, window=65),
}


@gpu
@pytest.mark.parametrize("name", MASKS)
@pytest.mark.parametrize("dim", [16, 24])
def test_exact_gradients_over_several_spans(dim, name):
    _compare((1, 144, 144, 2, 1, dim), MASKS[name], 31, False, tight=0.0 if "cap" in name else 0.2)


@gpu
@pytest.mark.parametrize("dim", [130, 256])
def test_exact_gradients_of_wide_heads(dim):
    _compare((1, 70, 70, 1, 1, dim), {}, 32, False, tight=0.1)


@gpu
@pytest.mark.parametrize("approx", [True, False, (True, False), (False, True), (False, False)], ids=str)
@pytest.mark.parametrize("offset", [None, 0.77, 1.0552, 1.4])
@pytest.mark.parametrize("more", [{}, dict(cap=4.0), dict(slopes=np.array([0.25, 0.5], np.float32))], ids=["plain", "cap", "slopes"])
def test_gradients_of_either_kind_and_offset(more, offset, approx):
    _compare((1, 7, 9, 2, 1, 8), more, 34, approx, offset=offset, tight=0.25)
    _compare((1, 30, 75, 2, 1, 24), more, 35, approx, offset=offset)


@gpu
@pytest.mark.parametrize("approx", [True, False, (True, False), (False, True)], ids=str)
@pytest.mark.parametrize("offset", [None, 1.05, 1.4])
def test_pairs_without_a_gradient_give_none(offset, approx):
    """Values that are all zeros, and queries of a single key: zeros to the bit, in the full definition (offsets, mixed slopes, values out of the usual range) too."""
    pam = __import__("pam_amd")
    for dim in (1, 18, 64, 130):
        q, k, v, dy = _inputs(dim, 1, 70, 70, 4, 2, dim)
        dy[:, 50] *= np.float32(1e14)
        for values, window in ((np.zeros_like(v), None), (v, 1)):
            if window and (isinstance(approx, tuple) or approx and offset):              # (the quotient's slopes are of two kinds, or have the offset another number of times, and do not cancel)
                continue
            leaves = [_cuda(x).requires_grad_() for x in (q, k, values)]
            y = pam.attention(*leaves, window=window, offset=offset, approx_bwd=approx)
            dq, dk, dv = torch.autograd.grad(y, leaves, _cuda(dy))
            assert (dq == 0).all() and (dk == 0).all() and torch.isfinite(dv).all() and (dv != 0).any()


# ---------------------------------------------------------------- scratch

class _Shape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_long) for n in ("batch", "tokens", "keys", "heads", "kv_heads", "dim", "values")] + [(n, ctypes.c_float) for n in ("scale", "cap", "offset")] + [
        ("causal", ctypes.c_int), ("window", ctypes.c_long), ("prefix", ctypes.c_void_p), ("documents", ctypes.c_void_p), ("slopes", ctypes.c_void_p)]


def _scratch(tokens, heads, kv_heads, dim, window, batch=1, keys=None, causal=True):
    from pam_amd import _abi
    lib = ctypes.CDLL(str(_abi.library_path()))
    forward, backward = lib.pam_hip_attention_workspace_bytes, lib.pam_hip_attention_bwd_workspace_bytes
    forward.restype = backward.restype = ctypes.c_size_t
    s = _Shape(batch, tokens, keys or tokens, heads, kv_heads, dim, dim, 0.125, 0.0, 1.0, causal, window, None, None, None)
    return forward(ctypes.byref(s)), backward(ctypes.byref(s), 1, 1)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [1, 64, 256, 1000, 5000])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim", [(2048, 8, 2, 64), (32768, 32, 8, 128), (131072, 32, 8, 128), (524288, 8, 2, 64), (8192, 1, 1, 16), (100001, 3, 3, 256)])
def test_scratch_of_a_window_is_what_its_tiles_see(tokens, heads, kv_heads, dim, window, causal):
    """A tile of at most 256 rows of one head sees a window's worth of keys: cut into two spans of 64 at least, that many parts of every row; and no more
    than some turns of the chip's units, whatever the length."""
    forward, backward = _scratch(tokens, heads, kv_heads, dim, window, causal=causal)
    rows = tokens * heads * dim * 4
    parts = (256 + (1 if causal else 2) * window) // 128 + 2
    assert forward <= rows * parts + (rows // dim * parts * 2 + 4096)
    seen_rows = (256 + (1 if causal else 2) * window) * (heads // kv_heads) // 128 + 2
    records = 2 * rows + 4 * rows // dim + 4096
    keys = 2 * tokens * kv_heads * dim * 4 * seen_rows
    assert backward <= records + rows * parts + keys + (1 << 24)
    assert max(forward, backward - records) <= max(4 * rows, 3 << 29)


@pytest.mark.parametrize("tokens,keys", [(1, 1 << 20), (64, 1 << 20), (4096, 4096), (32768, 32768), (300, 100000)])
def test_scratch_of_long_rows_is_bounded(tokens, keys):
    forward, backward = _scratch(tokens, 8, 2, 64, 0, keys=keys)
    assert max(forward, backward - 2 * tokens * 8 * 65 * 4) <= 3 << 29


@gpu
@pytest.mark.parametrize("shape,masks", [((1, 700, 700, 2, 1, 16), dict(window=100)), ((1, 1100, 1100, 1, 1, 16), dict(window=65)), ((2, 300, 1000, 2, 2, 20), dict(window=333)),
                                         ((1, 900, 900, 1, 1, 20), dict(window=90, causal=False)), ((1, 500, 700, 1, 1, 16), dict(window=80, prefix=np.array([130]))),
                                         ((1, 64, 2000, 1, 1, 16), dict(window=1500)), ((1, 40, 20, 1, 1, 16), dict(window=5)), ((1, 300, 200, 2, 1, 16), dict(window=90, causal=False))],
                         ids=lambda x: "x".join(map(str, x)) if isinstance(x, tuple) else "_".join(x))
def test_windows_of_many_tiles(shape, masks):
    test_attention._compare(shape, masks, seed=sum(shape))


@gpu
@pytest.mark.parametrize("dim", [40, 64, 128, 130, 256])
@pytest.mark.parametrize("tokens,window,heads,kv_heads", [(3000, 256, 6, 2), (2500, 700, 2, 2), (5000, 65, 3, 1)])
def test_a_long_window_by_pieces(tokens, window, heads, kv_heads, dim):
    """A window over many tiles against the same by some hundred queries at a time, each over the keys that they see."""
    pam = __import__("pam_amd")
    torch.manual_seed(dim)
    q, k, v = (torch.randn(1, tokens, n, dim, device="cuda") for n in (heads, kv_heads, kv_heads))
    dy = torch.randn_like(q)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    y = pam.attention(*leaves, window=window, approx_bwd=True)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    want = [torch.zeros_like(x, dtype=torch.float64) for x in (q, q, k, v)]
    for begin in range(0, tokens, 500):
        end, first = min(tokens, begin + 500), max(0, begin - window + 1)
        rows, seen = slice(begin, end), slice(first, end)
        piece = [x[:, at].clone().requires_grad_() for x, at in ((q, rows), (k, seen), (v, seen))]
        part = pam.attention(*piece, window=window, approx_bwd=True)
        for total, at, add in zip(want, (rows, rows, seen, seen), (part.detach(), *torch.autograd.grad(part, piece, dy[:, rows]))):
            total[:, at] += add
    # (sums of dim and of window x heads terms in other orders, the steps between at most twice as sensitive each)
    for name, a, b in zip(("y", "dq", "dk", "dv"), got, want):
        assert (a - b).norm() <= 4 * 2.0 ** -24 * (dim + window * (heads // kv_heads)) * b.norm(), name


@gpu
@pytest.mark.parametrize("approx", [True, False, (True, False)], ids=str)
def test_the_full_definition_in_a_graph(approx):
    """Units that begin again, and zeros' loops, recorded and replayed on other values."""
    pam = __import__("pam_amd")
    sets = [[_cuda(x) for x in _inputs(seed, 1, 150, 150, 4, 2, 40)] for seed in (1, 2)]
    for q, k, v, dy in sets:
        v[:, 33] *= 1e14; k[:, 70, :, 3] = 0; q[:, 5] = 0; dy[:, 20, 0, 0] = 1e30
    eager = []
    for q, k, v, dy in sets:
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        y = pam.attention(*leaves, window=100, approx_bwd=approx)
        eager.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    del leaves, y
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    static = [x.clone() for x in sets[0]]
    with torch.cuda.stream(side):
        leaves = [x.requires_grad_() for x in static[:3]]
        torch.autograd.grad(pam.attention(*leaves, window=100, approx_bwd=approx), leaves, static[3])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pam.attention(*leaves, window=100, approx_bwd=approx)
        grads = torch.autograd.grad(y, leaves, static[3])
    for turn in (1, 0, 1, 0):
        with torch.no_grad():
            for to, x in zip(static, sets[turn]):
                to.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([y, *grads], eager[turn]):
            assert torch.equal(a, b) or torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())
        torch.randn(1000, 1000, device="cuda").sum()
