"""pam.cached_attention at the ends of its windows, for heads of whole quads and others, and with an offset."""
import numpy as np
import pytest
import torch

import _attention_general as general
from _attention_ref import visible
from test_cached_attention import _cache, _compare, _cuda, _sequence

gpu = pytest.mark.gpu
DIMS = pytest.mark.parametrize("dim", [18, 66, 64, 20])


@gpu
@DIMS
@pytest.mark.parametrize("tokens", [1, 3])
def test_zero_queries_beside_large_keys(dim, tokens):
    """A zero times anything is zero, also where a key is out of the usual range."""
    def change(q, k, v):
        q[..., : dim // 2] = 0; k[..., : dim // 2] *= np.float32(2.0 ** 100)
    _compare(2, tokens, 4, 2, dim, 16, [150, 37], seed=dim, change=change)


@gpu
@DIMS
@pytest.mark.parametrize("large", [2.0 ** 85, 2.0 ** 39])
def test_the_power_of_two_that_zeros_stand_as(dim, large):
    def queries(q, k, v):
        q[:] = np.float32(2.0 ** -86) * np.sign(q); k[:] = np.float32(large) * np.sign(k)

    def keys(q, k, v):
        k[:] = np.float32(2.0 ** -86) * np.sign(k); q[:] = np.float32(large) * np.sign(q)
    for change in (queries, keys):
        _compare(1, 2, 4, 2, dim, 16, [150], seed=dim, change=change, scale=1.0)


@gpu
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 4), (6, 4)])
@pytest.mark.parametrize("what", ["values", "keys", "queries", "all", "wild", "small", "far", "large_query", "zero_rows"])
@pytest.mark.parametrize("dim", [18, 66])
def test_values_out_of_the_ordinary_in_heads_of_any_size(dim, what, tokens, heads):
    def change(q, k, v):
        rng = np.random.RandomState(5)
        for name, x in (("queries", q), ("keys", k), ("values", v)):
            if what in (name, "all"):
                x[rng.random_sample(x.shape) < 0.1] = 0
        if what == "wild":
            v[:, 2] *= np.float32(2.0 ** 60); k[1::3, 1] *= np.float32(2.0 ** -100); q[:, 0, 0] *= np.float32(2.0 ** -70)
        elif what == "small":
            v *= np.float32(1e-30); k[:, 1] *= np.float32(1e-20)
        elif what == "far":
            q[:] = np.abs(q); k[:] = np.abs(k) * np.linspace(-30, 30, k.shape[0], dtype=np.float32)[:, None, None, None]
        elif what == "large_query":
            q[:, :, 0] *= np.float32(1e26); k *= np.float32(1e-26)
        elif what == "zero_rows":
            k[:, 3] = 0; v[:, 5] = 0; q[:, 0, 0] = 0
    _compare(2, tokens, heads, 1, dim, 16, [150, 300], seed=7, change=change)


@gpu
@pytest.mark.parametrize("dim", [18, 66])
@pytest.mark.parametrize("scoring", [dict(window=1), dict(window=50), dict(window=1000), dict(cap=5.0), dict(slopes=np.array([0.5, 0.01, 0.0, 1.0], np.float32)), dict(scale=0.07),
                                     dict(cap=20.0, slopes=np.array([0.1, 0.2, 0.3, 0.4], np.float32), window=70)], ids=lambda s: "_".join(s))
def test_scores_and_windows_in_heads_of_any_size(dim, scoring):
    _compare(2, 3, 4, 2, dim, 16, [200, 31], seed=3, **scoring)
    _compare(2, 1, 4, 1, dim, 16, [200, 31], seed=4, **scoring)


@gpu
@DIMS
@pytest.mark.parametrize("seen", [1e-12, 0.0])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 4), (3, 4)])
def test_masked_values_are_in_no_result(tokens, heads, seen, dim):
    """Large values outside the window, and those of later tokens, beside small ones within it."""
    pam = __import__("pam_amd")
    rng = np.random.RandomState(0)
    k, v, table = _cache(rng, 1, 16, 14, 1, dim)
    length = 150
    v[:] = np.float32(1e12)
    places = [(table[0, j // 16], j % 16) for j in range(length + tokens)]
    for t in range(tokens):
        v[places[length + t]] = np.float32(seen) * (1.0 + rng.random_sample(dim))
    q = rng.standard_normal((1, tokens, heads, dim)).astype(np.float32)
    got = pam.cached_attention(_cuda(q), _cuda(k), _cuda(v), _cuda(table), _cuda(np.array([length])), window=1)
    want = torch.stack([_cuda(v[places[length + t]][0]) for t in range(tokens)])[None, :, None].expand(-1, -1, heads, -1)
    assert torch.equal(got, want)


@gpu
@DIMS
@pytest.mark.parametrize("offset", [0.7501, 0.76, 0.78, 1.0552, 1.45])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_no_numbers_beside_an_offset(value, offset, dim):
    pam = __import__("pam_amd")
    rng = np.random.RandomState(1)
    k, v, table = _cache(rng, 3, 8, 6, 2, dim)
    q = _cuda(rng.standard_normal((3, 2, 4, dim)).astype(np.float32))
    k, v, table, lengths = _cuda(k), _cuda(v), _cuda(table), _cuda(np.array([30, 30, 30]))
    clean = pam.cached_attention(q, k, v, table, lengths, offset=offset)
    assert torch.isfinite(clean).all()
    hidden = k.clone()
    hidden[table[0, 4]] = value
    hidden[table[1, 3], 7, 1, 5] = value                                    # place 31: the second token's own
    y = pam.cached_attention(q, hidden, v, table, lengths, offset=offset)
    assert torch.equal(y[0], clean[0]) and y[1, 1, 2:].isnan().all() and torch.equal(y[1, 0], clean[1, 0]) and torch.equal(y[1, 1, :2], clean[1, 1, :2])
    asked = q.clone()
    asked[2, 0, 1, 3] = value
    y = pam.cached_attention(asked, k, v, table, lengths, offset=offset)
    assert y[2, 0, 1].isnan().all() and torch.equal(y[2, 1], clean[2, 1]) and torch.equal(y[:2], clean[:2])
    broken = table.clone()
    broken[1, 1] = -1
    y = pam.cached_attention(q, k, v, broken, lengths, offset=offset)
    assert y[1].isnan().all() and torch.equal(y[0], clean[0])


@gpu
@DIMS
@pytest.mark.parametrize("offset", [None, 1.45])
def test_scores_at_both_ends(dim, offset):
    pam = __import__("pam_amd")
    q = torch.zeros(1, 1, 1, dim, device="cuda")
    q[..., 0] = 2.0 ** 63
    top = 2.0 ** (63 if offset is None else 62)
    k, v = torch.zeros(30, 16, 1, dim, device="cuda"), torch.randn(30, 16, 1, dim, device="cuda")
    table, lengths = torch.arange(30, dtype=torch.int32, device="cuda")[None], torch.tensor([470], device="cuda")
    k[..., 0] = -1.4 * top
    for most in (1.2 * top, -1.39 * top):
        k[11, 3, 0, 0] = most
        y = pam.cached_attention(q, k, v, table, lengths, scale=1.0, offset=offset)
        assert torch.equal(y[0, 0, 0], v[11, 3, 0])
    for sign in (1.0, -1.0):
        k[11, 3, 0, 0] = sign * 2.5 * top
        assert pam.cached_attention(q, k, v, table, lengths, scale=1.0, offset=offset).isnan().all()


@gpu
@DIMS
@pytest.mark.parametrize("offset", [0.77, 1.0552, 1.4])
@pytest.mark.parametrize("more", [{}, dict(cap=4.0), dict(window=60, slopes=np.array([0.25, 0.5, 0.01, 1.0], np.float32))], ids=lambda s: "_".join(s) or "plain")
def test_offset_moves_every_product(more, offset, dim):
    pam = __import__("pam_amd")
    rng = np.random.RandomState(dim)
    batch, tokens, heads, kv_heads, page = 2, 3, 4, 2, 16
    k, v, table = _cache(rng, batch, page, 12, kv_heads, dim)
    q = rng.standard_normal((batch, tokens, heads, dim)).astype(np.float32)
    lengths = np.array([150, 9])
    on = {n: _cuda(x) if isinstance(x, np.ndarray) else x for n, x in more.items()}
    got = pam.cached_attention(_cuda(q), _cuda(k), _cuda(v), _cuda(table), _cuda(lengths), offset=offset, **on).cpu().double().numpy()
    scoring = {n: x for n, x in more.items() if n == "cap"}
    for b in range(batch):
        end = lengths[b] + tokens
        keys, values, see = _sequence(k, table, b, end), _sequence(v, table, b, end), visible(tokens, end, True, more.get("window"))
        for h in range(heads):
            head = general.Head(q[b, :, h], keys[:, h // 2], values[:, h // 2], see, more["slopes"][h] if "slopes" in more else None, offset=offset, **scoring)
            assert (np.abs(got[b, :, h] - head.y.v) <= head.y.o).all()
