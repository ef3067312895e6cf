"""pam.rotary_append and pam.cached_attention: a paged cache against the definition, against pam.rotary and pam.attention, and their refusals."""
import numpy as np
import pytest
import torch

import _attention_ref as ref

gpu = pytest.mark.gpu


def _pam():
    import pam_amd as pam
    return pam


def _cache(rng, batch, page, per_sequence, kv_heads, dim, spare=3):
    """Random keys and values in pages that belong to the sequences in any order."""
    total = batch * per_sequence + spare
    table = rng.permutation(total)[:batch * per_sequence].reshape(batch, per_sequence).astype(np.int32)
    k, v = (rng.standard_normal((total, page, kv_heads, dim)).astype(np.float32) for _ in range(2))
    return k, v, table


def _sequence(cache, table, b, end):
    return cache[table[b]].reshape(-1, *cache.shape[2:])[:end]


def _cuda(x):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _expected(q, k, v, table, lengths, counts, **scoring):
    batch, tokens, heads, dim = q.shape
    group = heads // k.shape[2]
    y, off = np.zeros(q.shape), np.zeros(q.shape)
    slopes = scoring.pop("slopes", None)
    window = scoring.pop("window", None)
    for b in range(batch):
        n = tokens if counts is None else counts[b]
        end = lengths[b] + n
        if n == 0:
            continue
        see = ref.visible(n, end, True, window)
        keys, values = _sequence(k, table, b, end), _sequence(v, table, b, end)
        for h in range(heads):
            head = ref.Head(q[b, :n, h], keys[:, h // group], values[:, h // group], see, None if slopes is None else slopes[h], **scoring)
            y[b, :n, h], off[b, :n, h] = head.y, head.y_off
    return y, off


def _compare(batch, tokens, heads, kv_heads, dim, page, lengths, counts=None, seed=0, change=None, **scoring):
    pam = _pam()
    rng = np.random.RandomState(seed)
    lengths = np.array(lengths, np.int64)
    per_sequence = int((lengths.max() + tokens + page - 1) // page) + 1
    k, v, table = _cache(rng, batch, page, per_sequence, kv_heads, dim)
    q = rng.standard_normal((batch, tokens, heads, dim)).astype(np.float32)
    if change:
        change(q, k, v)
    counts = None if counts is None else np.array(counts, np.int64)
    want, off = _expected(q, k, v, table, lengths, counts, **dict(scoring))
    on = {n: _cuda(x) if isinstance(x, np.ndarray) else x for n, x in scoring.items()}
    got = pam.cached_attention(_cuda(q), _cuda(k), _cuda(v), _cuda(table), _cuda(lengths), _cuda(counts), **on).cpu().double().numpy()
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > off
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / np.maximum(off, 1e-300)):.2f} times the bound"
    return got


CASES = [  # batch, tokens, heads, kv heads, dim, page, lengths, counts
    (1, 1, 1, 1, 4, 1, [0], None), (1, 1, 4, 2, 64, 16, [37], None), (3, 1, 8, 2, 128, 64, [0, 63, 300], None), (2, 5, 3, 1, 80, 17, [100, 7], None),
    (2, 9, 4, 2, 32, 16, [5, 40], [9, 2]), (2, 3, 2, 1, 256, 4, [70, 0], [0, 3]), (1, 2, 6, 2, 100, 256, [513], None), (2, 1, 3, 3, 18, 5, [9, 64], None),
    (70, 1, 2, 1, 32, 16, [(i * 37) % 300 for i in range(70)], None), (64, 1, 2, 2, 16, 16, [(i * 91) % 1100 for i in range(64)], [i % 2 for i in range(64)]),
    (9, 6, 4, 1, 64, 32, [1500, 0, 700, 3, 64, 63, 65, 1, 128], [6, 6, 1, 2, 6, 6, 6, 0, 5]), (2, 11, 2, 1, 96, 16, [900, 100], None), (3, 2, 4, 1, 66, 16, [700, 64, 1], None),
    (1, 5, 5, 1, 128, 64, [2000], None), (1, 3, 4, 1, 112, 64, [800], None), (1, 2, 8, 1, 8, 64, [800], None), (1, 1, 20, 1, 256, 64, [300], None),
    (1, 7, 6, 1, 48, 32, [129], None), (1, 1, 1, 1, 1, 3, [10], None), (1, 1, 2, 1, 16, 8, [5000], None), (4, 4, 16, 4, 24, 16, [1, 2, 3, 400], [4, 3, 1, 4]),
]


@gpu
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_attention_over_pages(case):
    _compare(*case[:7], counts=case[7], seed=sum(case[:6]))


@gpu
@pytest.mark.parametrize("scoring", [dict(window=1), dict(window=50), dict(window=1000), dict(cap=5.0), dict(slopes=np.array([0.5, 0.01, 0.0, 1.0], np.float32)), dict(scale=0.07),
                                     dict(cap=20.0, slopes=np.array([0.1, 0.2, 0.3, 0.4], np.float32), window=70)], ids=lambda s: "_".join(s))
def test_scores_and_windows(scoring):
    _compare(2, 3, 4, 2, 64, 16, [200, 31], seed=3, **scoring)
    _compare(2, 1, 4, 1, 20, 16, [200, 31], seed=4, **scoring)


@gpu
@pytest.mark.parametrize("what", ["zero_rows", "zeros", "small", "far", "large_query", "zero_query"])
def test_values_out_of_the_ordinary(what):
    def change(q, k, v):
        if what == "zero_rows":
            k[:, 3] = 0; v[:, 5] = 0
        elif what == "zeros":
            for x in (q, k, v):
                x.reshape(-1)[::41] = 0
        elif what == "small":
            v *= np.float32(1e-30); k[:, 1] *= np.float32(1e-20)
        elif what == "far":
            q[:] = np.abs(q); k[:] = np.abs(k) * np.linspace(-30, 30, k.shape[0], dtype=np.float32)[:, None, None, None]
        elif what == "large_query":
            q[:, :, 0] *= np.float32(1e26); k *= np.float32(1e-26)
        else:
            q[:, :, 1] = 0
    for rows in ((2, 1, 4, 2, 64), (1, 6, 4, 1, 64)):
        _compare(*rows, 8, [130] * rows[0], seed=6, change=change)


@gpu
@pytest.mark.parametrize("rows", [(1, 1), (2, 4), (3, 4), (6, 4)])
@pytest.mark.parametrize("what", ["values", "keys", "queries", "all", "wild"])
def test_zeros_and_wild_values(rows, what):
    def change(q, k, v):
        rng = np.random.RandomState(5)
        for name, x in (("queries", q), ("keys", k), ("values", v)):
            if what in (name, "all"):
                x[rng.random_sample(x.shape) < 0.1] = 0
        if what == "wild":
            v[:, 2] *= np.float32(2.0 ** 60); k[1::3, 1] *= np.float32(2.0 ** -100); q[:, 0, 0] *= np.float32(2.0 ** -70)
    tokens, heads = rows
    _compare(2, tokens, heads, 1, 64, 16, [150, 300], seed=7, change=change)
    _compare(1, tokens, heads, 1, 20, 16, [150], seed=7, change=change)


@gpu
@pytest.mark.parametrize("window", [1, 64, 65, 700])
def test_windows_over_parts(window):
    _compare(5, 2, 8, 2, 32, 16, [1400, 90, 0, 777, 64], [2, 2, 1, 2, 0], seed=9, window=window)


@gpu
def test_no_numbers_and_pages_that_are_not_there():
    pam = _pam()
    rng = np.random.RandomState(1)
    k, v, table = _cache(rng, 3, 8, 6, 2, 32)
    q = _cuda(rng.standard_normal((3, 2, 4, 32)).astype(np.float32))
    lengths = _cuda(np.array([30, 30, 30]))
    k, v, good = _cuda(k), _cuda(v), _cuda(table)
    clean = pam.cached_attention(q, k, v, good, lengths)
    # a NaN behind a sequence's last token is in no result; one before it in all of its key head's
    hidden = k.clone()
    hidden[table[0, 4], 0] = float("nan")
    hidden[table[0, 5]] = float("inf")
    assert torch.equal(pam.cached_attention(q, hidden, v, good, lengths), clean)
    hidden[table[1, 3], 7, 1, 5] = float("nan")                              # place 31: the second token's own
    y = pam.cached_attention(q, hidden, v, good, lengths)
    assert y[1, 1, 2:].isnan().all() and torch.equal(y[1, 0], clean[1, 0]) and torch.equal(y[1, 1, :2], clean[1, 1, :2])
    spoilt = v.clone()
    spoilt[table[2, 0], 2, 0, 9] = float("inf")
    y = pam.cached_attention(q, k, spoilt, good, lengths)
    assert y[2, :, :2, 9].isnan().all() and torch.isfinite(y[2, :, :2, :9]).all() and torch.equal(y[2, :, 2:], clean[2, :, 2:]) and torch.equal(y[:2], clean[:2])
    # entries of the table that are no page, before and behind what a sequence has
    for bad in (-1, k.shape[0], 1 << 30):
        broken = good.clone()
        broken[0, 5] = bad; broken[1, 1] = bad
        y = pam.cached_attention(q, k, v, broken, lengths)
        assert torch.equal(y[0], clean[0]) and y[1].isnan().all() and torch.equal(y[2], clean[2])
    # more tokens than the table has places for, a negative length (none), no pages at all
    assert pam.cached_attention(q, k, v, good, _cuda(np.array([30, 47, 1 << 40])))[1:, 1].isnan().all()
    for window in (None, 3, 100):
        assert pam.cached_attention(q, k, v, good, _cuda(np.array([2 ** 63 - 1, 48, 1 << 31])), window=window).isnan().all()
    y = pam.cached_attention(q, k, v, good, _cuda(np.array([-5, 0, 30])))
    assert torch.equal(y[0], pam.cached_attention(q, k, v, good, _cuda(np.array([0, 0, 30])))[0])
    none = pam.cached_attention(q, k[:0], v[:0], good[:, :0], lengths)
    assert none.isnan().all()
    assert (pam.cached_attention(q, k, v, good, lengths, _cuda(np.array([0, 0, 0]))) == 0).all()
    assert pam.cached_attention(q[:, :0], k, v, good, lengths).shape == (3, 0, 4, 32)


@gpu
@pytest.mark.parametrize("dim,rotated,interleaved,norm", [(128, 128, False, True), (80, 40, True, False), (64, 64, False, False), (100, 100, False, True), (18, 6, True, True), (32, 0, False, True)])
@pytest.mark.parametrize("page", [1, 16, 17])
def test_append(dim, rotated, interleaved, norm, page):
    """The queries and the cache as pam.rotary and copies make them, bit for bit, and every other place as it was."""
    pam = _pam()
    rng = np.random.RandomState(dim + page)
    batch, tokens, heads, kv_heads = 3, 5, 4, 2
    k, v, table = _cache(rng, batch, page, 40 // page + 2, kv_heads, dim)
    cache_k, cache_v = _cuda(k), _cuda(v)
    qkv = torch.randn(batch, tokens, heads + 2 * kv_heads, dim, device="cuda")
    qkv[0, 0, 1] = 0                                                         # (a head of zeros takes the checked functions)
    q, new_k, new_v = qkv.split((heads, kv_heads, kv_heads), 2)
    weights = dict(q_weight=torch.randn(dim, device="cuda"), k_weight=torch.randn(dim, device="cuda")) if norm else {}
    cos, sin = pam.rotary_tables(64, rotated, device="cuda") if rotated else (torch.empty(64, 0, device="cuda"),) * 2
    lengths, counts = np.array([0, 33, 12]), np.array([5, 2, 0])
    got = pam.rotary_append(q, new_k, new_v, cos, sin, cache_k, cache_v, _cuda(table), _cuda(lengths), _cuda(counts), interleaved=interleaved, **weights)
    positions = _cuda(lengths)[:, None] + torch.arange(tokens, device="cuda")
    want_q, want_k = pam.rotary(q, new_k, cos, sin, positions, interleaved=interleaved, **weights)
    k, v = torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda()
    for b in range(batch):
        assert torch.equal(got[b, :counts[b]], want_q[b, :counts[b]]) and (got[b, counts[b]:] == 0).all()
        for t in range(counts[b]):
            at = lengths[b] + t
            k[table[b, at // page], at % page] = want_k[b, t]
            v[table[b, at // page], at % page] = new_v[b, t]
    assert torch.equal(cache_k, k) and torch.equal(cache_v, v)


@gpu
def test_append_leaves_places_that_are_not_there():
    pam = _pam()
    rng = np.random.RandomState(0)
    k, v, table = _cache(rng, 4, 4, 3, 1, 8)
    cos, sin = pam.rotary_tables(11, 8, device="cuda")
    q, new = torch.randn(4, 3, 2, 8, device="cuda"), torch.randn(4, 3, 1, 8, device="cuda")
    table[0, 1] = -1; table[1, 1] = k.shape[0]
    lengths = np.array([3, 3, 10, -1])
    cache_k, cache_v = _cuda(k), _cuda(v)
    got = pam.rotary_append(q, new, new, cos, sin, cache_k, cache_v, _cuda(table), _cuda(lengths))
    want_q, want_k = pam.rotary(q, new, cos, sin, _cuda(lengths)[:, None] + torch.arange(3, device="cuda"))
    want = torch.from_numpy(k).cuda()
    want[table[0, 0], 3] = want_k[0, 0]
    want[table[1, 0], 3] = want_k[1, 0]
    want[table[2, 2], 2] = want_k[2, 0]                                       # place 10
    want[table[2, 2], 3] = want_k[2, 1]                                       # place 11: in the pages, not in the tables
    same = (cache_k == want) | (cache_k.isnan() & want.isnan())
    assert same.all() and cache_k[table[2, 2], 3].isnan().all()
    for far in (1 << 40, 2 ** 63 - 1):
        before = cache_k.clone(), cache_v.clone()
        assert pam.rotary_append(q, new, new, cos, sin, cache_k, cache_v, _cuda(table), torch.full((4,), far, device="cuda")).isnan().all()
        assert torch.equal(cache_k.view(torch.int32), before[0].view(torch.int32)) and torch.equal(cache_v, before[1])
    assert torch.equal(got[:2], want_q[:2]) and got[2, 1:].isnan().all() and got[3].isnan().all()
    assert (cache_v[table[2, 2], 3] == new[2, 1]).all() and torch.equal(cache_v[table[3]], torch.from_numpy(v).cuda()[table[3]])


@gpu
def test_a_run_as_a_model_makes_it():
    """A prompt and then tokens one by one through the cache, against attention over everything at once."""
    pam = _pam()
    torch.manual_seed(0)
    batch, total, heads, kv_heads, dim, page = 2, 40, 4, 2, 64, 16
    q, k, v = (torch.randn(batch, total, n, dim, device="cuda") for n in (heads, kv_heads, kv_heads))
    cos, sin = pam.rotary_tables(total, dim, device="cuda")
    rotated_q, rotated_k = pam.rotary(q, k, cos, sin)
    want = pam.attention(rotated_q, rotated_k, v, window=20)
    cache_k, cache_v = (torch.zeros(8, page, kv_heads, dim, device="cuda") for _ in range(2))
    table = torch.tensor([[3, 1, 7], [0, 5, 2]], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(batch, dtype=torch.int64, device="cuda")
    out = []
    for begin, end in [(0, 25), (25, 28)] + [(i, i + 1) for i in range(28, total)]:
        step = [t[:, begin:end] for t in (q, k, v)]
        new_q = pam.rotary_append(*step, cos, sin, cache_k, cache_v, table, lengths)
        out.append(pam.cached_attention(new_q, cache_k, cache_v, table, lengths, window=20))
        lengths += end - begin
    # (scores of 64 terms, weights of 20: the same values in other orders of sums; e is twice as sensitive as a score, which is below 8)
    size = v.abs().max().item()
    assert (torch.cat(out, 1) - want).abs().max().item() < 2.0 ** -24 * (4 * 66 * 8 + 2 * 40) * 4 * size


@gpu
def test_graph_replays():
    """One decoding step recorded, replayed while the lengths grow; two graphs side by side have scratch of their own."""
    pam = _pam()
    rng = np.random.RandomState(3)
    k, v, table = _cache(rng, 2, 16, 60, 2, 64)
    cos, sin = pam.rotary_tables(1000, 64, device="cuda")
    table = _cuda(table)
    make = lambda: (_cuda(k), _cuda(v), torch.tensor([600, 700], device="cuda"))
    q, new_k, new_v = (torch.randn(2, 1, n, 64, device="cuda") for n in (8, 2, 2))

    def step(cache_k, cache_v, lengths):
        new_q = pam.rotary_append(q, new_k, new_v, cos, sin, cache_k, cache_v, table, lengths)
        y = pam.cached_attention(new_q, cache_k, cache_v, table, lengths)
        lengths += 1
        return y
    eager = make()
    want = [step(*eager).clone() for _ in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*make())
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        state, graph = make(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step(*state)
        state[2].copy_(torch.tensor([600, 700], device="cuda"))
        state[0].copy_(_cuda(k)); state[1].copy_(_cuda(v))
        graphs.append((graph, y, state))
    other = torch.cuda.Stream()
    for i in range(4):
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.synchronize()
        for _, y, _ in graphs:
            assert torch.equal(y, want[i]), i
        torch.randn(1000, 1000, device="cuda").sum()


@gpu
def test_strides_of_a_cache():
    """Caches whose heads come before their places, or that are two halves of one tensor."""
    pam = _pam()
    rng = np.random.RandomState(4)
    k, v, table = _cache(rng, 2, 8, 5, 2, 32)
    q, lengths, table = torch.randn(2, 2, 4, 32, device="cuda"), _cuda(np.array([30, 9])), _cuda(table)
    want = pam.cached_attention(q, _cuda(k), _cuda(v), table, lengths)
    by_head = [_cuda(x).transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    assert torch.equal(pam.cached_attention(q, *by_head, table, lengths), want)
    both = torch.empty(k.shape[0], 2, *k.shape[1:], device="cuda")
    both[:, 0], both[:, 1] = _cuda(k), _cuda(v)
    assert torch.equal(pam.cached_attention(q, both[:, 0], both[:, 1], table, lengths), want)
    cos, sin = pam.rotary_tables(64, 32, device="cuda")
    new = torch.randn(2, 2, 2, 32, device="cuda")
    plain = [_cuda(k), _cuda(v)]
    pam.rotary_append(q, new, new, cos, sin, *plain, table, lengths)
    pam.rotary_append(q, new, new, cos, sin, both[:, 0], both[:, 1], table, lengths)
    assert torch.equal(both[:, 0], plain[0]) and torch.equal(both[:, 1], plain[1])
    wide = torch.randn(2, 2, 4, 64, device="cuda")[..., ::2]
    assert torch.equal(pam.cached_attention(wide, _cuda(k), _cuda(v), table, lengths), pam.cached_attention(wide.contiguous(), _cuda(k), _cuda(v), table, lengths))


def _refused(device):
    def t(*s, **kw):
        return torch.zeros(*s, device=device, **kw)
    q, kv, cache = t(2, 1, 4, 8), t(2, 1, 2, 8), t(6, 4, 2, 8)
    table, lengths, cos = t(2, 3, dtype=torch.int32), t(2, dtype=torch.int64), t(12, 4)
    good = dict(cache_k=cache, cache_v=t(6, 4, 2, 8), pages=table, lengths=lengths)
    both = [
        (ValueError, dict(cache_v=t(6, 4, 2, 4))), (ValueError, dict(cache_v=t(6, 4, 1, 8))), (ValueError, dict(cache_v=t(6, 2, 4, 8).transpose(1, 2))),
        (TypeError, dict(cache_k=t(6, 4, 2, 8, dtype=torch.float64), cache_v=t(6, 4, 2, 8, dtype=torch.float64))), (TypeError, dict(pages=table.long())),
        (ValueError, dict(pages=t(3, 3, dtype=torch.int32))), (TypeError, dict(lengths=lengths.int())), (ValueError, dict(lengths=t(3, dtype=torch.int64))),
        (ValueError, dict(counts=t(1, dtype=torch.int64))), (ValueError, dict(cache_k=t(6, 4, 3, 8), cache_v=t(6, 4, 3, 8))),
        (ValueError, dict(cache_k=t(6, 4, 2, 16)[..., ::2], cache_v=t(6, 4, 2, 16)[..., ::2])),
    ]
    append = both + [
        (ValueError, dict(cache_k=cache, cache_v=cache)), (ValueError, dict(cache_k=t(1, 4, 2, 8).expand(6, 4, 2, 8), cache_v=t(1, 4, 2, 8).expand(6, 4, 2, 8))),
        (RuntimeError, dict(cache_k=t(6, 4, 2, 8).requires_grad_())), (ValueError, dict(cos=t(12, 5), sin=t(12, 5))), (ValueError, dict(v=t(2, 1, 4, 8))),
        (ValueError, dict(q_weight=t(7))), (ValueError, dict(k=t(2, 2, 2, 8), v=t(2, 2, 2, 8))),
    ]
    attend = both + [(ValueError, dict(window=0)), (ValueError, dict(cap=0.0)), (ValueError, dict(scale=-1.0)), (ValueError, dict(offset=3.0)), (ValueError, dict(slopes=t(2))),
                     (RuntimeError, dict(q=q.clone().requires_grad_())), (ValueError, dict(q=t(2, 1, 3, 8)))]
    return dict(q=q, k=kv, v=kv.clone(), cos=cos, sin=cos.clone(), **good), append, dict(q=q, **good), attend


@gpu
def test_refusals():
    pam = _pam()
    append, append_cases, attend, attend_cases = _refused("cuda")
    pam.rotary_append(**append)
    pam.cached_attention(**attend)
    for error, kw in append_cases:
        with pytest.raises(error):
            pam.rotary_append(**{**append, **kw})
    for error, kw in attend_cases:
        with pytest.raises(error):
            pam.cached_attention(**{**attend, **kw})
    # a cache that is read by the same call
    cache = torch.zeros(6, 4, 2, 8, device="cuda")
    with pytest.raises(ValueError):
        pam.rotary_append(**{**append, "cache_k": cache, "k": cache[:2, :1]})


def test_refuses_cpu_tensors():
    pam = _pam()
    append, append_cases, attend, attend_cases = _refused("cpu")
    for call, args, cases in ((pam.rotary_append, append, append_cases), (pam.cached_attention, attend, attend_cases)):
        for _, kw in [(None, {})] + cases:
            with pytest.raises((RuntimeError, ValueError, TypeError)):
                call(**{**args, **kw})


@gpu
def test_writing_counts_as_a_change():
    """A graph that has saved the cache is not run on the new values."""
    pam = _pam()
    append, *_ = _refused("cuda")
    weight = torch.ones(8, device="cuda", requires_grad=True)
    y = (append["cache_k"] * weight).sum()
    pam.rotary_append(**append)
    with pytest.raises(RuntimeError, match="modified"):
        y.backward()
