"""The sums of the layers' products (linear_act, gated_linear and their gradients): chains of at most 1024 terms whatever the sizes, and no
more scratch than the plain products take.

The order that include/pam_hip_block.h states is computed here from products of one chain each, added in float32: equal to the last bit.
"""
import ctypes

import numpy as np
import pytest
import torch

import pam_amd as pam
from pam_amd import _abi
from _util import assert_same_bits
from test_block_ops import chain_act

_f, _i, _l, _p, _z = ctypes.c_float, ctypes.c_int, ctypes.c_long, ctypes.c_void_p, ctypes.c_size_t


def entry(name, argtypes, restype=_i):
    f = getattr(_abi.load_library(), name)
    return ctypes.CFUNCTYPE(restype, *argtypes)(ctypes.cast(f, _p).value)          # (the package's own declarations stay)


SIZES = [(2577, 2600, 2560), (6144, 6144, 2080), (1000, 2000, 3000), (130, 640, 131072), (40, 30, 5000)]


@pytest.mark.parametrize("m,n,k", SIZES + [(8192, 4096, 22016), (11008, 2048, 65536), (4096, 4096, 131072), (22016, 4096, 16384), (64, 64, 1 << 24)])
def test_scratch_is_that_of_the_plain_product(m, n, k):
    """Pieces of cut tiles as the plain product's plan has them; the chains in them take none."""
    sizes = [entry(f"pam_hip_{name}_workspace_bytes", [_l] * 3, _z)(m, n, k) for name in ("layer_grad", "linear_act")]
    plain = entry("pam_hip_gemm_workspace_bytes", [_l] * 4, _z)
    assert sizes == [plain(1, m, n, k)] * 2
    assert entry("pam_hip_gated_linear_workspace_bytes", [_l] * 3, _z)(m, n // 2, k) == plain(1, m, n // 4 * 4, k)


# ---------------------------------------------------------------- the order of the sums

def matrix(t):
    return t.data_ptr(), *t.stride()


def layer_grad(kind, left, right, forward):
    m, n, k = left.shape[0], right.shape[1], left.shape[1]
    out = torch.empty(m, n, device="cuda")
    size = entry("pam_hip_layer_grad_workspace_bytes", [_l] * 3, _z)(m, n, k)
    scratch = torch.empty(size // 4 + 4, device="cuda")
    call = entry("pam_hip_layer_grad", [_p, _l, _l] * 4 + [_l] * 3 + [_i, _f, _p, _z, _p])
    rc = call(*matrix(left), *matrix(right), *matrix(forward), *matrix(out), m, n, k, kind, 1.0, scratch.data_ptr(), size, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out


def one_chain(kind, left, right, forward):
    m, n, k = left.shape[0], right.shape[1], left.shape[1]
    out, stream = torch.empty(m, n, device="cuda"), torch.cuda.current_stream().cuda_stream
    _abi.load_library().pam_hip_set_tuning(32, 1)
    try:
        if kind == 0:
            rc = entry("pam_hip_pam_matmul_fwd", [_p, _l, _l] * 3 + [_l] * 3 + [_f, _p, _z, _p])(
                *matrix(left), *matrix(right), *matrix(out), m, n, k, 1.0, None, 0, stream)
        else:
            rc = entry("pam_hip_pam_matmul_bwd", [_p, _l, _l] * 4 + [_l] * 3 + [_i, _f, _p, _z, _p])(
                *matrix(left), *matrix(right), *matrix(forward), *matrix(out), m, n, k, int(kind == 1), 1.0, None, 0, stream)
    finally:
        _abi.load_library().pam_hip_set_tuning(0, 0)
    assert rc == 0
    return out


def in_order(kind, left, right, forward, n_planned=None, piece=None):
    """Pieces as the product's plan cuts them, each in equal chains of whole 32 terms, at most 1024; everything added from +0 upwards."""
    m, n, k = left.shape[0], right.shape[1], left.shape[1]
    piece = piece or min(_abi.gemm_plan(1, m, n_planned or n, k), (k + 31) // 32 * 32)
    tiles = (piece + 31) // 32
    chain = piece if piece <= 1024 else -(-tiles // -(-tiles // 32)) * 32
    total = torch.zeros(m, n, device="cuda")
    for p in range(0, k, piece):
        part = torch.zeros(m, n, device="cuda")
        for c in range(p, min(p + piece, k), chain):
            e = min(c + chain, p + piece, k)
            part += one_chain(kind, left[:, c:e], right[c:e], forward)
        total += part
    return total, piece, chain


def operand(generator, rows, cols, how):
    t = torch.randn(rows, cols, device="cuda", generator=generator)
    t[rows // 3] = 0.0
    t[rows // 2, cols // 2:cols // 2 + 3] = torch.tensor([0.0, 1e-39, -3e20], device="cuda")
    if how == "columns":
        return t.t().contiguous().t()
    if how == "odd address":
        return torch.empty(rows * cols + 1, device="cuda")[1:].view(rows, cols).copy_(t)
    if how == "every second":
        return torch.empty(rows, 2 * cols, device="cuda")[:, ::2].copy_(t)
    return t


LAYOUTS = [("rows", "rows"), ("rows", "columns"), ("columns", "rows"), ("columns", "columns"), ("odd address", "odd address"), ("every second", "rows")]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("m,n,k,layouts", [(*SIZES[0], LAYOUTS[:3]), (*SIZES[1], LAYOUTS[:1]), (*SIZES[2], LAYOUTS), (*SIZES[3], LAYOUTS[:1]), (*SIZES[4], LAYOUTS[:1])])
def test_gradients_are_added_in_chains(kind, m, n, k, layouts):
    generator = torch.Generator("cuda").manual_seed(k + kind)
    for left_how, right_how in layouts:
        left, right, forward = operand(generator, m, k, left_how), operand(generator, k, n, right_how), operand(generator, m, n, "rows")
        want, piece, chain = in_order(kind, left, right, forward)
        assert chain <= 1024 and (m == 40 or piece > chain)
        got = layer_grad(kind, left, right, forward)
        same = (got.view(torch.int32) == want.view(torch.int32)) | (got.isnan() & want.isnan())
        assert same.all(), (left_how, right_how, int((~same).sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("pieces,piece", [(1, 2528), (2, 1280), (3, 848)])
def test_chains_of_a_forced_depth(pieces, piece):
    """16-deep k-tiles, as a plan may have them: 157 in pieces of 157 and 79, which are longer than a chain and become 79 and 40 of 32, or 53."""
    generator = torch.Generator("cuda").manual_seed(pieces)
    left, right, forward = operand(generator, 100, 2500, "rows"), operand(generator, 2500, 70, "rows"), operand(generator, 100, 70, "rows")
    for kind in (0, 1, 2):
        want, _, chain = in_order(kind, left, right, forward, piece=piece)
        assert chain in (864, 640, 848)
        _abi.load_library().pam_hip_set_tuning(16, pieces)
        try:
            got = layer_grad(kind, left, right, forward)
        finally:
            _abi.load_library().pam_hip_set_tuning(0, 0)
        assert ((got.view(torch.int32) == want.view(torch.int32)) | (got.isnan() & want.isnan())).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2577, 2600, 2080), (1000, 2001, 3000), (6144, 6144, 1056)])
@pytest.mark.parametrize("how", ["rows", "odd address", "columns"])
def test_products_are_added_in_chains(m, n, k, how):
    generator = torch.Generator("cuda").manual_seed(m + k)
    x, w = operand(generator, m, k, how), operand(generator, n, k, how)
    bias, residual = torch.randn(n, device="cuda", generator=generator), torch.randn(m, n, device="cuda", generator=generator)
    kw = dict(approx_bwd=True)
    with torch.no_grad():
        z, piece, chain = in_order(0, x, w.t(), None)
        assert piece > chain and chain <= 1024
        z = z + bias
        assert_same_bits(pam.linear_act(x, w, bias, "silu", residual, **kw).cpu().numpy(), (chain_act(z, "silu", kw) + residual).cpu().numpy())
    y = pam.linear_act(x, w.clone().requires_grad_(), bias, "gelu", **kw)               # with z written
    assert_same_bits(y.detach().cpu().numpy(), chain_act(z, "gelu", kw).cpu().numpy())
    f = n // 2
    with torch.no_grad():
        z, _, _ = in_order(0, x, w[:2 * f].t(), None, (f + 1) // 2 * 4)
        want = pam.mul(chain_act(z[:, :f].contiguous(), "silu", kw), z[:, f:].contiguous())
        assert_same_bits(pam.gated_linear(x, w[:2 * f], **kw).cpu().numpy(), want.cpu().numpy())


@pytest.mark.gpu
def test_a_call_beyond_any_scratch():
    """The weight's gradient of 131 072 tokens: 256 tiles, whose pieces of 1024 terms each would be 537 MB."""
    x = torch.randn(131072, 1024, device="cuda").requires_grad_()
    w = torch.randn(1024, 1024, device="cuda").requires_grad_()
    y = pam.linear_act(x, w, approx_bwd=True)
    dy = torch.randn_like(y)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    dw, = torch.autograd.grad(y, w, dy)
    assert torch.cuda.max_memory_allocated() - before <= (64 << 20) + 2 * dw.numel() * 4
