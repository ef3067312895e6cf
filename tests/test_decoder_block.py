"""The decoder block and the example that trains one: the operators together."""
import importlib.util
import pathlib

import pytest
import torch

from pam_amd.blocks import Attention, DecoderBlock, GatedFeedForward


def example():
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "decoder_lm.py"
    spec = importlib.util.spec_from_file_location("decoder_lm", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_parameters_and_refusals():
    block = DecoderBlock(32, 4, 2, 8, 48)
    shapes = {name: tuple(p.shape) for name, p in block.named_parameters()}
    assert shapes["attention.qkv"] == (64, 32) and shapes["attention.out"] == (32, 32) and shapes["attention.q_weight"] == (8,)
    assert shapes["feed_forward.gate_up"] == (96, 32) and shapes["feed_forward.down"] == (32, 48)
    with pytest.raises(ValueError):
        Attention(32, 4, 3, 8)
    with pytest.raises(RuntimeError):                    # no fallback
        GatedFeedForward(8, 8)(torch.ones(1, 8))


@pytest.mark.gpu
def test_the_example_learns_and_continues():
    lm = example()
    torch.manual_seed(0)
    model = lm.Decoder().cuda()
    generator = torch.Generator().manual_seed(1)
    losses = lm.train(model, 60, generator, report=None)
    assert losses[0] > 3.5 and sum(losses[-5:]) / 5 < 0.5 * losses[0]
    # the cached pass computes what the whole one does, up to the order of the sums (kernels for few rows) amplified by two blocks
    tokens = lm.batch(generator, 3)[:, :20]
    with torch.no_grad():
        whole = model(tokens)
        caches = [{} for _ in model.blocks]
        parts = [model(tokens[:, :11], caches)] + [model(tokens[:, i:i + 1], caches) for i in range(11, 20)]
    cached = torch.cat(parts, 1)
    assert (cached - whole).abs().max() <= 1e-4 * whole.abs().max()
    assert lm.continue_sequence(model, tokens[:, :5], 4).shape == (3, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("approx", [True, False])
def test_gradients_reach_every_parameter(approx):
    torch.manual_seed(3)
    block = DecoderBlock(32, 4, 2, 8, 48, approx_bwd=approx).cuda()
    lm = example()
    cos, sin = lm.pam.rotary_tables(10, 8, device="cuda")
    x = torch.randn(2, 10, 32, device="cuda", requires_grad=True)
    block(x, cos, sin).square().sum().backward()
    for name, p in [("x", x), *block.named_parameters()]:
        assert p.grad is not None and p.grad.isfinite().all() and p.grad.abs().max() > 0, name
