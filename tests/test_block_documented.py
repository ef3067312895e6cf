"""What the documentation shows of the decoder block's operators, as a program that has imported the package and nothing else writes it."""
import subprocess
import sys

import pytest
import torch

import pam_amd as pam


def test_the_package_alone_reaches_its_modules():
    """In a process of its own: here other tests have imported them."""
    code = "import pam_amd as pam; pam.optim.clip_grad_norm_, pam.optim.Adam, pam.blocks.DecoderBlock, pam.rotary_tables"
    subprocess.run([sys.executable, "-c", code], check=True)


@pytest.mark.gpu
def test_a_step_as_documented():
    model = torch.nn.ParameterDict({name: torch.randn(*shape, device="cuda") * 0.1 for name, shape in
                                    dict(wq=(128,), wk=(128,), gate_up=(192, 64), down=(64, 96)).items()})
    q, k, x = (torch.randn(*shape, device="cuda") for shape in ((2, 5, 4, 128), (2, 5, 2, 128), (2, 5, 64)))
    positions = torch.arange(5, device="cuda")
    cos, sin = pam.rotary_tables(4096, 128, device="cuda")
    q, k = pam.rotary(q, k, cos, sin, positions, q_weight=model["wq"], k_weight=model["wk"])
    h = pam.gated_linear(x, model["gate_up"], activation="silu")
    y = pam.linear_act(h, model["down"], residual=x)
    (y.sum() + q.sum() + k.sum()).backward()
    norm = pam.optim.clip_grad_norm_(model.parameters(), 1.0)
    assert float(norm) > 1.0 and all(p.grad.isfinite().all() for p in model.parameters())
    assert float(pam.optim.grad_norm([p.grad for p in model.parameters()])) < 1.3          # (quotient, products and root each off by up to an eighth)
    pam.optim.Adam(list(model.parameters()), opt_functional_cfg="pam").step()
