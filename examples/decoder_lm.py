"""A small decoder-only language model in PAM arithmetic: trains on sequences that count upwards by a step of their own, then
continues one, token by token, from a cache.

    python examples/decoder_lm.py [--steps 200]
"""
import argparse
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))
import pam_amd as pam                                    # noqa: E402
from pam_amd.blocks import DecoderBlock                  # noqa: E402
from pam_amd.optim import Adam, clip_grad_norm_          # noqa: E402

VOCABULARY, LENGTH = 61, 32


class Decoder(torch.nn.Module):
    def __init__(self, vocabulary=VOCABULARY, width=64, heads=4, kv_heads=2, dim=16, hidden=128, blocks=2, length=LENGTH):
        super().__init__()
        kw = dict(approx_bwd=True)
        self.embedding = torch.nn.Embedding(vocabulary, width)
        torch.nn.init.normal_(self.embedding.weight, std=width ** -0.5)
        self.blocks = torch.nn.ModuleList(DecoderBlock(width, heads, kv_heads, dim, hidden, **kw) for _ in range(blocks))
        self.norm = pam.LayerNorm(width, **kw)
        cos, sin = pam.rotary_tables(length, dim, device="cpu")
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)

    def forward(self, tokens, caches=None):
        x = self.embedding(tokens)
        for i, block in enumerate(self.blocks):
            x = block(x, self.cos, self.sin, None if caches is None else caches[i])
        return pam.linear(self.norm(x), self.embedding.weight, approx_bwd=True)


def batch(generator, size):
    start, step = (torch.randint(low, high, (size, 1), generator=generator) for low, high in ((0, VOCABULARY), (1, 8)))
    return ((start + step * torch.arange(LENGTH)) % VOCABULARY).cuda()


def train(model, steps, generator, report=print):
    optimizer = Adam(list(model.parameters()), lr=3e-3, betas=(0.9, 0.98), opt_functional_cfg="pam")
    losses = []
    for i in range(steps):
        tokens = batch(generator, 32)
        log_p = pam.log_softmax(model(tokens[:, :-1]), dim=-1, approx_bwd=True)
        loss = -log_p.gather(-1, tokens[:, 1:, None]).mean()
        optimizer.zero_grad()
        loss.backward()
        norm = clip_grad_norm_(model.parameters(), 1.0)
        optimizer.step()
        losses.append(loss.item())
        if report and (i % 20 == 0 or i == steps - 1):
            report(f"step {i:4d}  loss {losses[-1]:.3f}  gradient norm {float(norm):.3f}")
    return losses


@torch.no_grad()
def continue_sequence(model, prompt, count):
    """The prompt at once, then a token at a time from the caches."""
    caches = [{} for _ in model.blocks]
    tokens, fed = prompt, prompt
    for _ in range(count):
        fed = model(fed, caches)[:, -1].argmax(-1, keepdim=True)
        tokens = torch.cat((tokens, fed), 1)
    return tokens


def main():
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--steps", type=int, default=200)
    steps = parser.parse_args().steps
    torch.manual_seed(0)
    model = Decoder().cuda()
    generator = torch.Generator().manual_seed(1)
    train(model, steps, generator)
    sequence = batch(generator, 4)
    print("prompt and continuation:", *continue_sequence(model, sequence[:, :8], 16).tolist(), sep="\n  ")
    print("as it goes on:", *sequence[:, :24].tolist(), sep="\n  ")


if __name__ == "__main__":
    main()
