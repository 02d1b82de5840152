"""GPU tier: the gated MLP that runs the 8-bit operators together
(fp64-emu_amd/callers/f8_mlp.py): its step's outputs and gradients against
float32, training beside float32 training, single tokens against the batch."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "fp64-emu_amd"))
from callers import f8_mlp  # noqa: E402

pytestmark = pytest.mark.gpu


def _off(got, want):
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


@pytest.mark.parametrize("d,f,tokens", [(256, 384, 300), (200, 130, 77)])
def test_step_beside_float32(dev, d, f, tokens):
    """Each operand of a product is off by at most 2^-4 of its elements, about 2.6% in norm (a
    uniform error over half-steps between 2^-5 and 2^-4), so a product of two by 3.7%; the step
    chains at most three of them and the activation: 10%."""
    print("case f8 mlp step", d, f, tokens, flush=True)
    net = f8_mlp.GatedMlp(d, f)
    plain = f8_mlp.PlainMlp(net)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(tokens, d, generator=g).to(dev, torch.bfloat16)
    dout = (torch.randn(tokens, d, generator=g) * 1e-3).to(dev, torch.bfloat16)
    out, kept = net.forward(x)
    dx = net.backward(dout, kept)
    xf = x.float().requires_grad_()
    want = plain.forward(xf)
    wx, w1, w2 = torch.autograd.grad(want, (xf, plain.w1, plain.w2), dout.float())
    for name, a, b in (("out", out, want), ("dx", dx, wx), ("dw1", net.g1, w1), ("dw2", net.g2, w2)):
        print(name, _off(a, b), flush=True)
        assert _off(a, b) < 0.10, name
    # Gradients are added to what is there: a second step doubles them.
    once = net.g2.clone()
    net.backward(dout, net.forward(x)[1])
    assert _off(net.g2, 2 * once) < 1e-6
    # What waits for the backward pass takes a byte an element and its scales.
    held = sum(t.numel() * t.element_size() for pair in kept for t in pair)
    blocks = lambda n: -(-n // 128)  # noqa: E731
    assert held <= tokens * (d + 3 * f) + 4 * (d * blocks(tokens) + f * blocks(tokens) + 2 * tokens * blocks(f))


def test_single_tokens(dev):
    """A token by itself takes other kernels than in a batch: the same codes, sums in another order."""
    print("case f8 mlp token", flush=True)
    net = f8_mlp.GatedMlp(512, 640)
    x = torch.randn(300, 512, generator=torch.Generator().manual_seed(6)).to(dev, torch.bfloat16)
    batch, _ = net.forward(x)
    for i in (0, 7, 299):
        # one bfloat16 rounding apart, and what a changed h moves past a code's edge: 2%
        assert _off(net.serve(x[i:i + 1]), batch[i:i + 1]) < 0.02


def test_training_keeps_up(dev):
    """The loss of 8-bit training falls as float32's does: to within a quarter of the start
    above it."""
    print("case f8 mlp training", flush=True)
    loss = f8_mlp.train()
    print(loss, flush=True)
    assert loss["plain"] < 0.5 * loss["start"]
    assert loss["f8"] < loss["plain"] + 0.25 * loss["start"]
