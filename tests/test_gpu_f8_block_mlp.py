"""GPU tier: the block around the gated MLP (fp64-emu_amd/callers/f8_mlp.py), which runs the norms,
the dropout and the 8-bit operators together: its step against float32 autograd with the same mask, single
tokens against the batch, a captured step."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fp64-emu_amd"))
from callers import f8_mlp  # noqa: E402
from f8_block_util import factors, rng  # noqa: E402

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _off(got, want):
    return ((got.float() - want.float()).norm() / want.float().norm()).item()


def _norm(v, w):
    return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w


def _plain(block, r, drop):
    """(r', x') in float32, and the leaves that need gradients."""
    mlp = f8_mlp.PlainMlp(block.mlp)
    leaves = {n: getattr(block, n).clone().requires_grad_() for n in block.NAMES}
    y = mlp.forward(_norm(r, leaves["w0"]))
    new = r + leaves["gate"] * drop * _norm(y, leaves["post"])
    return new, _norm(new, leaves["w1"]), {**leaves, "w1_mlp": mlp.w1, "w2_mlp": mlp.w2}


def _inputs(d, tokens, dev):
    g = torch.Generator().manual_seed(5)
    return [(torch.randn(tokens, d, generator=g) * scale).to(dev, BF16) for scale in (1.0, 1e-3, 1e-3)]


@pytest.mark.parametrize("d,f,tokens,p", [(256, 384, 300, 0.1), (200, 130, 77, 0.5), (1152, 256, 40, 0.0)])
def test_block_beside_float32(dev, d, f, tokens, p):
    """An operand of a product is off by about 2.6% in norm, a product by 3.7%; the step chains at most three of them,
    the activation and the norms' slopes: 12%.  The stream itself keeps r: half of that."""
    print("case f8 block step", d, f, tokens, p, flush=True)
    block, state = f8_mlp.Block(d, f, p=p), rng(9, 2, dev)
    r, dnew, dout = _inputs(d, tokens, dev)
    new, out, kept = block.forward(r, state)
    dr = block.backward(dnew, dout, kept)
    rf = r.float().requires_grad_()
    drop = factors(9, 2, p, tokens, d).float().to(dev)
    wnew, wout, leaves = _plain(block, rf, drop)
    want = dict(zip(("r", *leaves), torch.autograd.grad((wnew, wout), (rf, *leaves.values()), (dnew.float(), dout.float()))))
    assert _off(new, wnew) < 0.06 and _off(out, wout) < 0.06
    assert _off(dr, want["r"]) < 0.12
    for name in block.NAMES:
        print(name, _off(block.g[name], want[name]), flush=True)
        assert _off(block.g[name], want[name]) < 0.12, name
    assert _off(block.mlp.g1, want["w1_mlp"]) < 0.12 and _off(block.mlp.g2, want["w2_mlp"]) < 0.12


def test_block_tokens(dev):
    """A token by itself, nothing dropped, against the batch: other kernels, the same formulas."""
    print("case f8 block token", flush=True)
    block = f8_mlp.Block(512, 640, p=0.0)
    r = _inputs(512, 300, dev)[0]
    new, out, _ = block.forward(r, None)
    for i in (0, 7, 299):
        # one bfloat16 rounding apart, and what a changed h moves past a code's edge: 2%
        a, b = block.serve(r[i:i + 1])
        assert _off(a, new[i:i + 1]) < 0.02 and _off(b, out[i:i + 1]) < 0.02


def test_block_step_captured(dev):
    """The whole step in a graph, replayed with other masks: each replay gives the eager step's bits."""
    print("case f8 block graph", flush=True)
    r, dnew, dout = _inputs(256, 200, dev)
    block, state = f8_mlp.Block(256, 384), rng(1, 0, dev)

    def step():
        for g in (*block.g.values(), block.mlp.g1, block.mlp.g2):
            g.zero_()
        new, out, kept = block.forward(r, state)
        return [new, out, block.backward(dnew, dout, kept)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    grads = [*block.g.values(), block.mlp.g1, block.mlp.g2]
    for turn in range(3):
        state += torch.tensor([0, 1], device=dev)
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in (*got, *grads)]
        want = [*step(), *grads]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(seen, want)), turn
