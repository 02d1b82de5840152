"""GPU tier: the operators around the 8-bit products under tracing: the fakes' shapes, strides and types are
the kernels' own, and compiled programs give the eager bits, gradients among them."""
import pytest
import torch

import fp64_emu
from f8_block_util import randn, rng
from f8_util import operand
from test_gpu_f8_traced import _same_layout

pytestmark = pytest.mark.gpu

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
FORMS = (None, "rows", "both")


@pytest.mark.parametrize("M,D", [(1, 1), (1, 128), (5, 777), (128, 256), (300, 130), (0, 64), (2, 9000)])
def test_layouts_of_fakes(dev, M, D):
    print("case block fakes", M, D, flush=True)
    r, y, w, state = torch.randn(M, D, device=dev), torch.randn(M, D, device=dev).to(BF16), torch.randn(D, device=dev), rng(1, 0, dev)
    stats = torch.ones(2, M, device=dev)
    for quant in FORMS:
        for keep in (True, False):
            _same_layout(lambda *a: fp64_emu.norm_f8(*a, quant=quant, keep=keep), r, w)
            _same_layout(lambda r, w, y, s: fp64_emu.norm_f8(r, w, y, w, y, 0.5, 0.1, s, quant, keep), r, w, y, state)
        _same_layout(lambda x, s: fp64_emu.dropout_f8(x, 0.1, s, quant), y, state)
        for bias in (True, False):
            _same_layout(lambda d, h: fp64_emu.act_f8_backward(d, h, "silu", quant, bias), y, y)
    for gate in (w, y):
        _same_layout(lambda y, r, w, s, g: fp64_emu.norm_f8_backward(y, r, r, w, s, y, w, g), y, r, w, stats, gate)
    _same_layout(lambda r, w, s: [t for t in fp64_emu.norm_f8_backward(r, None, r, w, s) if t is not None], r, w, stats[:1])
    q, s = fp64_emu.quant_f8(r)
    for dtype in (BF16, F32):
        bias, res = torch.randn(M, device=dev), torch.randn(M, M, device=dev).to(dtype)
        for keep in (True, False):
            _same_layout(lambda q, s, b, r: fp64_emu.mm_f8(q, s, q, s, dtype, bias=b, act="gelu", residual=r, keep=keep), q, s, bias, res)
    q, s = fp64_emu.quant_f8(r[None])
    _same_layout(lambda q, s: fp64_emu.bmm_f8(q, s, q, s, act="relu", keep=True), q, s)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_block(dev, backend):
    print("case compiled block", backend, flush=True)
    t = {n: randn(*s, seed=i, scale=k).to(dev) for i, (n, s, k) in enumerate(
        [("r", (70, 256), 1.0), ("w", (256,), 1.0), ("v", (256,), 1.0), ("u", (384, 256), 0.05), ("b", (384,), 0.1), ("d", (256, 384), 0.05)])}
    leaves = [v.requires_grad_() for v in t.values()]
    state = rng(3, 4, dev)

    def net(r, w, v, u, b, d, state):
        x = fp64_emu.residual_norm_f8(r, w)
        h = fp64_emu.seeded_dropout_f8(fp64_emu.linear_f8(x, u, bias=b, act="silu"), 0.25, state)
        return fp64_emu.residual_norm_f8(r, v, fp64_emu.linear_f8(h, d, residual=x), w, v, 0.5, 0.1, state)

    want = net(*leaves, state)
    dy = [randn(70, 256, seed=9 + i).to(dev) for i in range(2)]
    grads = torch.autograd.grad(want, leaves, dy)
    torch._dynamo.reset()
    got = torch.compile(net, backend=backend, fullgraph=True)(*leaves, state)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, dy), grads))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_operators(dev, backend):
    print("case compiled block operators", backend, flush=True)
    r, y, w = randn(130, 300, seed=1).to(dev), randn(130, 300, seed=2, dtype=FP16).to(dev), randn(300, seed=3).to(dev)
    wq, ws = operand((64, 300), 3, tiles=True, device=dev)
    state = rng(5, 6, dev)

    def step(r, y, w, state):
        new, q, s, qt, st, stats = fp64_emu.norm_f8(r, w, y, w, w, 0.5, 0.25, state, "both", True)
        out, h = fp64_emu.mm_f8(q, s, wq, ws, bias=w[:64], act="gelu_tanh", keep=True)
        got = fp64_emu.act_f8_backward(out, h, "gelu_tanh", "rows", bias=True)
        return [new, qt, st, stats, out, h, *got, *fp64_emu.dropout_f8(y, 0.5, state)]

    want = step(r, y, w, state)
    torch._dynamo.reset()
    got = torch.compile(step, backend=backend, fullgraph=True)(r, y, w, state)
    assert len(got) == len(want) and all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_shared_gates(dev, backend):
    print("case compiled shared gates", backend, flush=True)
    t = [randn(*s, seed=i).to(dev) for i, s in enumerate([(3, 50, 256), (256,), (3, 50, 256), (3, 1, 256), (3, 50, 1)])]
    leaves = [v.requires_grad_() for v in t]

    def net(r, w, y, g, h):
        new, x = fp64_emu.residual_norm_f8(r, w, y, gate=g)
        return fp64_emu.residual_norm_f8(new, w, x.to(BF16), gate=h)

    want = net(*leaves)
    dy = [randn(3, 50, 256, seed=9 + i, dtype=v.dtype).to(dev) for i, v in enumerate(want)]
    grads = torch.autograd.grad(want, leaves, dy)
    torch._dynamo.reset()
    got = torch.compile(net, backend=backend, fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, dy), grads))


def test_layouts_of_fakes_of_sums(dev):
    """The forms that autograd uses: a gate's gradient in float32, a bias's gradient alone."""
    print("case fakes of sums", flush=True)
    r, w, stats = randn(70, 300, seed=1).to(dev), randn(300, seed=2).to(dev), torch.ones(1, 70, device=dev)
    y = r.to(BF16)
    ops = torch.ops.fp64_emu
    _same_layout(lambda r, w, y, s: ops.fp64_emu_norm_f8_backward(y, r, r, w, s, y, None, y, 1.0, 0, None, True), r, w, y, stats)
    _same_layout(lambda r: ops.fp64_emu_act_f8_backward(r, None, 0, 3, True), r)
