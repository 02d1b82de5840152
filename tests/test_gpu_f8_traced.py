"""GPU tier: the 8-bit operators under tracing: the fakes' shapes, strides and types are the kernels' own, and
compiled programs give the eager bits, gradients and written outputs among them."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fp64_emu
from f8_util import E4M3, E5M2, operand

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _same_layout(fn, *args):
    real = fn(*args)
    with FakeTensorMode() as mode:
        fake = fn(*(mode.from_tensor(a) if torch.is_tensor(a) else a for a in args))
    real, fake = ([t] if torch.is_tensor(t) else list(t) for t in (real, fake))
    assert len(real) == len(fake)
    for r, f in zip(real, fake):
        assert r.shape == f.shape and r.dtype == f.dtype and r.device == f.device
        if r.numel():
            assert r.stride() == f.stride() and r.storage_offset() == f.storage_offset(), (r.shape, r.stride(), f.stride())


@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (5, 777), (128, 256), (300, 130), (0, 64), (4, 0), (3, 40, 200), (1, 7, 129)])
def test_layouts_of_fakes(dev, shape):
    print("case fakes", shape, flush=True)
    x = torch.randn(shape, device=dev)
    for fmt in (E4M3, E5M2):
        for rows, cols in ((True, False), (False, True), (True, True)):
            _same_layout(lambda t: fp64_emu.quant_f8(t, rows=rows, cols=cols, fmt=fmt), x)
        _same_layout(lambda t: fp64_emu.quant_f8_tiles(t, transposed=True, fmt=fmt), x)
    q, s = fp64_emu.quant_f8(x)
    fn = fp64_emu.mm_f8 if x.dim() == 2 else fp64_emu.bmm_f8
    for dtype in (BF16, F32):
        _same_layout(lambda *a: fn(*a, out_dtype=dtype), q, s, q, s)
    if x.dim() == 2:
        h = torch.randn(shape[0], 2 * shape[1], device=dev)
        _, hq, hs = fp64_emu.swiglu_f8(h)
        for quant in (None, "rows", "both"):
            for keep in (True, False):
                _same_layout(lambda t: fp64_emu.swiglu_f8(t, quant=quant, keep=keep), h)
            _same_layout(lambda *a: fp64_emu.swiglu_f8_backward(*a, quant=quant), x, hq, hs)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_layers(dev, backend):
    print("case compiled layers", backend, flush=True)
    g = torch.Generator(dev).manual_seed(1)
    x = torch.randn(70, 256, device=dev, generator=g).to(BF16).requires_grad_()
    w1 = (torch.randn(384, 256, device=dev, generator=g) * 0.05).requires_grad_()
    w2 = (torch.randn(256, 192, device=dev, generator=g) * 0.05).requires_grad_()

    def net(x, w1, w2):
        return fp64_emu.linear_f8(fp64_emu.swiglu_ckpt_f8(fp64_emu.linear_f8(x, w1)), w2)

    y = net(x, w1, w2)
    dy = torch.randn(y.shape, device=dev, generator=g).to(BF16)
    want = torch.autograd.grad(y, (x, w1, w2), dy)
    torch._dynamo.reset()
    got_y = torch.compile(net, backend=backend, fullgraph=True)(x, w1, w2)
    got = torch.autograd.grad(got_y, (x, w1, w2), dy)
    assert torch.equal(got_y, y) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_operators(dev, backend):
    """Operators and a product added to a buffer, which the compiled program writes."""
    print("case compiled operators", backend, flush=True)
    x = torch.randn(200, 300, device=dev, generator=torch.Generator(dev).manual_seed(2))
    wq, ws = operand((130, 300), 3, tiles=True, device=dev)

    def step(x, out):
        q, s = fp64_emu.quant_f8(x)
        h = fp64_emu.mm_f8(q, s, wq, ws)
        fp64_emu.mm_f8(q, s, wq, ws, out=out, accumulate=True)
        return fp64_emu.swiglu_f8(h, quant="both")

    out, again = (torch.ones(200, 130, device=dev) for _ in range(2))
    want = step(x, out)
    torch._dynamo.reset()
    got = torch.compile(step, backend=backend, fullgraph=True)(x, again)
    assert torch.equal(out, again) and all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
