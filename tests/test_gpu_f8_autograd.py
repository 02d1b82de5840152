"""GPU tier: the 8-bit operators and autograd: what has a gradient gives it, what has none says so."""
import pytest
import torch

import fp64_emu

pytestmark = pytest.mark.gpu

F32 = torch.float32


def test_second_derivatives_are_refused(dev):
    print("case second derivatives", flush=True)
    x, w = (torch.randn(40, 256, device=dev, requires_grad=True) for _ in range(2))
    (dx,) = torch.autograd.grad(fp64_emu.linear_f8(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.square().sum().backward()
    (dh,) = torch.autograd.grad(fp64_emu.swiglu_ckpt_f8(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dh.square().sum().backward()


def test_ops_without_a_gradient_say_so(dev):
    print("case no gradient", flush=True)
    h = torch.randn(40, 512, device=dev, requires_grad=True)
    q, s = fp64_emu.quant_f8(h.detach())
    _, hq, hs = fp64_emu.swiglu_f8(h.detach())
    scales = s.clone().requires_grad_()
    for call in (lambda: fp64_emu.quant_f8(h)[1], lambda: fp64_emu.quant_f8_tiles(h)[1],
                 lambda: fp64_emu.mm_f8(q, scales, q, s, out_dtype=F32),
                 lambda: fp64_emu.bmm_f8(q[None], scales[None], q[None], s[None], out_dtype=F32),
                 lambda: fp64_emu.swiglu_f8(h, keep=False)[0],
                 lambda: fp64_emu.swiglu_f8_backward(h[:, :256], hq, hs)):
        with pytest.raises(RuntimeError, match="not implemented"):
            call().sum().backward()
    out = torch.zeros(40, 40, device=dev)
    kept = torch.ones(40, 40, device=dev, requires_grad=True) * out
    assert out._version == 0
    fp64_emu.mm_f8(q, s, q, s, out=out)
    assert out._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        kept.sum().backward()                  # it had saved out
    with pytest.raises(RuntimeError, match="requires a gradient"):
        fp64_emu.mm_f8(q, scales, q, s, out=out)


def test_empty_last_dimension(dev):
    for shape, n in (((3, 4, 0), 5), ((0, 4, 256), 5), ((3, 256), 0), ((0, 0), 0)):
        print("case empty", shape, n, flush=True)
        x, w = torch.ones(shape, device=dev, requires_grad=True), torch.ones(n, shape[-1], device=dev, requires_grad=True)
        y = fp64_emu.linear_f8(x, w)
        assert y.shape == (*shape[:-1], n) and (y == 0).all()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and (dx == 0).all() and (dw == 0).all()
    for shape in ((3, 4, 0), (0, 256), (0, 0)):
        h = torch.ones(shape, device=dev, requires_grad=True)
        y = fp64_emu.swiglu_ckpt_f8(h)
        assert y.shape == (*shape[:-1], shape[-1] // 2)
        (dh,) = torch.autograd.grad(y, h, torch.ones_like(y))
        assert dh.shape == h.shape


def test_nothing_is_kept_without_gradients(dev):
    print("case no_grad", flush=True)
    x, w = (torch.randn(40, 256, device=dev, requires_grad=True) for _ in range(2))
    wq = fp64_emu.quant_f8_tiles(w.detach())
    want, y = fp64_emu.linear_f8(x, w).detach(), fp64_emu.swiglu_ckpt_f8(x).detach()
    for off in (torch.no_grad, torch.inference_mode):
        with off():
            assert torch.equal(fp64_emu.linear_f8(x, w), want) and torch.equal(fp64_emu.linear_f8(x, w, wq), want)
            assert torch.equal(fp64_emu.swiglu_ckpt_f8(x), y)


def test_empty_activation(dev):
    """With no elements each form gives its empty results."""
    for M, F in ((0, 256), (5, 0), (0, 0)):
        print("case empty activation", M, F, flush=True)
        h, dy = torch.empty(M, 2 * F, device=dev), torch.empty(M, F, device=dev)
        for keep in (False, True):
            for quant in (None, "rows", "both"):
                y, *_ = fp64_emu.swiglu_f8(h, quant=quant, keep=keep)
                assert y.shape == (M, F)
        _, hq, hs = fp64_emu.swiglu_f8(h)
        assert fp64_emu.swiglu_f8_backward(dy, hq, hs).shape == (M, 2 * F)
        q, s, qt, st = fp64_emu.swiglu_f8_backward(dy, hq, hs, quant="both")
        assert q.shape == (M, 2 * F) and qt.shape == (2 * F, M)
