"""CPU tier: the 8-bit operators and autograd.  The layer's and the checkpoint's autograd forms run on host
stand-ins of the ops (the tests' plain forms); the ops themselves are seen with fake tensors."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import fp64_emu
from fp64_emu import f8
from f8_util import BLOCK, E4M3, quantised, values

F32 = torch.float32


def _quant(x, rows, cols, tiles, fmt):
    CALLS.append(("quant", rows, cols, tiles))
    tall, out = BLOCK if tiles else 1, []
    if rows:
        out += quantised(x, fmt, tall)
    if cols:
        out += quantised(x.t(), fmt, tall)
    return out


def _mm(A, sA, B, sB, dtype):
    return (values(A, sA) @ values(B, sB).t()).to(dtype)


def _kept(h):
    F = h.shape[1] // 2
    halves = [quantised(v, E4M3) for v in (h[:, :F], h[:, F:])]
    return [torch.cat([a.view(torch.uint8) for a, _ in halves], 1).view(E4M3), torch.cat([s for _, s in halves], 1)]


def _swiglu(h, quant, keep):
    CALLS.append(("swiglu", keep))
    g, u = h.detach().double().chunk(2, 1)
    return [(g * torch.sigmoid(g) * u).to(h.dtype)] + (_kept(h) if keep else [])


def _swiglu_backward(dy, hq, hs, quant):
    F, blocks = dy.shape[1], hs.shape[1] // 2
    g, u = values(hq[:, :F], hs[:, :blocks]), values(hq[:, F:], hs[:, blocks:])
    s = torch.sigmoid(g)
    return [torch.cat((dy * u * s * (1 + g * (1 - s)), dy * g * s), 1).to(dy.dtype)]


CALLS = []


@pytest.fixture
def host(monkeypatch):
    """The ops on the host, and what they were asked for."""
    CALLS.clear()
    for name, fn in (("_quant", _quant), ("_mm", _mm), ("_swiglu", _swiglu), ("_swiglu_backward", _swiglu_backward)):
        monkeypatch.setattr(f8, name, fn)
    return CALLS


def _leaf(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).requires_grad_()


def test_second_derivatives_are_refused(host):
    """The backward passes are not differentiable: a penalty on a gradient fails instead of losing its term."""
    x, w = _leaf(8, 256), _leaf(40, 256, seed=1)
    (dx,) = torch.autograd.grad(fp64_emu.linear_f8(x, w).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.square().sum().backward()
    h = _leaf(8, 256, seed=2)
    (dh,) = torch.autograd.grad(fp64_emu.swiglu_ckpt_f8(h).square().sum(), h, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dh.square().sum().backward()


def test_ops_without_a_gradient_say_so():
    """The operators' results carry a gradient function that raises (NotImplemented), not one that warns and gives
    nothing; the passes that would reach it run on the GPU tier."""
    with FakeTensorMode():
        h = torch.empty(4, 512, device="cuda", requires_grad=True)
        q, s = (torch.empty(4, 256, dtype=E4M3, device="cuda"), torch.empty(4, 2, device="cuda", requires_grad=True))
        for call in (lambda: fp64_emu.quant_f8(h)[1], lambda: fp64_emu.quant_f8_tiles(h)[1],
                     lambda: fp64_emu.mm_f8(q, s, q, s.detach(), out_dtype=F32),
                     lambda: fp64_emu.bmm_f8(q[None], s[None], q[None], s.detach()[None], out_dtype=F32),
                     lambda: fp64_emu.swiglu_f8(h, keep=False)[0],
                     lambda: fp64_emu.swiglu_f8_backward(h, torch.empty(4, 1024, dtype=E4M3, device="cuda"),
                                                         torch.empty(4, 8, device="cuda"))):
            assert call().grad_fn.name().endswith("::NotImplemented")
            with torch.no_grad():
                assert not call().requires_grad


def test_out_counts_as_written():
    """A product into `out` raises its version; an out or scales that require a gradient are refused."""
    with FakeTensorMode():
        q, s = torch.empty(4, 256, dtype=E4M3, device="cuda"), torch.empty(4, 2, device="cuda")
        out = torch.empty(4, 4, device="cuda")
        before = out._version
        fp64_emu.mm_f8(q, s, q, s, out=out, accumulate=True)
        assert out._version == before + 1
        leaf = torch.empty(4, 4, device="cuda", requires_grad=True)
        for o, scales in ((leaf, s), (leaf * 2, s), (out, s.clone().requires_grad_())):
            with pytest.raises(RuntimeError, match="requires a gradient"):
                fp64_emu.mm_f8(q, scales, q, s, out=o)
        with torch.no_grad():
            fp64_emu.mm_f8(q, s, q, s, out=leaf)
            assert leaf._version == 1


def test_nothing_is_kept_without_gradients(host):
    """Under no_grad a layer of parameters quantises what the forward product reads and no more, and takes a
    weight without its transposed half."""
    x, w = _leaf(8, 256), _leaf(40, 256, seed=1)
    wq = tuple(_quant(w, True, False, True, E4M3))
    want = fp64_emu.linear_f8(x, w).detach()
    for off in (torch.no_grad, torch.inference_mode):
        host.clear()
        with off():
            assert torch.equal(fp64_emu.linear_f8(x, w), want)
            assert host == [("quant", True, False, False), ("quant", True, False, True)]
            assert torch.equal(fp64_emu.linear_f8(x, w, wq), want)
            host.clear()
            fp64_emu.swiglu_ckpt_f8(x)
            assert host == [("swiglu", False)]
    with pytest.raises(ValueError, match="transposed half"):
        fp64_emu.linear_f8(x, w, wq)


def test_empty_last_dimension(host):
    """No elements to sum: zeros; no rows and no outputs: empty results, and gradients of their shapes."""
    for shape, n in (((3, 4, 0), 5), ((0, 4, 256), 5), ((3, 256), 0), ((0, 0), 0)):
        x, w = _leaf(*shape), _leaf(n, shape[-1], seed=1)
        y = fp64_emu.linear_f8(x, w)
        assert y.shape == (*shape[:-1], n) and (y == 0).all()
        dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and (dx == 0).all() and (dw == 0).all()
    for shape in ((3, 4, 0), (0, 256), (0, 0)):
        h = _leaf(*shape)
        y = fp64_emu.swiglu_ckpt_f8(h)
        assert y.shape == (*shape[:-1], shape[-1] // 2)
        (dh,) = torch.autograd.grad(y, h, torch.ones_like(y))
        assert dh.shape == h.shape
