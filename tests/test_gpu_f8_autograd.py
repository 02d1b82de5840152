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
