"""Autograd of the matrix products with the kernels themselves."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def inputs():
    g = torch.Generator().manual_seed(11)
    x = torch.randn(9, 64, generator=g).to(torch.bfloat16)
    w = torch.randn(3, 40, 64, generator=g).to(torch.bfloat16)
    dy = torch.randn(20, 40, generator=g).to(torch.bfloat16)
    index = torch.randint(0, 9, (20,), generator=g, dtype=torch.int32)
    return x, w, dy, torch.tensor([0, 7, 7, 20], dtype=torch.int32), index


@pytest.mark.parametrize("x_at,w_at", [("cpu", DEV), (DEV, "cpu"), ("cpu", "cpu")])
def test_gradients_are_on_their_operands_devices(x_at, w_at):
    """Rows staged from the host, experts on the device, and the other way round."""
    x, w, dy, off, idx = inputs()
    want = []
    for a, b in ((DEV, DEV), (x_at, w_at)):
        xg, wg = x.to(a).detach().requires_grad_(), w.to(b).detach().requires_grad_()
        y = linear.grouped_linear(xg, wg, off, idx)
        assert y.device == xg.device
        y.backward(dy.to(y.device))
        assert xg.grad.device == xg.device and wg.grad.device == wg.device
        want.append((xg.grad.cpu(), wg.grad.cpu()))
    assert all(torch.equal(p, q) for p, q in zip(*want))


@pytest.mark.parametrize("which", ["offsets", "index"])
def test_routing_written_again_before_the_backward(which):
    """A device buffer is refused, a host list is the one the forward ran on."""
    x, w, dy, off, idx = inputs()
    xg, wg = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    offd, idxd = off.to(DEV), idx.to(DEV)
    y = linear.grouped_linear(xg, wg, offd, idxd, validate=False)
    (offd if which == "offsets" else idxd).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy.to(DEV))
    host = off.tolist()
    y = linear.grouped_linear(xg, wg, host, idx.to(DEV))
    host[1] = 20
    y.backward(dy.to(DEV))
    assert torch.equal(wg.grad, linear.grouped_linear_wgrad(dy.to(DEV), x.to(DEV), off, idx.to(DEV)))
    assert torch.equal(xg.grad, linear.grouped_linear_dgrad(dy.to(DEV), w.to(DEV), off, idx.to(DEV), 9))
