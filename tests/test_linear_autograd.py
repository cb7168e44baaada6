"""What autograd sees of the matrix products, on the CPU: the launches are
replaced by host_products, everything around them runs as it is."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear
from tests import host_products


@pytest.fixture
def calls(monkeypatch):
    return host_products.install(monkeypatch)


def inputs(dtype=torch.float16):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4, 8, generator=g).to(dtype).requires_grad_()
    w = torch.randn(2, 3, 8, generator=g).to(dtype).requires_grad_()
    dy = torch.randn(6, 3, generator=g).to(dtype)
    offsets = torch.tensor([0, 2, 6], dtype=torch.int32)
    index = torch.tensor([0, 1, 1, 2, 3, 3], dtype=torch.int32)
    return x, w, dy, offsets, index


def reference(x, w, dy, offsets, index):
    xs, ws = x.detach().float().requires_grad_(), w.detach().float().requires_grad_()
    o = [int(v) for v in offsets]
    rows = xs[index.long()]
    y = torch.cat([rows[o[g] : o[g + 1]] @ ws[g].T for g in range(ws.shape[0])])
    y.backward(dy.float())
    return xs.grad, ws.grad


def assert_gradients(x, w, want):
    """Sums of at most 6 terms of magnitude below 16 in fp32, rounded to f16 once
    (2^-11 relative, and its subnormal step)."""
    for got, ref in zip((x.grad, w.grad), want):
        assert bool(((got.float() - ref).abs() <= 2.0**-11 * ref.abs() + 2.0**-16).all())


def test_gradients(calls):
    x, w, dy, offsets, index = inputs()
    linear.grouped_linear(x, w, offsets, index).backward(dy)
    assert_gradients(x, w, reference(x, w, dy, offsets, index))


@pytest.mark.parametrize("which", ["offsets", "index"])
def test_lists_written_between_forward_and_backward_are_refused(calls, which):
    """Routing buffers that the next layer's routing is written into."""
    x, w, dy, offsets, index = inputs()
    y = linear.grouped_linear(x, w, offsets, index, validate=False)
    if which == "offsets":
        offsets.copy_(torch.tensor([0, 6, 6], dtype=torch.int32))
    else:
        index.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_host_lists_are_read_once(calls):
    """The caller's list, or a tensor that had to be converted, may change after the
    forward: the gradients are those of the lists that it ran on."""
    x, w, dy, offsets, index = inputs()
    host, index64 = offsets.tolist(), index.to(torch.int64)
    y = linear.grouped_linear(x, w, host, index64)
    host[1] = 6
    index64.zero_()
    y.backward(dy)
    assert_gradients(x, w, reference(x, w, dy, offsets, index))


def test_lists_made_in_inference_mode(calls):
    x, w, dy, offsets, index = inputs()
    with torch.inference_mode():
        off, idx = offsets.clone(), index.clone()
    linear.grouped_linear(x, w, off, idx).backward(dy)
    assert_gradients(x, w, reference(x, w, dy, offsets, index))


@pytest.mark.parametrize("operand", ["x", "w", "dy"])
def test_a_second_derivative_is_refused(calls, operand):
    """A penalty on a gradient would lose the product's part: the gradients come
    from kernels that autograd does not see. dx depends on w and dy, dw on x and dy."""
    x, w, dy, offsets, index = inputs()
    if operand == "dy":
        dy.requires_grad_()
    y = linear.grouped_linear(x, w, offsets, index)
    (grad,) = torch.autograd.grad(y, w if operand == "x" else x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="has no gradient"):
        (y.float().sum() + grad.float().square().sum()).backward()


def test_a_first_derivative_may_keep_its_graph(calls):
    """create_graph for another term of the loss leaves the product's gradients usable."""
    x, w, dy, offsets, index = inputs()
    y = linear.grouped_linear(x, w, offsets, index)
    got = torch.autograd.grad(y, (x, w), dy, create_graph=True)
    x.grad, w.grad = (g.detach() for g in got)
    assert_gradients(x, w, reference(x, w, dy, offsets, index))
    (y.float().square().sum() + got[0].detach().float().sum()).backward()
