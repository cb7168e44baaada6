"""What autograd sees of the matrix products, on the CPU: the launches are
replaced by host_products, everything around them runs as it is."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from mlx_gptq import linear
from mlx_gptq.experts import ExpertMLP
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


def mx_inputs():
    return torch.zeros(3, 4, dtype=torch.int32), torch.full((3, 1), 127, dtype=torch.uint8)


def int8_inputs():
    return torch.ones(3, 32, dtype=torch.int8), torch.ones(3)


def products(x):
    """Every product whose weight has no gradient, of rows x [4, 32]."""
    words, scales = mx_inputs()
    w8, ws = int8_inputs()
    yield linear.mxfp_linear(x, words, scales, "mxfp4")
    yield linear.int8_linear(*linear.quantize_rows_int8(x), w8, ws)


def test_rows_of_quantized_products_do_not_lose_their_gradient_silently(calls):
    x = torch.ones(4, 32, dtype=torch.bfloat16, requires_grad=True)
    for y in products(x):  # the forward runs
        assert y.requires_grad
        with pytest.raises(NotImplementedError, match="no gradient"):
            y.float().sum().backward()
    for y in products(x.detach()):
        assert not y.requires_grad
    with torch.no_grad():
        for y in products(x):
            assert not y.requires_grad


@pytest.mark.parametrize("name", ["x_scale", "w_scale", "bias"])
def test_int8_scales_and_bias_do_not_lose_their_gradient_silently(calls, name):
    w8, ws = int8_inputs()
    args = {"x_scale": torch.ones(4), "w_scale": ws, "bias": torch.zeros(3)}
    args[name].requires_grad_()
    y = linear.int8_linear(torch.ones(4, 32, dtype=torch.int8), args["x_scale"], w8, args["w_scale"],
                           args["bias"])
    with pytest.raises(NotImplementedError, match="no gradient"):
        y.float().sum().backward()


def test_int8_weights_rounded_from_parameters_are_constants(calls):
    """ExpertMLP.from_weights takes a module's parameters; a training program's loss
    may reach other tensors past them."""
    w = torch.ones(2, 64, 32, dtype=torch.bfloat16, requires_grad=True)
    mlp = ExpertMLP.from_weights(w, torch.ones(2, 32, 32, dtype=torch.bfloat16), "int8")
    assert not any(t.requires_grad for t in (*mlp.gate_up, *mlp.down))


def test_a_tangent_is_refused(calls):
    """Forward-mode derivatives: a result without a tangent would read as a constant."""
    x, w, dy, offsets, index = (t.detach() for t in inputs())
    rows = torch.ones(4, 32, dtype=torch.bfloat16)
    w8, ws = int8_inputs()
    q = torch.ones(4, 32, dtype=torch.int8)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for call in (lambda: linear.grouped_linear(dual(x), w, offsets, index),
                     lambda: linear.grouped_linear(x, dual(w), offsets, index),
                     lambda: linear.grouped_linear(x.requires_grad_(), dual(w), offsets, index),
                     lambda: linear.grouped_linear_dgrad(dual(dy), w, offsets, index, 4),
                     lambda: linear.grouped_linear_wgrad(dy, dual(x.detach()), offsets, index),
                     lambda: linear.mxfp_linear(dual(rows), *mx_inputs(), "mxfp4"),
                     lambda: linear.quantize_rows_int8(dual(rows)),
                     lambda: linear.int8_linear(q, torch.ones(4), w8, dual(ws))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        linear.grouped_linear(x.detach(), w, offsets, index)  # no tangent: runs


@pytest.mark.parametrize("which", ["x", "w"])
def test_only_what_the_gradient_reads_is_saved(calls, which):
    """Frozen experts keep no rows alive, frozen rows no weight."""
    x, w, dy, offsets, index = inputs()
    want = reference(x, w, dy, offsets, index)
    (w if which == "x" else x).requires_grad_(False)
    y = linear.grouped_linear(x, w, offsets, index)
    saved = [t for t in y.grad_fn.saved_tensors if t is not None and t.is_floating_point()]
    assert len(saved) == 1 and saved[0].shape == (w if which == "x" else x).shape
    y.backward(dy)
    got, ref = (x.grad, want[0]) if which == "x" else (w.grad, want[1])
    assert bool(((got.float() - ref).abs() <= 2.0**-11 * ref.abs() + 2.0**-16).all())
    assert (w if which == "x" else x).grad is None


def test_results_without_a_gradient_can_be_written_in_place(calls):
    """A residual added in place, as to any operator's result."""
    x = torch.ones(4, 32, dtype=torch.bfloat16, requires_grad=True)
    for y in products(x):
        before = y.detach().clone()
        y += 2.0
        y[0] = 0.0
        assert torch.equal(y[1:].detach(), before[1:] + 2.0) and y.requires_grad
        with pytest.raises(NotImplementedError, match="no gradient"):
            y.float().sum().backward()
    q, s = linear.quantize_rows_int8(x)
    s.mul_(2.0)
