"""The router's choice and its gradient.

The choice is exact: the order of the logits, the lower index first among equal ones.
Weights are w = exp(l - m) / Z in fp32: l - m is off by 2^-24 |l - m| (an argument's
error is a factor of the exponential), expf by 2^-23, the sum of up to 1024 terms by
1024 2^-24 relative (all are positive) and the division by 2^-24:
(|l - m| + E + 8) 2^-24 relative, with a subnormal step of 2^-149. The gradient's terms
carry two such factors, its inner sum over k another; rounding it to the logits' type
adds half a step (2^-8 bf16, 2^-11 f16 with 2^-25, 2^-24 f32).
"""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import experts
from mlx_gptq.experts import ExpertMLP, top_k_softmax, top_k_softmax_grad

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


def oracle(logits, k, renorm):
    """(index, weights, softmax) in float64, by a stable order."""
    l = logits.double()
    order = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :k]
    v = l.gather(1, order)
    some = ~(v == -torch.inf)
    m = torch.where(some[:, :1], v[:, :1], 0.0)
    p = torch.exp(l - m)
    total = torch.where(some, p.gather(1, order), 0.0).sum(1, keepdim=True) if renorm else \
        p.sum(1, keepdim=True)
    p = torch.where(some[:, :1], p / total, 0.0)
    w = torch.where(some, p.gather(1, order), 0.0)
    return torch.where(some, order, -1), w, p


def grad_oracle(dw, index, w, p, renorm):
    """(gradient, magnitude of its terms)."""
    k, E = index.shape[1], p.shape[1]
    hit = (index[:, :, None] == torch.arange(E)).double()
    wd = torch.where(w != 0, w * dw.double(), 0.0)
    dot, mag = wd.sum(1, keepdim=True), wd.abs().sum(1, keepdim=True)
    q = (hit * w[:, :, None]).sum(1) if renorm else p
    first = (hit * wd[:, :, None]).sum(1)
    return first - q * dot, first.abs() + q * mag


def spread(logits):
    """At least the largest |l - m|."""
    l = logits.double()
    return 2 * max([0.0] + l[l > -torch.inf].abs().tolist())


def check(logits, k, renorm, seed=0):
    E = logits.shape[1]
    index, weights = top_k_softmax(logits.to(DEV), k, renorm)
    assert index.dtype == torch.int64 and weights.dtype == torch.float32
    want, w, p = oracle(logits, k, renorm)
    assert torch.equal(index.cpu(), want)
    tol = (spread(logits) + E + 8) * 2.0**-24
    assert bool(((weights.cpu().double() - w).abs() <= tol * w + 2.0**-149).all())
    dw = torch.randn(logits.shape[0], k, generator=torch.Generator().manual_seed(seed))
    g = top_k_softmax_grad(dw.to(DEV), logits.to(DEV), index, renorm)
    assert g.dtype == logits.dtype and g.shape == logits.shape
    grad, mag = grad_oracle(dw, want, w, p, renorm)
    bound = (2 * tol + (k + 4) * 2.0**-24) * mag + UNIT[g.dtype] * 1.01 * grad.abs() + STEP[g.dtype] + 2.0**-140
    d = (g.cpu().double() - grad).abs()
    assert bool((d <= bound).all()), (float((d - bound).max()),)


def logits_of(T, E, dtype, seed=0):
    return (torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * 2).to(TYPES[dtype])


SIZES = [(1, 1, 1), (1, 128, 8), (3, 7, 7), (15, 8, 2), (16, 60, 4), (17, 100, 16), (33, 129, 8),
         (5, 256, 1), (40, 257, 6), (64, 511, 8), (9, 512, 16), (7, 1000, 8), (1000, 128, 8),
         (21, 1024, 16), (0, 16, 2)]


@pytest.mark.parametrize("T,E,k", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
def test_choice_weights_and_gradient(T, E, k, dtype, renorm):
    check(logits_of(T, E, dtype, T + E), k, renorm)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E", [24, 33, 200])
def test_equal_logits_go_to_the_lower_index(dtype, E):
    g = torch.Generator().manual_seed(1)
    l = torch.randint(-2, 3, (50, E), generator=g).to(TYPES[dtype])
    l[::2] *= -1.0  # zeros of both signs
    l[7] = 0.0
    check(l, 8, True)
    check(l, 8, False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("E", [40, 45])
@pytest.mark.parametrize("renorm", [True, False])
def test_masked_experts(dtype, E, renorm):
    l = logits_of(30, E, dtype, 3)
    g = torch.Generator().manual_seed(4)
    l[torch.rand(30, E, generator=g) < 0.9] = -torch.inf  # a few left, fewer than k in most rows
    l[4] = -torch.inf
    l[5] = -torch.inf
    l[5, E - 1] = -3.0
    check(l, 6, renorm)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
def test_extreme_logits(dtype, renorm):
    top = torch.finfo(TYPES[dtype]).max
    l = logits_of(6, 32, dtype)
    l[0, 3], l[0, 9] = top, -top
    l[1] = -top
    l[2, 5] = torch.finfo(TYPES[dtype]).tiny / 8  # subnormal
    l[3] = l[3] * 0 + 1e-3
    l[4] = l[4] / 16
    for t in range(6):
        index, w = top_k_softmax(l[t:t + 1].to(DEV), 4, renorm)
        want, ww, _ = oracle(l[t:t + 1], 4, renorm)
        assert torch.equal(index.cpu(), want)
        # (l - m of the largest numbers may pass fp32: its exponential is 0 either way)
        assert bool(((w.cpu().double() - ww).abs() <= 200 * 2.0**-24 * ww + 2.0**-140).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("renorm", [True, False])
def test_rows_that_are_no_numbers_stay_alone(dtype, renorm):
    l = logits_of(20, 48, dtype)
    clean = top_k_softmax(l.to(DEV), 3, renorm)
    l[6, 40], l[11, 2] = torch.nan, torch.inf
    l[12, 3] = -torch.tensor(torch.nan)
    index, w = top_k_softmax(l.to(DEV), 3, renorm)
    assert int(index[6, 0]) == 40 and int(index[11, 0]) == 2 and int(index[12, 0]) == 3
    assert bool(w[[6, 11, 12]].isnan().all())
    keep = [t for t in range(20) if t not in (6, 11, 12)]
    assert torch.equal(index[keep], clean[0][keep]) and torch.equal(w[keep], clean[1][keep])
    g = top_k_softmax_grad(torch.ones(20, 3, device=DEV), l.to(DEV), index, renorm)
    assert bool(g[6, 40].isnan()) and not bool(g[keep].isnan().any())


@pytest.mark.parametrize("renorm", [True, False])
def test_gradient_is_the_functions_derivative(renorm):
    """Central differences of sum(c w) in float64, in a direction that changes no
    choice (the steps are far below the gaps between the logits). The second-order
    error of a difference of step h is h^2 / 6 times a third derivative of at most 6
    per unit direction, and the gradient's own bound is check()'s."""
    l = torch.stack([torch.randperm(40, generator=torch.Generator().manual_seed(t)) for t in range(9)]) * 0.1
    leaf = l.to(DEV).requires_grad_()
    index, w = top_k_softmax(leaf, 5, renorm)
    c = torch.randn(9, 5, generator=torch.Generator().manual_seed(1))
    w.backward(c.to(DEV))
    d = torch.randn(9, 40, generator=torch.Generator().manual_seed(2)).double()
    h = 1e-4
    vals = [float((c.double() * oracle((l.double() + s * h * d), 5, renorm)[1]).sum()) for s in (1, -1)]
    numeric, analytic = (vals[0] - vals[1]) / (2 * h), float((leaf.grad.cpu().double() * d).sum())
    mag = float((leaf.grad.cpu().double().abs() * d.abs()).sum()) + float(c.abs().sum())
    assert abs(numeric - analytic) <= 1e-5 * mag


def test_autograd():
    l = logits_of(12, 30, "bf16")
    leaf = l.to(DEV).requires_grad_()
    index, w = top_k_softmax(leaf, 4, False)
    assert not index.requires_grad and w.requires_grad
    (w * w.detach()).sum().backward()
    assert torch.equal(leaf.grad, top_k_softmax_grad(w.detach(), leaf.detach(), index, False))
    # no second derivative
    leaf = l.to(DEV).requires_grad_()
    _, w = top_k_softmax(leaf, 4)
    (g,) = torch.autograd.grad(w[:, 0].sum(), leaf, create_graph=True)
    with pytest.raises(NotImplementedError, match="top_k_softmax_grad"):
        g.sum().backward()
    # logits written between forward and backward
    leaf = l.to(DEV).requires_grad_()
    x = leaf * 1
    _, w = top_k_softmax(x, 4)
    x.mul_(2)
    with pytest.raises(RuntimeError):
        w.sum().backward()


@pytest.mark.parametrize("E", [64, 72, 65])
def test_strides_and_alignment(E):
    wide = logits_of(20, E + 11, "bf16").to(DEV)
    for start in (0, 3, 8):
        l = wide[:, start:start + E]
        index, w = top_k_softmax(l, 4, False)
        i2, w2 = top_k_softmax(l.contiguous(), 4, False)
        # rows on 16-byte boundaries are added up in another order than others: two sums of
        # the same E positive terms are within 2 E 2^-24 of each other, the gradient's (dot
        # is at most 4 here) within 4 times that before both are rounded to bf16
        assert torch.equal(index, i2) and bool(((w - w2).abs() <= 2 * (E + 8) * 2.0**-24 * w2).all())
        dw = torch.ones(4, 20, device=DEV).t()
        a = top_k_softmax_grad(dw, l, index.to(torch.int32), False).double()
        b = top_k_softmax_grad(dw.contiguous(), l.contiguous(), index, False).double()
        assert bool(((a - b).abs() <= 8 * (E + 8) * 2.0**-24 + 2.0**-7 * b.abs()).all())
    turned = logits_of(E, 20, "f32").to(DEV).t()
    assert torch.equal(top_k_softmax(turned, 3)[0], top_k_softmax(turned.contiguous(), 3)[0])


def test_more_rows_than_a_grid_has_groups():
    """2^20 workgroups of 16 rows go round."""
    T = (1 << 24) + 37
    l = torch.zeros(T, 4, dtype=torch.bfloat16, device=DEV)
    l[:, 2] = 1.0
    l[-1, 3] = 2.0
    l[1 << 24, 1] = 3.0
    index, w = top_k_softmax(l, 1)
    want = torch.full((T, 1), 2, device=DEV)
    want[-1], want[1 << 24] = 3, 1
    assert torch.equal(index, want) and bool((w == 1).all())


def test_captured_and_replayed():
    l = logits_of(50, 64, "f32").to(DEV)
    dw = torch.ones(50, 8, device=DEV)
    step = lambda: (lambda i, w: (i, w, top_k_softmax_grad(dw, l, i)))(*top_k_softmax(l, 8))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in (1, 2, 3):
        l.copy_(logits_of(50, 64, "f32", seed))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_indexes_out_of_range_add_nothing():
    l = logits_of(5, 16, "f32").to(DEV)
    index, _ = top_k_softmax(l, 3)
    bad = index.clone()
    bad[:, 1] = torch.tensor([16, -1, 2**40, -(2**40), 99], device=DEV)
    dw = torch.ones(5, 3, device=DEV)
    dw[:, 1] = torch.nan
    g = top_k_softmax_grad(dw, l, bad)
    i2 = torch.stack((index[:, 0], index[:, 2]), 1)
    assert torch.equal(g, top_k_softmax_grad(dw[:, [0, 2]], l, i2))


def test_the_whole_layer():
    """Router, experts for few rows and the prompt's forward together, with rows whose
    experts are all masked."""
    g = torch.Generator().manual_seed(6)
    E, H, I, T = 12, 96, 64, 20
    up = (torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(torch.bfloat16).to(DEV)
    down = (torch.randn(E, H, I, generator=g) * I**-0.5).to(torch.bfloat16).to(DEV)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    router = torch.randn(E, H, generator=g).to(DEV) * H**-0.5
    logits = x.float() @ router.t()
    logits[3] = -torch.inf
    logits[4, 2:] = -torch.inf
    for mode in ("dense", "mxfp4", "affine"):
        layer = ExpertMLP.from_weights(up, down, mode, group_size=32)
        index, w = experts.top_k_softmax(logits, 4)
        y, f = layer.decode(x, index, w), layer(x, index, w)
        assert not bool(y[3].any()) and not bool(f[3].any())
        assert float((y.double() - f.double()).norm() / f.double().norm()) < 3 * 2.0**-8
    # a training step reaches the router through the experts
    r = router.clone().requires_grad_()
    index, w = experts.top_k_softmax(x.float() @ r.t(), 4)
    ExpertMLP(up, down)(x, index, w).float().square().sum().backward()
    assert bool(torch.isfinite(r.grad).all()) and float(r.grad.norm()) > 0
