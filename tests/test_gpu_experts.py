"""The experts' MLP on the grouped products, in every weight format.

The oracle is the eager loop over experts in float64. Each tensor the product
forms carries the bound of its error: a product's sums as in
tests/test_gpu_linear.py (n 2^-23 sum|terms|, half an ulp 2^-8 of bf16), the
activation's through |silu'| <= 1.1 and |silu(g)| <= |g|, and for int8 half a step
of the row's scale for every quantized value.
"""

from __future__ import annotations

import importlib.util
import os

import pytest
import torch

from mlx_gptq import grid, linear
from mlx_gptq.experts import ExpertMLP, route

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
ULP = 2.0**-8


def layer(E, H, I, T, k, seed=0, drop=False):
    g = torch.Generator().manual_seed(seed)
    gate_up = (torch.randn(E, 2 * I, H, generator=g) * H**-0.5).to(torch.bfloat16)
    down = (torch.randn(E, H, I, generator=g) * I**-0.5).to(torch.bfloat16)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16)
    index = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T else \
        torch.zeros(0, k, dtype=torch.int64)
    if drop:
        index[::3, 0] = E
        index[1::3, -1] = -1
    weights = torch.softmax(torch.randn(T, k, generator=g), dim=1)
    return gate_up, down, x, index, weights


def oracle(gate_up, down, x, index, weights, step=0.0):
    """(out, bound) with weights in float64; step 1/254 for int8 rows: half a
    quantization step relative to the row's largest value."""
    E, I2, H = gate_up.shape
    I = I2 // 2
    out = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64)
    err = torch.zeros_like(out)
    xd = x.double()
    ex = xd.abs().amax(1, keepdim=True) * step * 1.01
    for t in range(x.shape[0]):
        for j in range(index.shape[1]):
            e = int(index[t, j])
            if not 0 <= e < E:
                continue
            h = gate_up[e] @ xd[t]
            eh = (H + 8) * 2.0**-23 * (gate_up[e].abs() @ xd[t].abs()) + \
                (gate_up[e].abs() @ ex[t].expand(H)) + ULP * h.abs() * 1.01
            g, u, eg, eu = h[:I], h[I:], eh[:I], eh[I:]
            a = torch.nn.functional.silu(g) * u
            ea = 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu
            ea = ea + ULP * 1.01 * (a.abs() + ea)
            ea = ea + (a.abs() + ea).max() * step * 1.01
            y = down[e] @ a
            ey = down[e].abs() @ ea + (I + 8) * 2.0**-23 * (down[e].abs() @ (a.abs() + ea))
            ey = ey + ULP * 1.01 * (y.abs() + ey)
            w = float(weights[t, j])
            out[t] += w * y
            err[t] += abs(w) * ey * (1 + 2.0**-20) + 2.0**-20 * abs(w) * y.abs()
    return out, err + ULP * 1.01 * (out.abs() + err)


def check(y, want, bound):
    d = (y.cpu().double() - want).abs()
    assert bool((d <= bound).all()), float((d - bound).max())


SHAPES = [(8, 64, 32, 1, 2, False), (8, 64, 32, 1, 8, False), (5, 96, 64, 33, 3, True),
          (16, 128, 96, 70, 4, False), (4, 160, 32, 50, 1, True)]


@pytest.mark.parametrize("E,H,I,T,k,drop", SHAPES)
@pytest.mark.parametrize("mode", ExpertMLP.MODES)
def test_forward(E, H, I, T, k, drop, mode):
    gate_up, down, x, index, weights = layer(E, H, I, T, k, seed=E + T, drop=drop)
    mlp = ExpertMLP.from_weights(gate_up.to(DEV), down.to(DEV), mode)
    y = mlp(x.to(DEV), index.to(DEV), weights.to(DEV))
    assert y.dtype == torch.bfloat16 and tuple(y.shape) == (T, H)
    if mode == "dense":
        ws = (gate_up.double(), down.double())
    elif mode == "int8":
        ws = tuple(q.cpu().double() * s.cpu().double().unsqueeze(-1)
                   for q, s in (linear.quantize_rows_int8(w.to(DEV)) for w in (gate_up, down)))
    else:
        ws = tuple(grid.rtn_quantize_mxfp(w.to(DEV), mode)[3].cpu().double() for w in (gate_up, down))
    check(y, *oracle(*ws, x, index, weights, step=1 / 254 if mode == "int8" else 0.0))


def test_no_rows():
    gate_up, down, x, index, weights = layer(4, 64, 32, 0, 2)
    y = ExpertMLP(gate_up.to(DEV), down.to(DEV))(x.to(DEV), index.to(DEV), weights.to(DEV))
    assert tuple(y.shape) == (0, 64)


def test_route():
    index = torch.tensor([[2, 0], [9, 2], [0, -1], [2, 1]], device=DEV)
    r = route(index, 3)
    assert r.offsets.tolist() == [0, 2, 3, 6]
    assert r.row_index.tolist() == [0, 2, 3, 0, 1, 3, 1, 2]
    assert r.entry.tolist() == [3, 0, 6, 4, 1, 7, 5, 2]
    with pytest.raises(ValueError):
        route(index.float(), 3)


def test_gradients_reach_the_weights_and_the_rows():
    """The MLP's gradients against float32 autograd of the eager loop on the CPU:
    bf16 rounds the activations and their gradients at five places on the way, each
    by at most 2^-8 relative, so that the norm of the difference is below 5 2^-8."""
    E, H, I, T, k = 6, 96, 64, 40, 3
    gate_up, down, x, index, weights = layer(E, H, I, T, k, seed=5)
    g = torch.Generator().manual_seed(6)
    c = torch.randn(T, H, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (gate_up, down, x)]
    y = ExpertMLP(leaves[0], leaves[1])(leaves[2], index.to(DEV), weights.to(DEV))
    (y.float() * c.to(DEV)).sum().backward()
    ref = [t.float().requires_grad_() for t in (gate_up, down, x)]
    out = torch.zeros(T, H)
    for e in range(E):
        t, j = torch.nonzero(index == e, as_tuple=True)
        h = ref[2][t] @ ref[0][e].T
        a = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
        out = out.index_add(0, t, (a @ ref[1][e].T) * weights[t, j, None])
    (out * c).sum().backward()
    for a, b in zip(leaves, ref):
        rel = float((a.grad.cpu().float() - b.grad).norm() / b.grad.norm())
        assert rel < 5 * ULP, rel


def test_refusals():
    w = torch.zeros(2, 4, 32, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError):
        ExpertMLP(w, w, "int4")
    with pytest.raises(ValueError):
        ExpertMLP(w[:, :3], w)
    with pytest.raises(ValueError):
        ExpertMLP.from_codes((w, w), (w, w), "affine")


def test_example():
    path = os.path.join(os.path.dirname(__file__), "..", "examples", "experts_forward.py")
    spec = importlib.util.spec_from_file_location("experts_forward", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    e = mod.main(["--experts", "8", "--hidden", "256", "--inter", "128", "--tokens", "200",
                  "--top-k", "2"])
    # three weights multiply into an output (gate, up and down, the first through a
    # slope of at most 1.1), so its relative error stays below 1.1 + 1 + 1 times
    # theirs; int8 steps are 1/254 of a row's largest value
    for mode in ("mxfp4", "mxfp8"):
        assert 0 < e[f"{mode} nearest"] < 3.1 * e[f"{mode} weights"]
    assert e["mxfp4 solved"] < 3.1 * e["mxfp4 weights"] and e["int8 nearest"] < 0.1
    assert e["loss after"] < e["loss before"]
