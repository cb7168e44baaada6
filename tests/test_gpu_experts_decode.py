"""ExpertMLP.decode, a routed layer for a few rows, against float64.

The oracle is the loop over rows and their experts with the weights in float64. Each
tensor carries the bound of its error: a sum of n terms in fp32 n 2^-23 sum|terms|
(affine weights: of |x| (|q scale| + |bias|)), the activation's through |silu'| <= 1.1
and |silu(g)| <= |g| with its rounding to the rows' type, half a step 2^-8 for bf16 and
2^-11 (2^-25 below its normal numbers) for f16, fp32's own expf and division 2^-20.
"""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import grid, packing
from mlx_gptq.experts import ExpertMLP
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25}


def quantize(fmt, w, bits, group, params):
    """(the layer's weight on the device, float64 weight, magnitude of its terms)."""
    if fmt == "dense":
        return w.to(DEV), w.double(), w.double().abs()
    if fmt == "affine":
        q, s, b, _ = grid.rtn_quantize(w.to(DEV), bits, group, storage_dtype=params)
        return (packing.pack_q(q, bits), s, b), *ref.affine(q.cpu(), s.cpu(), b.cpu())
    q, s, _, _ = grid.rtn_quantize_mxfp(w.to(DEV), fmt)
    d = ref.decode(q.cpu(), s.cpu(), fmt)
    return (packing.pack_q(q, 4 if fmt == "mxfp4" else 8), s), d, d.abs()


class Layer:
    def __init__(self, fmt, E, H, I, dtype="bf16", bits=4, group=32, params="bf16", seed=0):
        g = torch.Generator().manual_seed(seed)
        dt = TYPES[dtype]
        up = (torch.randn(E, 2 * I, H, generator=g) * 1.5 * H**-0.5).to(dt)
        down = (torch.randn(E, H, I, generator=g) * I**-0.5).to(dt)
        self.dtype, self.E, self.H, self.I, self.gen = dt, E, H, I, g
        wu, self.up, self.up_mag = quantize(fmt, up, bits, group, TYPES[params])
        wd, self.down, self.down_mag = quantize(fmt, down, bits, group, TYPES[params])
        self.mlp = ExpertMLP(wu, wd, fmt)

    def inputs(self, T, k):
        x = torch.randn(T, self.H, generator=self.gen).to(self.dtype)
        index = torch.stack([torch.randperm(self.E, generator=self.gen)[:k] for _ in range(T)]) \
            if T else torch.zeros(0, k, dtype=torch.int64)
        return x, index, torch.softmax(torch.randn(T, k, generator=self.gen), dim=1)

    def oracle(self, x, index, weights):
        out = torch.zeros(x.shape[0], self.H, dtype=torch.float64)
        err = torch.zeros_like(out)
        unit, step = UNIT[self.dtype], STEP[self.dtype]
        xd, I = x.double(), self.I
        for t in range(x.shape[0]):
            for j in range(index.shape[1]):
                e = int(index[t, j])
                if not 0 <= e < self.E:
                    continue
                h = self.up[e] @ xd[t]
                eh = (self.H + 48) * 2.0**-23 * (self.up_mag[e] @ xd[t].abs())
                g, u, eg, eu = h[:I], h[I:], eh[:I], eh[I:]
                a = torch.nn.functional.silu(g) * u
                ea = 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0**-20 * a.abs()
                ea = ea + unit * 1.01 * (a.abs() + ea) + step
                y = self.down[e] @ a
                ey = self.down_mag[e] @ ea + (I + 48) * 2.0**-23 * (self.down_mag[e] @ (a.abs() + ea))
                w = float(weights[t, j])
                out[t] += w * y
                err[t] += abs(w) * (ey * 1.01 + 2.0**-20 * y.abs())
        return out, err + unit * 1.01 * (out.abs() + err) + step

    def check(self, x, index, weights, **kw):
        y = self.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV), **kw)
        assert y.dtype == self.dtype and y.shape == x.shape
        want, bound = self.oracle(x, index, weights)
        d = (y.cpu().double() - want).abs()
        assert bool((d <= bound).all()), (float((d - bound).max()), torch.nonzero(~(d <= bound))[:3])
        return y


FORMS = [("dense", "bf16", {}), ("dense", "f16", {}), ("mxfp4", "bf16", {}), ("mxfp8", "bf16", {})] + [
    ("affine", dt, dict(bits=bits, group=group, params=params)) for bits in (2, 4, 8)
    for dt, params, group in (("bf16", "bf16", 64), ("f16", "f16", 32), ("bf16", "f32", 32),
                              ("f16", "f32", 64))]


@pytest.mark.parametrize("fmt,dtype,kw", FORMS)
@pytest.mark.parametrize("T", [1, 3, 20])
def test_formats(fmt, dtype, kw, T):
    layer = Layer(fmt, 6, 192, 64, dtype, **kw)
    layer.check(*layer.inputs(T, 2))


# E, H, I, T, k: one expert, more entries than experts and fewer, more than 16 rows of
# an expert, steps that end inside the contraction, rows and columns off every tile
SHAPES = [(1, 32, 32, 1, 1), (1, 32, 32, 64, 1), (8, 64, 32, 1, 8), (3, 96, 160, 40, 3),
          (300, 64, 64, 7, 4), (700, 32, 32, 64, 16), (16, 128, 96, 64, 8), (16, 544, 288, 5, 16),
          (9, 32, 1056, 2, 1), (5, 1056, 32, 1, 3), (40, 160, 64, 4, 8), (4, 2080, 96, 17, 2)]


@pytest.mark.parametrize("E,H,I,T,k", SHAPES)
@pytest.mark.parametrize("fmt", ["dense", "mxfp4", "affine"])
def test_sizes(E, H, I, T, k, fmt):
    layer = Layer(fmt, E, H, I, seed=E + T)
    layer.check(*layer.inputs(T, k))


@pytest.mark.parametrize("H,I", [(1, 1), (7, 5), (33, 129), (130, 17), (257, 255)])
@pytest.mark.parametrize("T", [1, 2, 18])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_odd_dense_sizes(H, I, T, dtype):
    layer = Layer("dense", 4, H, I, dtype)
    layer.check(*layer.inputs(T, 2))


@pytest.mark.parametrize("T", [1, 4, 30])
def test_experts_outside_the_layer_add_nothing(T):
    layer = Layer("affine", 5, 64, 64)
    x, index, weights = layer.inputs(T, 4)
    index[:, 1] = 5
    index[::2, 2] = -1
    weights[:, 1] = torch.nan  # (whatever their weight is)
    index[T // 2] = torch.tensor([-7, 2**40, 5, 99])
    y = layer.check(x, index, torch.where(index >= 0, weights, torch.nan))
    assert not bool(y[T // 2].any())
    index[:] = -1
    assert not bool(layer.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV)).any())


@pytest.mark.parametrize("T", [1, 3, 40])
def test_a_row_may_name_an_expert_twice(T):
    layer = Layer("mxfp4", 4, 64, 96)
    x, index, weights = layer.inputs(T, 4)
    index[:, 3] = index[:, 0]
    index[0] = 2
    layer.check(x, index, weights)


def test_routing_that_is_lopsided():
    """One expert has every row, another a single one."""
    layer = Layer("affine", 40, 96, 64)
    x, index, weights = layer.inputs(64, 2)
    index[:, 0], index[:, 1] = 7, -1
    index[33, 1] = 39
    layer.check(x, index, weights)


def test_rows_and_weights_in_place():
    """A row pitch of its own, weights inside a larger tensor, 32-bit ids, weights in
    bf16 and in an order that is not contiguous."""
    layer = Layer("dense", 4, 40, 24)
    x, index, weights = layer.inputs(6, 2)
    want = layer.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV))
    wide = torch.zeros(6, 47, dtype=x.dtype, device=DEV)
    wide[:, 3:43] = x.to(DEV)
    up = torch.zeros(4, 50, 61, dtype=x.dtype, device=DEV)
    up[:, 1:49, 5:45] = layer.mlp.gate_up
    mlp = ExpertMLP(up[:, 1:49, 5:45], layer.mlp.down)
    turned = torch.empty(2, 6, device=DEV).t()
    turned.copy_(weights)
    for i in (index, index.to(torch.int32), index.to(torch.uint8)):
        assert torch.equal(mlp.decode(wide[:, 3:43], i.to(DEV), turned), want)
    half = weights.to(torch.bfloat16)
    layer.check(x, index, half)
    # host rows come back to the host
    y = layer.mlp.decode(x, index, weights)
    assert y.device.type == "cpu" and torch.equal(y, want.cpu())


@pytest.mark.parametrize("T", [1, 24])
def test_a_row_that_is_no_number_stays_alone(T):
    layer = Layer("mxfp8", 4, 64, 64)
    x, index, weights = layer.inputs(T + 1, 2)
    index[:, 0] = 1
    clean = layer.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV))
    x[T // 2, 5] = torch.inf
    x[T // 2, 6] = torch.nan
    y = layer.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV))
    keep = [t for t in range(T + 1) if t != T // 2]
    assert bool(y[T // 2].isnan().all()) and torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("fmt", ["mxfp4", "affine"])
def test_forward_and_decode_agree(fmt):
    layer = Layer(fmt, 8, 96, 64)
    x, index, weights = (t.to(DEV) for t in layer.inputs(12, 3))
    y, f = layer.mlp.decode(x, index, weights), layer.mlp(x, index, weights)
    # forward rounds the gate and up products, each expert's result and the sum: four
    # steps of 2^-8 where decode has two, on terms up to the largest result
    assert float((y.double() - f.double()).abs().max()) <= 6 * 2.0**-8 * float(f.double().abs().max()) * 3


@pytest.mark.parametrize("T", [1, 3, 24])
def test_captured_and_replayed(T):
    """New rows and another routing in the same buffers; two graphs with workspaces of
    their own, replayed in turn."""
    layer = Layer("affine", 12, 64, 64)
    state = [tuple(t.to(DEV) for t in layer.inputs(T, 4)) for _ in range(2)]
    graphs = []
    for s in state:
        layer.mlp.decode(*s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = layer.mlp.decode(*s)
        graphs.append((graph, y))
    for _ in range(3):
        for s in state:
            for t, new in zip(s, layer.inputs(T, 4)):
                t.copy_(new)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for s, (_, y) in zip(state, graphs):
            assert torch.equal(y, layer.mlp.decode(*s))


def test_two_streams_at_once():
    layer = Layer("dense", 6, 128, 64)
    inputs = [tuple(t.to(DEV) for t in layer.inputs(9, 3)) for _ in range(4)]
    want = [layer.mlp.decode(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = []
    for s, i in zip(streams, inputs):
        with torch.cuda.stream(s):
            got.append([layer.mlp.decode(*i) for _ in range(5)])
    torch.cuda.synchronize()
    for w, ys in zip(want, got):
        assert all(torch.equal(w, y) for y in ys)


def test_affine_layer():
    """from_weights and from_codes in the affine grid, forward and decode."""
    g = torch.Generator().manual_seed(2)
    up = (torch.randn(5, 128, 64, generator=g) * 0.1).to(torch.bfloat16).to(DEV)
    down = (torch.randn(5, 64, 64, generator=g) * 0.1).to(torch.bfloat16).to(DEV)
    codes = [grid.rtn_quantize(w, 8, 32)[:3] for w in (up, down)]
    one = ExpertMLP.from_weights(up, down, "affine", bits=8, group_size=32)
    two = ExpertMLP.from_codes(*codes, "affine", bits=8)
    dense = ExpertMLP(up, down)
    x = torch.randn(10, 64, generator=g).to(torch.bfloat16).to(DEV)
    index = torch.randint(0, 5, (10, 2), generator=g).to(DEV)
    weights = torch.rand(10, 2, generator=g).to(DEV)
    assert torch.equal(one(x, index, weights), two(x, index, weights))
    assert torch.equal(one.decode(x, index, weights), two.decode(x, index, weights))
    y = dense(x, index, weights).double()
    for f in (one(x, index, weights), one.decode(x, index, weights)):
        assert float((f.double() - y).norm() / y.norm()) < 0.03  # 8-bit codes


def test_a_gradient_raises():
    layer = Layer("dense", 4, 32, 32)
    x, index, weights = (t.to(DEV) for t in layer.inputs(3, 2))
    y = layer.mlp.decode(x.requires_grad_(), index, weights)
    with pytest.raises(NotImplementedError, match="decode"):
        y.sum().backward()


def test_a_gradient_of_the_scales_raises():
    layer = Layer("affine", 4, 32, 32)
    x, index, weights = (t.to(DEV) for t in layer.inputs(3, 2))
    layer.mlp.gate_up[1].requires_grad_()
    y = layer.mlp.decode(x, index, weights)
    with pytest.raises(NotImplementedError, match="decode"):
        y.sum().backward()


@pytest.mark.parametrize("T,k", [(2, 16), (20, 3), (64, 16)])
def test_more_experts_than_a_table_of_them_holds(T, k):
    layer = Layer("affine", 1500, 32, 32, group=32)
    x, index, weights = layer.inputs(T, k)
    index[:, 0] = 1499
    index[0] = torch.arange(k) % 2 + 1030  # (a row with two experts, many times)
    layer.check(x, index, weights)


@pytest.mark.parametrize("T", [1, 3, 20])
def test_far_weights(T):
    """An expert whose weights start behind 2^32 bytes, against float64 on the device."""
    E, H, I = 5, 16384, 16384
    up = torch.empty(E, 2 * I, H, dtype=torch.bfloat16, device=DEV).normal_(0, H**-0.5)
    down = torch.empty(E, H, I, dtype=torch.bfloat16, device=DEV).normal_(0, I**-0.5)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, H, generator=g).to(torch.bfloat16).to(DEV)
    weights = torch.rand(T, 1, generator=g).to(DEV) + 0.5
    y = ExpertMLP(up, down).decode(x, torch.full((T, 1), E - 1, device=DEV), weights)
    w, xd = up[-1].double(), x.double()
    h, eh = xd @ w.T, (H + 48) * 2.0**-23 * (xd.abs() @ w.abs().T)
    del w
    gate, u, eg, eu = h[:, :I], h[:, I:], eh[:, :I], eh[:, I:]
    a = torch.nn.functional.silu(gate) * u
    ea = 1.1 * eg * (u.abs() + eu) + (gate.abs() + eg) * eu + 2.0**-20 * a.abs()
    ea = ea + 2.0**-8 * 1.01 * (a.abs() + ea)
    w = down[-1].double()
    want = a @ w.T
    err = ea @ w.abs().T + (I + 48) * 2.0**-23 * ((a.abs() + ea) @ w.abs().T)
    want, err = weights.double() * want, weights.double() * (err * 1.01 + 2.0**-20 * want.abs())
    bound = err + 2.0**-8 * 1.01 * (want.abs() + err)
    d = (y.double() - want).abs()
    assert bool((d <= bound).all()), float((d - bound).max())
