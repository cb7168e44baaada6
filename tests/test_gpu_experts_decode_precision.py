"""The activation between ExpertMLP.decode's launches has more bits than the rows' type, for
up to eight rows.

The experts' inner rows come in pairs that differ in a few elements by a step of the type,
and the down weights of a pair are opposite: a result is a sum of small differences of
activations, which 16 bits of each would not leave anything of. Bounds as in
test_gpu_experts_decode.py, but for the activation: it is rounded to the rows' type, and
what that lost is rounded again, half a step of half a step: 2^-8 2^-8 in bf16, 2^-11 2^-11
and half of the subnormal step, 2^-25, in f16.
"""

from __future__ import annotations

import pytest
import torch

import tests.test_gpu_experts_decode as decode
from tests.test_gpu_experts_decode import Layer, quantize

pytestmark = pytest.mark.gpu


class Paired(Layer):
    def __init__(self, fmt, E, H, I, dtype="bf16", bits=4, group=32, params="f32", seed=0):
        super().__init__(fmt, E, H, I, dtype, bits, group, params, seed)
        g, dt = self.gen, self.dtype
        up = (torch.randn(E, 2, I // 2, 2, H, generator=g) * 1.5 * H**-0.5).to(dt)
        nudge = 1 + 4 * decode.UNIT[dt] * (torch.rand(E, 2, I // 2, H, generator=g) < 0.02)
        up[..., 1, :] = (up[..., 0, :].float() * nudge).to(dt)
        down = (torch.randn(E, H, I // 2, 2, generator=g) * I**-0.5).to(dt)
        down[..., 1] = -down[..., 0]
        grid = bits, group, decode.TYPES[params]
        self.mlp.gate_up, self.up, self.up_mag = quantize(fmt, up.view(E, 2 * I, H), *grid)
        self.mlp.down, self.down, self.down_mag = quantize(fmt, down.view(E, H, I), *grid)

    def oracle(self, x, index, weights):
        out = torch.zeros(x.shape[0], self.H, dtype=torch.float64)
        err = torch.zeros_like(out)
        unit, step = decode.UNIT[self.dtype], decode.STEP[self.dtype]
        xd, I = x.double(), self.I
        for t in range(x.shape[0]):
            for j in range(index.shape[1]):
                e = int(index[t, j])
                h = self.up[e] @ xd[t]
                eh = (self.H + 48) * 2.0**-23 * (self.up_mag[e] @ xd[t].abs())
                g, u, eg, eu = h[:I], h[I:], eh[:I], eh[I:]
                a = torch.nn.functional.silu(g) * u
                ea = 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0**-20 * a.abs()
                ea = ea + unit * unit * 1.01 * (a.abs() + ea) + step
                # (two terms a weight: the parts of the activation)
                y = self.down[e] @ a
                ey = self.down_mag[e] @ ea + (2 * I + 48) * 2.0**-23 * (self.down_mag[e] @ (a.abs() + ea))
                w = float(weights[t, j])
                out[t] += w * y
                err[t] += abs(w) * (ey * 1.01 + 2.0**-20 * y.abs())
        return out, err + unit * 1.01 * (out.abs() + err) + step


@pytest.mark.parametrize("fmt,dtype,kw", [
    ("dense", "bf16", {}), ("dense", "f16", {}), ("mxfp4", "bf16", {}), ("mxfp8", "bf16", {}),
    ("affine", "bf16", dict(bits=8)), ("affine", "f16", dict(bits=8, group=64)),
    ("affine", "bf16", dict(bits=4, group=64)), ("affine", "bf16", dict(bits=2, group=64))])
@pytest.mark.parametrize("T", [1, 3, 6, 8])
@pytest.mark.parametrize("I", [64, 192])
def test_differences_of_activations(fmt, dtype, kw, T, I):
    layer = Paired(fmt, 6, 128, I, dtype, **kw)
    x, index, weights = layer.inputs(T, 2)
    layer.check(x, index, weights)


@pytest.mark.parametrize("T", [1, 3, 7, 8, 9])
@pytest.mark.parametrize("I", [1, 33, 255])
def test_odd_sizes(T, I):
    """Both parts of rows that end anywhere."""
    layer = Layer("dense", 4, 40, I)
    x, index, weights = layer.inputs(T, 2)
    index[:, 0] = 2  # (one expert has all rows)
    layer.check(x, index, weights)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T", [1, 3, 8, 20])
def test_activations_that_are_no_numbers(dtype, T):
    """An activation past the type's largest number is an infinity, not the difference of two."""
    layer = Layer("dense", 3, 32, 32, dtype)
    x, index, weights = layer.inputs(T, 1)
    top = torch.finfo(layer.dtype).max
    x[:], index[:] = 1.0, 1
    weights[:] = 1.0
    layer.mlp.gate_up[1] = top / 64
    layer.mlp.gate_up[1, 32:] = 8.0
    layer.mlp.down[1] = 1.0
    y = layer.mlp.decode(x.to(decode.DEV), index.to(decode.DEV), weights.to(decode.DEV))
    assert bool((y == torch.inf).all())
