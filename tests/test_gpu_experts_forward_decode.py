"""ExpertMLP.forward and ExpertMLP.decode against the same float64 layer.

decode's bound is test_gpu_experts_decode.py's. forward also rounds the gate and up products
and each expert's result to the rows' type: half a step of each, 2^-8 relative in bf16 and
2^-11 (2^-25 below its normal numbers) in f16, carried on as that test carries the sums'
errors. The rows are few enough for products that do not round the weights.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_experts_decode import DEV, STEP, UNIT, Layer

pytestmark = pytest.mark.gpu


def forward_oracle(layer, x, index, weights):
    out = torch.zeros(x.shape[0], layer.H, dtype=torch.float64)
    err = torch.zeros_like(out)
    half = lambda v, e: 1.01 * UNIT[layer.dtype] * (v.abs() + e) + STEP[layer.dtype]
    xd, I = x.double(), layer.I
    for t in range(x.shape[0]):
        for j in range(index.shape[1]):
            e = int(index[t, j])
            h = layer.up[e] @ xd[t]
            eh = (layer.H + 48) * 2.0**-23 * (layer.up_mag[e] @ xd[t].abs())
            eh = eh + half(h, eh)
            g, u, eg, eu = h[:I], h[I:], eh[:I], eh[I:]
            a = torch.nn.functional.silu(g) * u
            ea = 1.1 * eg * (u.abs() + eu) + (g.abs() + eg) * eu + 2.0**-20 * a.abs()
            ea = ea + half(a, ea)
            y = layer.down[e] @ a
            ey = layer.down_mag[e] @ ea + (I + 48) * 2.0**-23 * (layer.down_mag[e] @ (a.abs() + ea))
            ey = ey + half(y, ey)
            w = float(weights[t, j])
            out[t] += w * y
            err[t] += abs(w) * (ey * 1.01 + 2.0**-20 * y.abs())
    return out, err + half(out, err)


@pytest.mark.parametrize("fmt,dtype,kw", [("dense", "bf16", {}), ("dense", "f16", {}), ("mxfp4", "bf16", {}),
                                          ("mxfp8", "bf16", {}), ("affine", "bf16", {}),
                                          ("affine", "f16", dict(bits=8, params="f32")),
                                          ("affine", "bf16", dict(bits=2, group=64, params="f16"))])
@pytest.mark.parametrize("T", [1, 5, 12])
def test_both_ways_through_a_layer(fmt, dtype, kw, T):
    layer = Layer(fmt, 8, 192, 64, dtype, **kw)
    x, index, weights = layer.inputs(T, 3)
    layer.check(x, index, weights)
    y = layer.mlp(x.to(DEV), index.to(DEV), weights.to(DEV))
    want, bound = forward_oracle(layer, x, index, weights)
    d = (y.cpu().double() - want).abs()
    assert bool((d <= bound).all()), float((d - bound).max())
