"""What the product with affine weights refuses, before any device work."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear

BF, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


def call(x=(4, 64), words=(3, 8), scales=(3, 2), biases=None, bits=4, x_type=BF, word_type=I32,
         types=(BF, BF), **kw):
    biases = scales if biases is None else biases
    return linear.affine_linear(torch.zeros(x, dtype=x_type), torch.zeros(words, dtype=word_type),
                                torch.zeros(scales, dtype=types[0]),
                                torch.zeros(biases, dtype=types[1]), bits, **kw)


@pytest.mark.parametrize("args,error", [
    ({"x_type": F32}, TypeError),
    ({"word_type": torch.uint8}, TypeError),
    ({"types": (BF, F32)}, TypeError),
    ({"types": (torch.int32, torch.int32)}, TypeError),
    ({"bits": 3}, ValueError),
    ({"bits": 16}, ValueError),
    ({"bits": 4.0}, TypeError),
    ({"bits": 8}, AssertionError),
    ({"x": (4, 65)}, AssertionError),
    ({"x": (4, 0), "words": (3, 0), "scales": (3, 0)}, AssertionError),
    ({"x": (2, 4, 64)}, ValueError),
    ({"scales": (3, 4)}, ValueError),   # groups of 16
    ({"scales": (3, 0)}, ValueError),
    ({"scales": (3, 3)}, ValueError),
    ({"x": (4, 256), "words": (3, 32), "scales": (3, 1)}, ValueError),  # of 256
    ({"scales": (2, 2)}, AssertionError),
    ({"biases": (3, 1)}, AssertionError),
    ({"words": (2, 3, 8), "scales": (2, 3, 2)}, ValueError),  # groups without offsets
    ({"offsets": [0, 4]}, ValueError),
])
def test_arguments(args, error):
    with pytest.raises(error):
        call(**args)


def test_entry_point_returns_a_status():
    ok = dict(X=16, dtype=nat.DTYPE_BF16, n_rows=4, ldx=64, row_index=None, n_entries=4, words=16,
              scales=16, biases=16, param_dtype=nat.DTYPE_BF16, bits=4, group_size=64, n_groups=1, N=3,
              K=64, offsets=None, Y=16, stream=None)
    entry = nat.load().mgq_affine_linear
    for change, status in ((dict(dtype=nat.DTYPE_F32), nat.ERR_VALUE), (dict(param_dtype=5), nat.ERR_VALUE),
                           (dict(bits=3), nat.ERR_VALUE), (dict(group_size=16), nat.ERR_VALUE),
                           (dict(K=96), nat.ERR_SHAPE), (dict(K=0), nat.ERR_SHAPE),
                           (dict(ldx=63), nat.ERR_SHAPE),
                           (dict(bits=8, K=(1 << 28) + 64, ldx=1 << 29), nat.ERR_SHAPE),
                           (dict(n_groups=2), nat.ERR_VALUE), (dict(n_entries=5), nat.ERR_SHAPE),
                           (dict(n_rows=0), nat.ERR_SHAPE), (dict(N=1 << 31), nat.ERR_SHAPE),
                           (dict(n_entries=1 << 30, n_rows=1 << 30, N=1 << 29), nat.ERR_SHAPE)):
        assert entry(*{**ok, **change}.values()) == status, change
        assert "affine_linear" in nat.last_error()
    assert entry(*{**ok, "n_entries": 0}.values()) == nat.OK


def test_a_tangent_is_refused():
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.zeros(4, 64, dtype=BF), torch.ones(4, 64, dtype=BF))
        with pytest.raises(NotImplementedError, match="affine_linear"):
            linear.affine_linear(x, torch.zeros(3, 8, dtype=I32), torch.zeros(3, 2, dtype=BF),
                                 torch.zeros(3, 2, dtype=BF), 4)
