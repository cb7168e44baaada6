"""What the router's choice refuses, before any device work."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq.experts import top_k_softmax, top_k_softmax_grad


def z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


I64 = torch.int64


@pytest.mark.parametrize("call,error", [
    (lambda: top_k_softmax(z(4, 8, dtype=torch.float64), 2), TypeError),
    (lambda: top_k_softmax(z(4, 8, dtype=I64), 2), TypeError),
    (lambda: top_k_softmax(z(8), 2), ValueError),
    (lambda: top_k_softmax(z(2, 4, 8), 2), ValueError),
    (lambda: top_k_softmax(z(4, 8), 0), ValueError),
    (lambda: top_k_softmax(z(4, 8), 9), ValueError),
    (lambda: top_k_softmax(z(4, 64), 17), ValueError),
    (lambda: top_k_softmax(z(4, 1025), 2), ValueError),
    (lambda: top_k_softmax(z(4, 0), 1), ValueError),
    (lambda: top_k_softmax_grad(z(4, 2), z(4, 8), z(4, 2)), ValueError),
    (lambda: top_k_softmax_grad(z(4, 2), z(4, 8), z(4, dtype=I64)), ValueError),
    (lambda: top_k_softmax_grad(z(4, 3), z(4, 8), z(4, 2, dtype=I64)), ValueError),
    (lambda: top_k_softmax_grad(z(3, 2), z(4, 8), z(3, 2, dtype=I64)), ValueError),
    (lambda: top_k_softmax_grad(z(4, 2, dtype=I64), z(4, 8), z(4, 2, dtype=I64)), ValueError),
    (lambda: top_k_softmax_grad(z(4, 2), z(4, 8, dtype=I64), z(4, 2, dtype=I64)), TypeError),
    (lambda: top_k_softmax_grad(z(4, 17), z(4, 64), z(4, 17, dtype=I64)), ValueError),
])
def test_arguments(call, error):
    with pytest.raises(error):
        call()


def test_a_tangent_is_refused():
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(z(4, 8), torch.ones(4, 8))
        with pytest.raises(NotImplementedError, match="top_k_softmax"):
            top_k_softmax(x, 2)


def test_entry_points_return_a_status():
    lib = nat.load()
    ok = dict(logits=16, dtype=nat.DTYPE_F32, T=4, E=8, ld=8, k=2, renorm=1, index=16, weights=16, stream=None)
    bad = ((dict(dtype=5), nat.ERR_VALUE), (dict(E=1025, ld=1025), nat.ERR_SHAPE), (dict(E=0), nat.ERR_SHAPE),
           (dict(ld=7), nat.ERR_SHAPE), (dict(k=9), nat.ERR_SHAPE), (dict(k=0), nat.ERR_SHAPE),
           (dict(E=64, ld=64, k=17), nat.ERR_SHAPE), (dict(T=-1), nat.ERR_SHAPE))
    for change, status in bad:
        assert lib.mgq_top_k_softmax(*{**ok, **change}.values()) == status, change
    assert lib.mgq_top_k_softmax(*{**ok, "T": 0}.values()) == nat.OK
    ok = dict(dw=16, logits=16, dtype=nat.DTYPE_F32, T=4, E=8, ld=8, index=16, k=2, renorm=1, out=16,
              stream=None)
    for change, status in bad:
        assert lib.mgq_top_k_softmax_grad(*{**ok, **change}.values()) == status, change
        assert "top_k_softmax_grad" in nat.last_error()
    assert lib.mgq_top_k_softmax_grad(*{**ok, "T": 0}.values()) == nat.OK
