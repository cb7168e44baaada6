"""What ExpertMLP.decode refuses, before any device work."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear
from mlx_gptq.experts import ExpertMLP

BF, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32


@pytest.fixture(autouse=True)
def host(monkeypatch):
    # (what passes the checks would go on to a launch)
    monkeypatch.setattr(linear, "_device", lambda *tensors: torch.device("cpu"))

    def launch(*args):
        raise RuntimeError("launched")

    monkeypatch.setattr(nat, "launch", launch)


def dense(E=4, H=64, I=32, dtype=BF):
    return ExpertMLP(torch.zeros(E, 2 * I, H, dtype=dtype), torch.zeros(E, H, I, dtype=dtype))


def words(mode, E=4, H=64, I=32, bits=4, params=BF, down_params=None):
    def w(n, k, dt):
        packed = torch.zeros(E, n, k * bits // 32, dtype=I32)
        if mode == "affine":
            return packed, torch.zeros(E, n, k // 32, dtype=dt), torch.zeros(E, n, k // 32, dtype=dt)
        return packed, torch.zeros(E, n, k // 32, dtype=torch.uint8)

    return ExpertMLP(w(2 * I, H, params), w(H, I, down_params or params), mode)


def call(layer, x=(3, 64), index=(3, 2), weights=None, dtype=BF, index_type=torch.int64,
         weights_type=F32):
    return layer.decode(torch.zeros(x, dtype=dtype), torch.zeros(index, dtype=index_type),
                        torch.zeros(index if weights is None else weights, dtype=weights_type))


def test_what_is_taken_reaches_the_launch():
    for layer in (dense(), words("mxfp4"), words("mxfp8", bits=8), words("affine"),
                  words("affine", bits=2, params=F32), words("affine", down_params=F32)):
        with pytest.raises(RuntimeError, match="launched"):
            call(layer)
    with pytest.raises(RuntimeError, match="launched"):
        call(dense(dtype=F16), dtype=F16, index=(3, 16), index_type=torch.uint8, weights_type=F16)
    assert call(dense(), x=(0, 64), index=(0, 2)).shape == (0, 64)


@pytest.mark.parametrize("layer,args,error", [
    (dense, dict(x=(65, 64), index=(65, 2)), ValueError),
    (dense, dict(index=(3, 17)), ValueError),
    (dense, dict(index=(3, 0)), ValueError),
    (dense, dict(index=(2, 2)), ValueError),
    (dense, dict(index=(3,)), ValueError),
    (dense, dict(index_type=F32), ValueError),
    (dense, dict(index_type=torch.bool), ValueError),
    (dense, dict(weights=(3, 3)), ValueError),
    (dense, dict(weights_type=torch.int64), ValueError),
    (dense, dict(x=(3, 2, 64)), ValueError),
    (dense, dict(dtype=F32), TypeError),
    (dense, dict(dtype=F16), TypeError),
    (dense, dict(x=(3, 63)), AssertionError),
    (lambda: words("mxfp4"), dict(dtype=F16), TypeError),
    (lambda: words("mxfp4"), dict(x=(3, 32)), AssertionError),
    (lambda: words("affine"), dict(x=(3, 32)), ValueError),
    (lambda: ExpertMLP((torch.zeros(4, 64, 64, dtype=torch.int8), torch.zeros(4, 64)),
                       (torch.zeros(4, 64, 32, dtype=torch.int8), torch.zeros(4, 64)), "int8"), {},
     ValueError),
    (lambda: ExpertMLP(torch.zeros(4, 64, 64, dtype=BF), torch.zeros(4, 64, 31, dtype=BF)), {},
     AssertionError),
    (lambda: ExpertMLP(torch.zeros(4, 64, 64, dtype=BF), torch.zeros(3, 64, 32, dtype=BF)), {},
     AssertionError),
])
def test_arguments(layer, args, error):
    with pytest.raises(error):
        call(layer(), **args)


def test_formats_of_a_layer():
    q = torch.zeros(2, 4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError):
        ExpertMLP.from_codes((q, q), (q, q), "int8")
    with pytest.raises(ValueError):
        ExpertMLP.from_codes((q, q), (q, q), "mxfp4", bits=8)


OK = dict(X=16, dtype=nat.DTYPE_BF16, T=3, ldx=64, index=16, index_bits=64, weights=16, k=2, E=4, H=64,
          I=32, up=None, down=None, out=16, ws=16, ws_bytes=1 << 20, stream=None)
UP = dict(data=16, scales=16, biases=16, ld=0, expert=0, group=32, format=nat.WEIGHT_AFFINE4,
          param_dtype=nat.DTYPE_BF16)
DOWN = dict(data=16, scales=None, biases=None, ld=32, expert=2048, group=0, format=nat.WEIGHT_DENSE,
            param_dtype=0)


def entry(up=None, down=None, **change):
    u, d = nat.Weight(**{**UP, **(up or {})}), nat.Weight(**{**DOWN, **(down or {})})
    args = {**OK, "up": ctypes.addressof(u), "down": ctypes.addressof(d), **change}
    return nat.load().mgq_experts_decode(*args.values())


@pytest.mark.parametrize("change,status", [
    (dict(dtype=nat.DTYPE_F32), nat.ERR_VALUE), (dict(index_bits=16), nat.ERR_VALUE),
    (dict(T=65), nat.ERR_SHAPE), (dict(k=17), nat.ERR_SHAPE), (dict(k=0), nat.ERR_SHAPE),
    (dict(E=0), nat.ERR_SHAPE), (dict(I=0), nat.ERR_SHAPE), (dict(ldx=63), nat.ERR_SHAPE),
    (dict(up=dict(format=6)), nat.ERR_VALUE), (dict(up=dict(group=16)), nat.ERR_VALUE),
    (dict(up=dict(param_dtype=7)), nat.ERR_VALUE),
    (dict(H=96, ldx=96, up=dict(group=64)), nat.ERR_SHAPE),
    (dict(down=dict(ld=31)), nat.ERR_SHAPE), (dict(down=dict(ld=1 << 29)), nat.ERR_SHAPE),
    (dict(down=dict(ld=(1 << 27) + 1)), nat.ERR_SHAPE),
    (dict(H=(1 << 28) + 64, ldx=1 << 29, up=dict(format=nat.WEIGHT_AFFINE8), ws_bytes=1 << 40),
     nat.ERR_SHAPE),
    (dict(down=dict(format=nat.WEIGHT_MXFP4), I=48), nat.ERR_SHAPE),
    (dict(dtype=nat.DTYPE_F16, down=dict(format=nat.WEIGHT_MXFP8)), nat.ERR_VALUE),
    (dict(ws_bytes=100), nat.ERR_WORKSPACE)])
def test_entry_point_returns_a_status(change, status):
    assert entry(**change) == status
    assert "experts_decode" in nat.last_error()
    assert entry(T=0) == nat.OK


def test_the_weights_are_described_anew_when_they_change():
    """A tensor put in another's place, moved or reshaped is seen; one that is written is
    the same."""
    layer = dense()
    cpu = torch.device("cpu")
    first = layer._decode_weights(64, BF, cpu)
    layer.gate_up.fill_(1.0)
    assert layer._decode_weights(64, BF, cpu) is first
    layer.gate_up = layer.gate_up.clone()
    second = layer._decode_weights(64, BF, cpu)
    assert second is not first and second.up.data == layer.gate_up.data_ptr()
    layer.down.data = layer.down.data.clone()
    third = layer._decode_weights(64, BF, cpu)
    assert third is not second and third.down.data == layer.down.data_ptr()
    with pytest.raises(AssertionError):
        layer._decode_weights(32, BF, cpu)
    # copies are made again for every call
    layer.down = torch.zeros(4, 32, 64, dtype=BF).transpose(1, 2)
    a = layer._decode_weights(64, BF, cpu)
    assert layer._decode_weights(64, BF, cpu) is not a
