"""mgq_experts_decode checks the weights' descriptions, which it reads on the host."""

from __future__ import annotations

import ctypes

import pytest

from mlx_gptq import _native as nat
from tests.test_experts_decode_refusals import OK, entry


@pytest.mark.parametrize("change", [
    dict(up=dict(data=None)), dict(up=dict(scales=None)), dict(up=dict(biases=None)),
    dict(down=dict(data=None)), dict(up=dict(format=nat.WEIGHT_MXFP4, scales=None)),
    dict(down=dict(format=nat.WEIGHT_AFFINE2, scales=16, group=32)),
])
def test_a_part_that_is_missing(change):
    assert entry(**change) == nat.ERR_VALUE
    assert "experts_decode" in nat.last_error()


def test_a_workspace_that_is_missing():
    assert entry(ws=None) == nat.ERR_WORKSPACE
    assert "experts_decode" in nat.last_error()


@pytest.mark.parametrize("missing", ["up", "down"])
def test_a_description_that_is_missing(missing):
    w = nat.Weight(data=16, scales=16, biases=16, ld=64, expert=4096, group=32,
                   format=nat.WEIGHT_DENSE, param_dtype=0)
    args = {**OK, "up": ctypes.addressof(w), "down": ctypes.addressof(w), missing: None}
    assert nat.load().mgq_experts_decode(*args.values()) == nat.ERR_VALUE
    assert "experts_decode" in nat.last_error()


@pytest.mark.parametrize("change", [
    # one row: 16 experts of 2^27 gate rows, 64 to a workgroup of 256
    dict(T=1, H=1, I=1 << 27, ldx=1, k=16, E=16, up=dict(format=nat.WEIGHT_DENSE, ld=1, expert=1 << 28),
         down=dict(ld=1 << 27)),
    # 2^27 columns of the result, 16 to a workgroup of 512
    dict(T=1, H=1 << 27, I=1, ldx=1 << 27, k=1, E=1,
         up=dict(format=nat.WEIGHT_DENSE, ld=1 << 27, expert=1 << 28), down=dict(ld=1)),
])
def test_more_workgroups_than_a_launch_holds(change):
    assert entry(ws_bytes=1 << 50, **change) == nat.ERR_SHAPE
    assert "too many output tiles" in nat.last_error()
