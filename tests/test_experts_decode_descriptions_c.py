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
