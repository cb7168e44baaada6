"""What the matrix products refuse, before any device work."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call,error", [
    (lambda: linear.grouped_linear(z(4, 8, dtype=F32), z(2, 3, 8, dtype=F32), [0, 2, 4]), TypeError),
    (lambda: linear.grouped_linear(z(4, 8), z(2, 3, 8, dtype=F16), [0, 2, 4]), TypeError),
    (lambda: linear.grouped_linear(z(4, 8), z(2, 3, 9), [0, 2, 4]), AssertionError),
    (lambda: linear.grouped_linear(z(4, 8), z(3, 8), [0, 4]), ValueError),
    (lambda: linear.grouped_linear(z(4, 8), z(2, 3, 8)), ValueError),
    (lambda: linear.grouped_linear(z(2, 4, 8), z(3, 8)), ValueError),
    (lambda: linear.grouped_linear_dgrad(z(4, 8), z(2, 3, 9), [0, 2, 4]), AssertionError),
    (lambda: linear.grouped_linear_dgrad(z(4, 3), z(2, 3, 9), [0, 2, 4],
                                         torch.zeros(4, dtype=torch.int32)), ValueError),
    (lambda: linear.grouped_linear_wgrad(z(4, 3), z(4, 8), [0, 4], out_dtype=F16), TypeError),
    (lambda: linear.grouped_linear_wgrad(z(4, 3), z(4, 8, dtype=F16), [0, 4]), TypeError),
    (lambda: linear.mxfp_linear(z(4, 32), z(3, 4, dtype=torch.int32), z(3, 1, dtype=torch.uint8),
                                "affine"), ValueError),
    (lambda: linear.mxfp_linear(z(4, 32, dtype=F16), z(3, 4, dtype=torch.int32),
                                z(3, 1, dtype=torch.uint8), "mxfp4"), TypeError),
    (lambda: linear.mxfp_linear(z(4, 32), z(3, 4, dtype=torch.uint8), z(3, 1, dtype=torch.uint8),
                                "mxfp4"), TypeError),
    (lambda: linear.mxfp_linear(z(4, 24), z(3, 3, dtype=torch.int32), z(3, 1, dtype=torch.uint8),
                                "mxfp4"), AssertionError),
    (lambda: linear.mxfp_linear(z(4, 32), z(3, 4, dtype=torch.int32), z(3, 2, dtype=torch.uint8),
                                "mxfp4"), AssertionError),
    (lambda: linear.quantize_rows_int8(z(4, 8, dtype=torch.int32)), TypeError),
    (lambda: linear.quantize_rows_int8(z(4, 0)), ValueError),
    (lambda: linear.int8_linear(z(4, 8), z(4, dtype=F32), z(3, 8, dtype=I8), z(3, dtype=F32)), TypeError),
    (lambda: linear.int8_linear(z(4, 8, dtype=I8), z(4), z(3, 8, dtype=I8), z(3, dtype=F32)), TypeError),
    (lambda: linear.int8_linear(z(4, 8, dtype=I8), z(4, dtype=F32), z(3, 8, dtype=I8),
                                z(3, dtype=F32), out_dtype=I8), TypeError),
    (lambda: linear.int8_linear(z(4, 8, dtype=I8), z(5, dtype=F32), z(3, 8, dtype=I8),
                                z(3, dtype=F32)), AssertionError),
    (lambda: linear.int8_linear(z(4, 8, dtype=I8), z(4, dtype=F32), z(3, 7, dtype=I8),
                                z(3, dtype=F32)), AssertionError),
])
def test_arguments(call, error):
    with pytest.raises(error):
        call()


CPU = torch.device("cpu")


@pytest.mark.parametrize("offsets,index,error", [
    ([0, 2], None, ValueError),  # one group's offsets for two groups
    ([0, 3, 2], None, ValueError),
    ([-1, 2, 3], None, ValueError),
    ([0, 2, 5], None, ValueError),  # more entries than rows
    (torch.tensor([0.0, 1.0, 2.0]), None, ValueError),
    ([0, 1, 3], torch.tensor([0, 1, 4]), IndexError),
    ([0, 1, 3], torch.tensor([0, -1, 2]), IndexError),
    ([0, 1, 3], torch.tensor([0.0, 1.0, 2.0]), ValueError),
    ([0, 1, 4], torch.tensor([0, 1, 2]), ValueError),
])
def test_lists(offsets, index, error):
    with pytest.raises(error):
        linear._list("fn", offsets, index, 2, 4, CPU, True)


def test_list_without_validation_leaves_the_device_alone():
    off, idx, entries = linear._list("fn", [0, 1, 3], torch.tensor([3, 2, 1, 0]), 2, 4, CPU, False)
    assert off.dtype == torch.int32 and idx.dtype == torch.int32 and entries == 4


def _rc(name, *args):
    return getattr(nat.load(), name)(*args)


def test_entry_points_return_a_status():
    """Bad sizes end at the C entry with a status and a message, before any
    pointer is used."""
    i8 = (1, 1, 1, 1, None, 1, 1, 1, None, 1, 4, 131072, 131072, 0, None, 1, nat.DTYPE_BF16, None)
    i8 = list(i8)
    i8[3] = 131072  # ldx
    assert _rc("mgq_int8_linear", *i8) == nat.ERR_SHAPE and "131071" in nat.last_error()
    gl = [1, nat.DTYPE_F32, 4, 8, None, 4, 1, 1, 3, 8, 8, 0, None, 1, None]
    assert _rc("mgq_grouped_linear", *gl) == nat.ERR_VALUE
    gl[1] = nat.DTYPE_BF16
    gl[3] = 7  # pitch below a row
    assert _rc("mgq_grouped_linear", *gl) == nat.ERR_SHAPE
    gl[3], gl[7] = 8, 2  # two groups, no offsets
    assert _rc("mgq_grouped_linear", *gl) == nat.ERR_VALUE and "offsets" in nat.last_error()
    gl[7], gl[5] = 1, 5  # more entries than rows
    assert _rc("mgq_grouped_linear", *gl) == nat.ERR_SHAPE
    mx = [1, 4, 32, None, 4, 1, 1, 7, 1, 3, 32, None, 1, None]
    assert _rc("mgq_mxfp_linear", *mx) == nat.ERR_VALUE
    mx[7], mx[10] = nat.MODE_MXFP4, 33
    assert _rc("mgq_mxfp_linear", *mx) == nat.ERR_SHAPE
    assert _rc("mgq_quantize_rows_int8", 1, 7, 4, 8, 8, 1, 1, None) == nat.ERR_VALUE
    assert _rc("mgq_rows_sum", 1, 1, 4, 4, 4, 1, nat.DTYPE_BF16, None, 0, None) == nat.ERR_WORKSPACE
    dg = [1, nat.DTYPE_BF16, 4, 8, 1, 1, 8, 3, 3, 0, None, 1, nat.DTYPE_F16, None]
    assert _rc("mgq_grouped_dgrad", *dg) == nat.ERR_VALUE
    wg = [1, nat.DTYPE_BF16, 4, 2, 1, 4, 8, None, 1, 3, 8, None, 1, nat.DTYPE_BF16, None, 0, None]
    assert _rc("mgq_grouped_wgrad", *wg) == nat.ERR_SHAPE  # lddy < N


def test_weight_gradient_takes_4096_groups():
    wg = [1, nat.DTYPE_BF16, 4, 8, 1, 4, 8, None, 4097, 8, 8, 1, 1, nat.DTYPE_BF16, 1, 1 << 40, None]
    assert _rc("mgq_grouped_wgrad", *wg) == nat.ERR_SHAPE and "4096" in nat.last_error()


def test_more_tiles_than_a_launch_holds_are_refused():
    gl = [16, nat.DTYPE_BF16, 1 << 30, 8, None, 1 << 30, 16, 1, 1 << 29, 8, 8, 0, None, 16, None]
    assert _rc("mgq_grouped_linear", *gl) == nat.ERR_SHAPE and "tiles" in nat.last_error()
