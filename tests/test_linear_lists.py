"""The lists that the matrix products take: their types and their conversion to
32 bits, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_gptq import linear

CPU = torch.device("cpu")
FAR = [2**31, 2**32, 2**32 + 3, 2**40 + 1, 2**63 - 1, -(2**31) - 1, -(2**32) + 2, -(2**63)]


@pytest.mark.parametrize("dtype", [torch.bool, torch.complex64])
def test_lists_are_integers(dtype):
    with pytest.raises(ValueError, match="integers"):
        linear._list("fn", [0, 1, 3], torch.ones(3, dtype=dtype), 2, 4, CPU, False)
    with pytest.raises(ValueError, match="integers"):
        linear._list("fn", torch.ones(3, dtype=dtype), None, 2, 4, CPU, False)


@pytest.mark.parametrize("offsets", [[0.0, 1.5, 3.0], np.array([0, 1.9, 2]), [0, float("nan"), 2]])
def test_host_offsets_are_whole(offsets):
    with pytest.raises(ValueError, match="integers"):
        linear._list("fn", offsets, None, 2, 4, CPU, True)


@pytest.mark.parametrize("offsets", [[0, 1, 3], (0, 1, 3), np.array([0.0, 1.0, 3.0]), range(0, 9, 4)])
def test_host_offsets(offsets):
    off, _, _ = linear._list("fn", offsets, None, 2, 8, CPU, True)
    assert off.tolist() == [int(v) for v in offsets] and off.dtype == torch.int32


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_integer_types(dtype):
    off, idx, entries = linear._list("fn", torch.tensor([0, 1, 3], dtype=dtype),
                                     torch.tensor([3, 0, 2], dtype=dtype), 2, 4, CPU, True)
    assert off.tolist() == [0, 1, 3] and idx.tolist() == [3, 0, 2] and entries == 3
    assert off.dtype == idx.dtype == torch.int32


def test_indexes_past_32_bits_are_clamped_not_wrapped():
    """2^32 + 3 is past every row and must not come to read row 3."""
    index = torch.tensor([1, *FAR])
    _, idx, _ = linear._list("fn", None, index, 1, 4, CPU, False)
    assert idx.tolist() == [min(max(v, -(2**31)), 2**31 - 1) for v in index.tolist()]


def test_offsets_past_32_bits_are_clamped_not_wrapped():
    """(a device's unvalidated offsets: host ones are always checked)"""
    offsets = torch.tensor([0, *FAR])
    assert linear._int32(offsets).tolist() == [min(max(v, -(2**31)), 2**31 - 1)
                                               for v in offsets.tolist()]
