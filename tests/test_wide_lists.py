"""Lists of 64-bit and unsigned integers: what 32 bits do not hold stays out of range."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear
from mlx_gptq.experts import ExpertMLP

TOP, LOW = 2**31 - 1, -(2**31)
CASES = [
    (torch.int64, [3, -1, 2**31, 2**32 + 3, -(2**32), 2**63 - 1, -(2**63)],
     [3, -1, TOP, TOP, LOW, TOP, LOW]),
    (torch.uint64, [3, 2**31, 2**32, 2**32 + 3, 2**63, 2**63 + 5, 2**64 - 1], [3] + [TOP] * 6),
    (torch.uint32, [3, 2**31 - 1, 2**31, 2**32 - 1], [3, TOP, TOP, TOP]),
    (torch.uint16, [3, 2**16 - 1], [3, 2**16 - 1]),
    (torch.uint8, [3, 255], [3, 255]),
    (torch.int16, [3, -(2**15)], [3, -(2**15)]),
]


@pytest.mark.parametrize("dtype,values,want", CASES)
def test_narrowing(dtype, values, want):
    got = linear._int32(torch.tensor(values, dtype=dtype))
    assert got.dtype is torch.int32 and got.tolist() == want


@pytest.mark.parametrize("dtype,value", [(torch.uint64, 2**32 + 1), (torch.uint64, 2**63 + 1),
                                         (torch.uint32, 2**31 + 1)])
def test_an_expert_that_32_bits_do_not_hold_is_none(dtype, value, monkeypatch):
    passed = []
    monkeypatch.setattr(linear, "_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(linear, "_dense", lambda t, dev: passed.append(t) or t)
    monkeypatch.setattr(nat, "launch", lambda *args: None)
    layer = ExpertMLP(torch.zeros(4, 64, 32, dtype=torch.bfloat16), torch.zeros(4, 32, 32, dtype=torch.bfloat16))
    layer.decode(torch.zeros(2, 32, dtype=torch.bfloat16), torch.tensor([[0], [value]], dtype=dtype),
                 torch.ones(2, 1))
    ids = passed[0].flatten().tolist()
    assert ids[0] == 0 and not 0 <= ids[1] < 4
