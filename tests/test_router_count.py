"""top_k_softmax takes a whole number of experts. No device work."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear
from mlx_gptq.experts import top_k_softmax


@pytest.mark.parametrize("k", [2.7, 2.0, "2", None, torch.tensor(2.5)])
def test_no_whole_number(k):
    with pytest.raises(TypeError):
        top_k_softmax(torch.zeros(4, 8), k)


@pytest.mark.parametrize("k", [2, np.int64(2), torch.tensor(2)])
def test_whole_numbers(k, monkeypatch):
    passed = []
    monkeypatch.setattr(linear, "_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(nat, "launch", lambda dev, name, *args: passed.append(args[5]))
    index, weights = top_k_softmax(torch.zeros(4, 8), k)
    assert index.shape == weights.shape == (4, 2) and passed == [2]
