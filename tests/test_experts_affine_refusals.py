"""What a routed layer with affine weights refuses in forward. No device work."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear
from mlx_gptq.experts import ExpertMLP

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def launches(monkeypatch):
    made = []
    monkeypatch.setattr(linear, "_device", lambda *tensors: torch.device("cpu"))
    monkeypatch.setattr(nat, "launch", lambda dev, name, *args: made.append((name, *args)))
    return made


def layer_of(bits, group, E=4, H=256, I=128):
    def w(n, k):
        return (torch.zeros(E, n, k * bits // 32, dtype=torch.int32),
                *(torch.zeros(E, n, k // group, dtype=BF) for _ in range(2)))

    return ExpertMLP(w(2 * I, H), w(H, I), "affine")


def forward(layer, H, T=3):
    return layer(torch.zeros(T, H, dtype=BF), torch.zeros(T, 2, dtype=torch.int64), torch.zeros(T, 2))


@pytest.mark.parametrize("bits,group,H", [(4, 64, 128), (4, 128, 128), (2, 128, 64), (2, 128, 128),
                                          (2, 64, 128), (4, 32, 512), (8, 32, 512), (8, 64, 512),
                                          (4, 64, 192), (4, 64, 0)])
def test_rows_of_another_width(bits, group, H, launches):
    """The same words are codes of half the bits for rows of twice the width: the layer's
    own sizes say how many bits its codes have."""
    with pytest.raises(AssertionError):
        forward(layer_of(bits, group), H)
    assert not launches


@pytest.mark.parametrize("bits,group", [(2, 32), (4, 64), (8, 128)])
def test_rows_of_its_width(bits, group, launches):
    assert forward(layer_of(bits, group), 256).shape == (3, 256)
    assert [(a[0], a[11]) for a in launches] == [("mgq_affine_linear", bits)] * 2
