"""Launches of the affine products, of a routed layer for a few rows and of the router's
choice go to the device of their tensors, whichever is current. The library and the
devices are stand-ins: this runs without a GPU."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import experts, linear
from tests.test_launch_device import devices  # noqa: F401


@pytest.mark.parametrize("index", [0, 1])
def test_launches_go_to_their_tensors_device(devices, monkeypatch, index):  # noqa: F811
    dev = torch.device("cpu", index)  # (host tensors, said to be of that device)
    for module in (linear, experts.linear):
        monkeypatch.setattr(module, "_device", lambda *tensors: dev)
    monkeypatch.setattr(nat, "device_for", lambda *tensors: dev)
    x = torch.ones(4, 32, dtype=torch.bfloat16)
    params = torch.ones(3, 1)
    linear.affine_linear(x, torch.zeros(3, 4, dtype=torch.int32), params, params, 4)
    mlp = experts.ExpertMLP(torch.ones(2, 64, 32, dtype=torch.bfloat16),
                            torch.ones(2, 32, 32, dtype=torch.bfloat16))
    mlp.decode(x, torch.zeros(4, 1, dtype=torch.int64), torch.ones(4, 1))
    logits = torch.ones(4, 8)
    chosen, weights = experts.top_k_softmax(logits, 2)
    experts.top_k_softmax_grad(weights, logits, chosen)
    launched = [c for c in devices.calls if not c[0].endswith("_size")]
    assert [c[0] for c in launched] == ["mgq_affine_linear", "mgq_experts_decode",
                                        "mgq_top_k_softmax", "mgq_top_k_softmax_grad"]
    assert {c[1] for c in launched} == {index} and devices.current == 0
