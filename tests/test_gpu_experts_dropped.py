"""Assignments to no expert add nothing to a row, whatever the router left as their
weight: a softmax over scores that are all masked is NaN."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq.experts import ExpertMLP

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("mode", ExpertMLP.MODES)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 3.0])
def test_weights_of_no_expert_count_for_nothing(mode, value):
    g = torch.Generator().manual_seed(2)
    gate_up = torch.randn(4, 64, 64, generator=g).to(DEV, torch.bfloat16)
    down = torch.randn(4, 64, 32, generator=g).to(DEV, torch.bfloat16)
    x = torch.randn(9, 64, generator=g).to(DEV, torch.bfloat16)
    index = torch.stack([torch.randperm(4, generator=g)[:2] for _ in range(9)]).to(DEV)
    weights = torch.rand(9, 2, generator=g).to(DEV)
    mlp = ExpertMLP.from_weights(gate_up, down, mode)
    drop = torch.zeros(9, 2, dtype=torch.bool, device=DEV)
    drop[::3, 0] = True
    drop[4] = True  # a row that reaches no expert
    index[drop] = torch.tensor([-1, 4, 2**40], device=DEV).repeat(3)[: int(drop.sum())]
    want = mlp(x, index, weights.masked_fill(drop, 0.0))
    left = weights.masked_fill(drop, value).requires_grad_()
    y = mlp(x, index, left)
    assert torch.equal(y, want) and not bool(y[4].any())
    y.float().sum().backward()
    assert bool(torch.isfinite(left.grad).all()) and not bool(left.grad[drop].any())


def test_gradients_of_rows_and_experts_stay_finite():
    g = torch.Generator().manual_seed(3)
    leaves = [torch.randn(*s, generator=g).to(DEV, torch.bfloat16).requires_grad_()
              for s in ((4, 64, 64), (4, 64, 32), (9, 64))]
    index = torch.randint(0, 4, (9, 1), generator=g).to(DEV)
    index[5] = -1
    weights = torch.ones(9, 1, device=DEV)
    weights[5] = float("nan")
    ExpertMLP(*leaves[:2])(leaves[2], index, weights).float().sum().backward()
    assert all(bool(torch.isfinite(t.grad).all()) for t in leaves)
    assert not bool(leaves[2].grad[5].any())
