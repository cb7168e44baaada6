"""A routed layer's forward in a graph: the routing stays on the device."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq.experts import ExpertMLP

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("mode", ExpertMLP.MODES)
@pytest.mark.parametrize("T,k", [(1, 2), (64, 4), (700, 2)])
def test_replays_give_the_eager_results(mode, T, k):
    g = torch.Generator(DEV).manual_seed(T)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV).to(torch.bfloat16)

    def routing():  # with ids of no expert on both sides
        return torch.randint(-1, 9, (T, k), generator=g, device=DEV)

    mlp = ExpertMLP.from_weights(randn(8, 128, 64), randn(8, 64, 64), mode)
    x, index, weights = randn(T, 64), routing(), torch.rand(T, k, generator=g, device=DEV)
    mlp(x, index, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(x, index, weights)
    for seed in range(4):
        x.copy_(randn(T, 64))
        index.copy_(routing())
        weights.copy_(torch.rand(T, k, generator=g, device=DEV))
        want = mlp(x, index, weights)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), seed
