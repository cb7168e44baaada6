"""Contractions of no terms: sums of nothing are zero, whatever kernel is chosen."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("M,G", [(1, 0), (5, 3), (700, 0), (3000, 9)])
def test_no_columns(M, G):
    gs = [G] if G else []
    off = torch.arange(G + 1, dtype=torch.int32, device=DEV) if G else None
    x = torch.empty(M, 0, dtype=torch.bfloat16, device=DEV)
    w = torch.empty(*gs, 130, 0, dtype=torch.bfloat16, device=DEV)
    y = linear.grouped_linear(x, w, off)
    assert y.shape == (M, 130) and not bool(y.any())
    dy = torch.ones(M, 130, dtype=torch.bfloat16, device=DEV)
    assert linear.grouped_linear_dgrad(dy, w, off).shape == (M, 0)
    assert linear.grouped_linear_wgrad(dy, x, off).shape == (*gs, 130, 0)
    y = linear.mxfp_linear(x, torch.empty(*gs, 130, 0, dtype=torch.int32, device=DEV),
                           torch.empty(*gs, 130, 0, dtype=torch.uint8, device=DEV), "mxfp4", off)
    assert not bool(y.any())
    bias = torch.arange(130, dtype=torch.float32, device=DEV).expand(*gs, 130).contiguous()
    y = linear.int8_linear(x.to(torch.int8), torch.ones(M, device=DEV), w.to(torch.int8),
                           torch.ones(*gs, 130, device=DEV), bias, torch.float32, off)
    n = G or M  # the entries of a group
    assert torch.equal(y[:n], bias.view(-1, 130)[:1].expand(n, -1)) and not bool(y[n:].any())


@pytest.mark.parametrize("M,G", [(4, 0), (4, 3)])
def test_no_output_features(M, G):
    gs = [G] if G else []
    off = torch.arange(G + 1, dtype=torch.int32, device=DEV) if G else None
    x = torch.ones(M, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.empty(*gs, 0, 64, dtype=torch.bfloat16, device=DEV)
    assert linear.grouped_linear(x, w, off).shape == (M, 0)
    dx = linear.grouped_linear_dgrad(torch.empty(M, 0, dtype=torch.bfloat16, device=DEV), w, off)
    assert dx.shape == (M, 64) and not bool(dx.any())
    idx = torch.zeros(M, dtype=torch.int32, device=DEV)
    dx = linear.grouped_linear_dgrad(torch.empty(M, 0, dtype=torch.bfloat16, device=DEV), w, off, idx, 7)
    assert dx.shape == (7, 64) and not bool(dx.any())
