"""Matrix products and their row operators at row counts past 2^24, 2^26 and 2^31."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
ULP = 2.0**-8  # of bf16


@pytest.mark.parametrize("K", [1, 8])
def test_more_rows_than_an_index_can_name(K):
    """Gathers from rows past 2^31 in all: the index names rows up to 2^31 - 1, by
    rows on 16-byte boundaries (K = 8) and off them. Sums of four small whole numbers
    are exact."""
    rows = 2**31 + 5
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device=DEV)
    index = torch.tensor([2**31 - 1, 0, 5, 2**31 - 1], dtype=torch.int32)
    values = torch.arange(1, 3 * K + 1, dtype=torch.bfloat16).view(3, K) % 13
    for i, r in enumerate((0, 5, 2**31 - 1)):
        x[r] = values[i]
    picked = values[torch.tensor([2, 0, 1, 2])]
    g = torch.Generator().manual_seed(K)
    dy = torch.randint(-4, 5, (4, 6), generator=g).to(torch.bfloat16)
    off = [0, 3, 4]
    dw = linear.grouped_linear_wgrad(dy.to(DEV), x, off, index.to(DEV), out_dtype=torch.float32)
    want, _ = ref.wgrad(dy, picked, off)
    assert torch.equal(dw.cpu().double(), want)
    w = torch.randint(-4, 5, (2, 6, K), generator=g).to(torch.bfloat16)
    y = linear.grouped_linear(x, w.to(DEV), off, index.to(DEV))
    want, _ = ref.forward(picked, w, off)
    assert bool(((y.cpu().double() - want).abs() <= ULP * want.abs()).all())
