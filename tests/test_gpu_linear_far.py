"""Matrix products and their row operators at row counts past 2^24, 2^26 and 2^31."""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
ULP = 2.0**-8  # of bf16


@pytest.fixture(autouse=True)
def large_tensors_go_back():
    yield
    torch.cuda.empty_cache()


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


@pytest.mark.parametrize("rows,cols", [(2**26 + 5, 3), (2**24 + 3, 1030)])
def test_quantizing_more_rows_than_one_launch_holds(rows, cols):
    """Past 2^26 rows of a wave and 2^24 of a workgroup (fp32 rows of 1030): the first
    and last rows, and those around 2^23 and its multiples, against the oracle."""
    x = torch.ones(rows, cols, device=DEV)
    at = sorted({r for k in range(0, rows + 2**23, 2**23) for r in (k - 1, k, k + 1)} | {rows - 1})
    at = torch.tensor([r for r in at if 0 <= r < rows])
    sample = torch.randn(len(at), cols, generator=torch.Generator().manual_seed(cols))
    x[at.to(DEV)] = sample.to(DEV)
    q, s = linear.quantize_rows_int8(x)
    del x
    wq, ws = ref.quantize_rows(sample)
    assert torch.equal(q[at.to(DEV)].cpu(), wq) and torch.equal(s[at.to(DEV)].cpu(), ws)
    # all the others are ones: scale 1 / 127, codes 127
    assert int((s != torch.tensor(1.0) / 127).sum()) <= len(at)
    assert int((q != 127).sum()) <= sample.numel()


def test_more_summed_rows_than_one_launch_holds():
    """dX of 2^26 + 7 rows of one column, of which seven are read."""
    rows = 2**26 + 7
    at = torch.tensor([0, 2**23 - 1, 2**23, 2**25 + 1, rows - 1, 3, 0], dtype=torch.int32)
    dy = torch.arange(1, 8, dtype=torch.bfloat16).view(7, 1)
    w = torch.full((1, 1), 2.0, dtype=torch.bfloat16)
    dx = linear.grouped_linear_dgrad(dy.to(DEV), w.to(DEV), row_index=at.to(DEV), n_rows=rows)
    want = torch.zeros(rows, dtype=torch.float64).index_add_(0, at.long(), 2.0 * dy.double()[:, 0])
    assert torch.equal(dx[:, 0].cpu().double(), want)


def test_a_product_past_the_few_rows_kernels_launch():
    """One entry for each of 4096 experts of 65536 rows: more workgroups of the kernel
    for few rows than a launch holds, but not of a tile kernel. Sums of 16 products up
    to 4 are exact in bf16."""
    G, N, K = 4096, 65536, 16
    g = torch.Generator(DEV).manual_seed(8)
    w = torch.randint(-2, 3, (G, N, K), generator=g, device=DEV, dtype=torch.int8).to(torch.bfloat16)
    x = torch.randint(-2, 3, (G, K), generator=g, device=DEV).to(torch.bfloat16)
    y = linear.grouped_linear(x, w, torch.arange(G + 1, device=DEV, dtype=torch.int32), validate=False)
    for a in range(0, G, 256):
        want = (w[a : a + 256].float() * x[a : a + 256, None].float()).sum(-1)
        assert torch.equal(y[a : a + 256].float(), want), a
