"""The sum of list entries per row that ends a gathered product's gradient, at every
number of entries a row can have.

The entries' sums are compared bit for bit with fp32 additions in the list's order, and
the product in front is exact: dY and W hold small whole numbers.
"""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def in_order(dy, w, index, n_rows):
    """fp32 sums in the list's order, on the CPU: the k-th entry of every row at once."""
    terms = (dy.double() @ w.double()).float()
    order = torch.sort(index.long(), stable=True).indices
    counts = torch.bincount(index.long(), minlength=n_rows)
    starts = counts.cumsum(0) - counts
    total = torch.zeros(n_rows, w.shape[1])
    for k in range(int(counts.max())):
        rows = torch.nonzero(counts > k).flatten()
        total[rows] += terms[order[starts[rows] + k]]
    return total


def case(counts, K, seed):
    g = torch.Generator().manual_seed(seed)
    index = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts))
    index = index[torch.randperm(len(index), generator=g)].to(torch.int32)
    # products up to 2^22 and 2^12, whose sum is exact in fp32; that of several is not
    dy = torch.randint(-64, 65, (len(index), 2), generator=g).to(torch.bfloat16)
    w = torch.randint(-64, 65, (2, K), generator=g).to(torch.bfloat16)
    dy[:, 0] *= 2.0**10
    return dy, w, index


def check(counts, K, seed):
    dy, w, index = case(counts, K, seed)
    want = in_order(dy, w, index, len(counts)).to(torch.bfloat16)
    got = [linear.grouped_linear_dgrad(dy.to(DEV), w.to(DEV), row_index=index.to(DEV),
                                       n_rows=len(counts)) for _ in range(3)]
    assert torch.equal(got[0].cpu(), want)
    assert all(torch.equal(got[0], g) for g in got[1:])


@pytest.mark.parametrize("K", [1, 70, 1030])
def test_every_count_around_its_limits(K):
    """0, the slots, one batch and several of a chain, and beside them enough other
    entries for the chain to be the shorter way."""
    counts = [0, 1, 15, 16, 17, 18, 31, 63, 64, 65, 127, 128, 129, 200, 300, 0]
    check(counts + [2] * 30000, K, K)


@pytest.mark.parametrize("M", [100, 5000, 70000])
def test_hot_rows(M):
    """Rows that hold a large part of the list, which is then read whole."""
    check([M // 2, 0, M // 4, 17, M // 8, 1], 33, M)


@pytest.mark.parametrize("top_k", [17, 24, 70])
def test_every_row_read_by_many(top_k):
    check([top_k] * 3000, 40, top_k)


def test_one_entry_and_none():
    check([0, 1, 0], 8, 1)
    w = torch.ones(1, 2, 8, dtype=torch.bfloat16, device=DEV)
    dx = linear.grouped_linear_dgrad(torch.empty(0, 2, dtype=torch.bfloat16, device=DEV), w, [0, 0],
                                     torch.empty(0, dtype=torch.int32, device=DEV), 300)
    assert dx.shape == (300, 8) and not bool(dx.any())


def test_time_grows_with_the_list():
    """16384 rows read 24 times each hold 1.5 times the entries of rows read 16 times.
    Reading the list once for every row would take some hundred times as long."""
    times = {}
    for top_k in (16, 24):
        dy, w, index = case([top_k] * 16384, 64, top_k)
        args = dy.to(DEV), w.to(DEV), None, index.to(DEV), 16384, False
        for _ in range(3):
            linear.grouped_linear_dgrad(*args)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            linear.grouped_linear_dgrad(*args)
        b.record()
        b.synchronize()
        times[top_k] = a.elapsed_time(b) / 5
    print(times)
    assert times[24] < 8 * times[16], times


def test_captured():
    """The sum's launches in a graph, replayed with new lists in the same tensors."""
    dy, w, index = case([30] * 200, 24, 3)
    dyd, wd, idx = dy.to(DEV), w.to(DEV), index.to(DEV)

    def call():
        return linear.grouped_linear_dgrad(dyd, wd, None, idx, 200, False)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        idx.copy_(torch.randint(0, 200 if seed % 2 else 3, index.shape, generator=g, dtype=torch.int32))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), seed
