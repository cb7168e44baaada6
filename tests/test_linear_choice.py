"""The choice of kernels holds every product that some kernel's launch holds. No GPU:
the choice is the host's."""

from __future__ import annotations

import math
import random

import pytest

from tests.linear_choice import DIRECT, FEW, PRODUCTS, STAGED, choice

# what a launch holds: less than 2^32 threads
MOST = {FEW: 2**24, DIRECT: 2**23, STAGED: 2**23}


def grid(M, G, cols, grouped, tile):
    rows = M // tile[0] + min(G + 2, M) if grouped else math.ceil(M / tile[0])
    return rows * math.ceil(cols / tile[1])


TILES = {FEW: [(16, 16), (32, 16), (64, 32)], DIRECT: [(64, 128), (64, 256), (128, 256), (256, 256)],
         STAGED: [(64, 128), (64, 256), (128, 256)]}


@pytest.mark.parametrize("product", sorted(PRODUCTS))
@pytest.mark.parametrize("M,G,N,K,grouped", [
    (4096, 4096, 65536, 32, True),  # one entry for each of many wide experts
    (524288, 1, 65536, 32, False),
    (1 << 20, 1, 1 << 17, 64, False), (1 << 24, 1, 4096, 32, False),
])
def test_a_product_that_some_kernel_holds_is_taken(product, M, G, N, K, grouped):
    if product.startswith("dgrad"):
        N, K = K, N
    tile = choice(product, M, G, N, K, grouped)
    assert grid(M, G, K if product.startswith("dgrad") else N, grouped, tile) < MOST[tile[2]], tile


def test_no_choice_passes_its_launch():
    rng = random.Random(4)

    def size(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))

    taken = refused = 0
    for _ in range(4000):
        product = rng.choice(sorted(PRODUCTS))
        M, N, K = size(1, 1 << 26), size(1, 1 << 22), 32 * size(1, 64)
        grouped = rng.random() < 0.5
        G = size(1, 1 << 16) if grouped else 1
        dgrad = product.startswith("dgrad")
        if dgrad:
            N, K = K, N
        cols = K if dgrad else N
        x = rng.choice((0, 0, 2, 4))
        # off 16 bytes: rows through registers
        direct = x == 0 and (dgrad and K % 8 == 0 or not dgrad)
        kinds = ([] if dgrad else [FEW]) + [DIRECT if direct else STAGED]
        fits = any(grid(M, G, cols, grouped, t) < MOST[k] for k in kinds for t in TILES[k])
        try:
            tile = choice(product, M, G, N, K, grouped, x=x)
        except AssertionError as e:
            assert "tiles" in str(e) and not fits, (product, M, G, N, K, grouped, x)
            refused += 1
            continue
        assert fits and tile[2] in kinds and tile[:2] in TILES[tile[2]]
        assert grid(M, G, cols, grouped, tile) < MOST[tile[2]], (product, M, G, N, K, tile)
        taken += 1
    assert taken > 1000 and refused > 100
