"""Every tile that a product with affine weights can take, for each number of bits: tiles of
two and of four row blocks, by loads straight into LDS and by way of registers, several
stages long with a last one that the rows end in. Tolerances are those of
test_gpu_affine_linear.py."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_affine_linear import DEV, TYPES, check, rows, weight

pytestmark = pytest.mark.gpu

# (bits, 2 direct / 3 staged, tile): entries, columns, K, groups, bytes that the rows are off 16
TILES = {
    (2, 2, 64, 128): (10987, 66, 192, 16, 0), (2, 2, 64, 256): (9387, 131, 192, 0, 0),
    (2, 2, 128, 256): (14468, 65, 192, 60, 0), (2, 2, 256, 256): (1310, 1296, 192, 60, 0),
    (2, 3, 64, 128): (12738, 66, 192, 8, 2), (2, 3, 64, 256): (5332, 281, 192, 8, 2),
    (2, 3, 128, 256): (15906, 66, 192, 60, 2),
    (4, 2, 64, 128): (11107, 68, 160, 2, 0), (4, 2, 64, 256): (9098, 135, 160, 8, 0),
    (4, 2, 128, 256): (16349, 74, 160, 4, 0), (4, 2, 256, 256): (1112, 1355, 160, 60, 0),
    (4, 3, 64, 128): (13164, 72, 160, 0, 2), (4, 3, 64, 256): (10379, 132, 160, 32, 2),
    (4, 3, 128, 256): (14633, 134, 160, 60, 2),
    (8, 2, 64, 128): (10898, 66, 160, 2, 0), (8, 2, 64, 256): (9278, 133, 160, 4, 0),
    (8, 2, 128, 256): (16132, 66, 160, 8, 0), (8, 2, 256, 256): (1148, 1292, 160, 60, 0),
    (8, 3, 64, 128): (12558, 66, 160, 8, 2), (8, 3, 64, 256): (11523, 131, 160, 8, 2),
    (8, 3, 128, 256): (16176, 67, 160, 60, 2),
}


@pytest.mark.parametrize("tile", sorted(TILES))
@pytest.mark.parametrize("dtype,params", [("bf16", "f32"), ("f16", "f16")])
def test_every_tile(tile, dtype, params):
    bits, *took = tile
    M, N, K, G, off16 = TILES[tile]
    q, s, b = weight(max(G, 1), N, K, bits, 32, params, seed=M)
    store = torch.zeros(M * K + 8, dtype=TYPES[dtype], device=DEV)
    x = store[off16 // 2:off16 // 2 + M * K].view(M, K)
    x.copy_(rows(M, K, dtype))
    offsets = None
    if G:
        cuts = torch.randint(0, M + 1, (G - 1,), generator=torch.Generator().manual_seed(5)).sort().values
        offsets = [0, *cuts.tolist(), M]
    assert list(check(x, q, s, b, bits, offsets)[1]) == took
