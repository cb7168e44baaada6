"""The kernel for few rows in every form that a call reaches: operand type, entries of
a workgroup (16, 32, 64), rows on and off 16-byte and 4-byte boundaries. Each test
asserts that the host chooses the form it is about.

The tolerance is that of the other products' tests: n 2^-23 sum|terms| for a sum of n
terms in fp32, and half an ulp of the result's type (2^-8 relative for bf16, 2^-11 for
f16, with half of its subnormal step); int8 sums are exact, their scaling is within
5 2^-24.
"""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear, packing
from oracle import linear_ref as ref
from tests.linear_choice import DIRECT, FEW, STAGED, choice, of_call

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25}
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "int8": torch.int8}

# (product, bytes that X's rows start past a boundary) -> entries of a workgroup ->
# entries, groups, N, K
SIZES = {
    ("bf16", 0): {16: (5, 3, 33, 544), 32: (20, 3, 2050, 800), 64: (400, 32, 257, 4128)},
    ("bf16", 2): {16: (5, 3, 33, 800), 32: (5, 3, 4100, 1824), 64: (27, 32, 16846, 32)},
    ("bf16", 4): {16: (5, 3, 33, 288), 32: (60, 8, 1030, 544), 64: (400, 32, 257, 416)},
    ("f16", 0): {16: (5, 3, 33, 544), 32: (20, 3, 2050, 800), 64: (400, 32, 257, 4128)},
    ("f16", 2): {16: (5, 3, 33, 800), 32: (5, 3, 4100, 1824), 64: (174, 128, 1545, 64)},
    ("f16", 4): {16: (5, 3, 33, 288), 32: (60, 8, 1030, 544), 64: (400, 32, 257, 416)},
    ("int8", 0): {16: (5, 3, 33, 1056), 32: (200, 32, 257, 1312), 64: (1000, 32, 4100, 32)},
    ("int8", 1): {16: (5, 3, 33, 1312), 32: (5, 3, 4100, 1824), 64: (1500, 32, 4100, 32)},
    ("int8", 2): {16: (5, 3, 33, 1312), 32: (5, 3, 4100, 1824), 64: (1500, 32, 4100, 32)},
    ("int8", 4): {16: (5, 3, 33, 544), 32: (150, 32, 4100, 96), 64: (400, 32, 257, 800)},
    ("mxfp4", 0): {16: (5, 3, 33, 544), 32: (3000, 32, 33, 800), 64: (1500, 32, 4100, 32)},
    ("mxfp4", 2): {16: (5, 3, 33, 800), 32: (20, 32, 4100, 800), 64: (40, 32, 4100, 288)},
    ("mxfp4", 4): {16: (5, 3, 33, 416), 32: (200, 32, 4100, 64), 64: (250, 32, 4100, 64)},
    ("mxfp8", 0): {16: (5, 3, 33, 544), 32: (200, 32, 257, 800), 64: (1500, 32, 4100, 32)},
    ("mxfp8", 2): {16: (5, 3, 33, 800), 32: (200, 32, 257, 1824), 64: (40, 32, 4100, 160)},
    ("mxfp8", 4): {16: (5, 3, 33, 288), 32: (200, 32, 257, 800), 64: (60, 8, 2050, 416)},
}
CASES = [(p, off, rows, *s) for (p, off), by in SIZES.items() for rows, s in by.items()]
MX_CASES = [c for c in CASES if c[0].startswith("mx")]
PARAMS = "product,off,rows,M,G,N,K"


class Product:
    """Weights [G, N, K], rows [T, K] that start `off` bytes past a boundary, their
    values in float64 and the call."""

    def __init__(self, product, off, T, G, N, K, seed=0):
        self.product, self.K = product, K
        g = self.g = torch.Generator(DEV).manual_seed(seed + N + K)
        dtype = self.dtype = TYPES.get(product, torch.bfloat16)
        e = off // dtype.itemsize
        if product == "int8":
            self.x = torch.randint(-127, 128, (T, K + 16), generator=g, device=DEV,
                                   dtype=torch.int8)[:, e : e + K]
            self.w = torch.randint(-128, 128, (G, N, K), generator=g, device=DEV, dtype=torch.int8)
            self.xs = torch.rand(T, generator=g, device=DEV) * 0.1 + 1e-3
            self.ws = torch.rand(G, N, generator=g, device=DEV) * 1e-2
            return
        self.x = torch.randn(T, K + 16, generator=g, device=DEV).to(dtype)[:, e : e + K]
        if product in TYPES:
            self.w = (torch.randn(G, N, K, generator=g, device=DEV) * 0.1).to(dtype)
            return
        self.bits = 4 if product == "mxfp4" else 8
        self.codes = torch.randint(0, 127, (G, N, K), generator=g, device=DEV,
                                   dtype=torch.uint8) % (1 << self.bits)
        self.scales = torch.randint(115, 131, (G, N, K // 32), generator=g, device=DEV,
                                    dtype=torch.uint8)
        self.w = packing.pack_q(self.codes, self.bits)

    def __call__(self, off, idx=None):
        if self.product == "int8":
            return linear.int8_linear(self.x, self.xs, self.w, self.ws, out_dtype=torch.float32,
                                      offsets=off, row_index=idx, validate=False)
        if self.product in TYPES:
            return linear.grouped_linear(self.x, self.w, off, idx, validate=False)
        return linear.mxfp_linear(self.x, self.w, self.scales, self.product, off, idx, validate=False)

    def weights(self, g):
        if self.product.startswith("mx"):
            return ref.decode(self.codes[g].cpu(), self.scales[g].cpu(), self.product).to(DEV)
        return self.w[g].double()

    def check(self, y, off, idx=None):
        """y against float64 over the spans of the (good) offsets, zeros elsewhere."""
        xs = self.x.double() if idx is None else self.x.double()[idx.long()]
        seen = torch.zeros(len(xs), dtype=torch.bool, device=DEV)
        for g, (a, b) in enumerate(zip(off[:-1], off[1:])):
            if a == b:
                continue
            seen[a:b] = True
            w = self.weights(g)
            want = xs[a:b] @ w.T
            if self.product == "int8":
                s = self.xs.double() if idx is None else self.xs.double()[idx.long()]
                want *= s[a:b, None] * self.ws[g].double()
                tol = 5 * 2.0**-24 * want.abs()
            else:
                mag = xs[a:b].abs() @ w.abs().T
                tol = ((self.K + 8) * 2.0**-23 * mag + UNIT[y.dtype] * want.abs() * 1.01
                       + STEP[y.dtype])
            assert bool(((y[a:b].double() - want).abs() <= tol).all()), g
        assert not bool(y[~seen].any())

    def assert_choice(self, M, off, rows):
        assert of_call(self.product, M, self.x, self.w, off) == (rows, 32 if rows == 64 else 16, FEW)


def spans(M, G, seed, before=0, after=0):
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(before, M - after + 1, (G - 1,), generator=g).sort().values.tolist()
    return [before, *cuts, M - after]


def on(off):
    return torch.tensor(off, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize(PARAMS, CASES)
def test_lists(product, off, rows, M, G, N, K):
    """Groups of every size, entries of no group on both sides, gathered rows, and lists
    that lie: clamped, never followed."""
    T = max(M // 2, 1)
    p = Product(product, off, T, G, N, K)
    idx = torch.randint(0, T, (M,), generator=torch.Generator().manual_seed(M), dtype=torch.int32)
    offsets = spans(M, G, M, before=1, after=2)
    p.assert_choice(M, offsets, rows)
    p.check(p(on(offsets), idx.to(DEV)), offsets, idx.to(DEV))
    offsets = spans(M, G, M + 1)
    lying = [-7, *offsets[1:-1], M + 9000]
    wild = idx.clone()
    wild[1], wild[M - 1] = -(2**31), 2**31 - 1
    p.check(p(on(lying), wild.to(DEV)), offsets, wild.clamp(0, T - 1).to(DEV))


@pytest.mark.parametrize(PARAMS, CASES)
def test_rows_in_their_order(product, off, rows, M, G, N, K):
    p = Product(product, off, M, G, N, K, seed=1)
    offsets = spans(M, G, M + 2)
    p.assert_choice(M, offsets, rows)
    p.check(p(on(offsets)), offsets)


@pytest.mark.parametrize(PARAMS, CASES)
def test_non_finite_values_stay_in_their_rows(product, off, rows, M, G, N, K):
    p = Product(product, off, M, G, N, K, seed=2)
    p.assert_choice(M, spans(M, G, 0), rows)
    # the first group has no entries, the last the second half
    offsets = [1] * (G - 1) + [M // 2, M - 1]
    bad = [M // 2 - 1, M - 2]
    outside = [0, M - 1]
    if product == "int8":
        p.xs[bad + outside] = float("nan")
        p.ws[0] = float("nan")
        p.ws[G - 1, 7] = float("nan")
    else:
        p.x[bad[0], K - 1] = float("nan")
        p.x[bad[1], 0] = float("inf")
        p.x[outside] = float("nan")
        if product in TYPES:
            p.w[0] = float("nan")
            p.w[G - 1, 7, K // 2] = float("nan")
        else:
            p.scales[0] = 255
            p.scales[G - 1, 7, K // 64] = 255
    y = p(on(offsets))
    want = torch.ones_like(y, dtype=torch.bool)
    want[bad] = False
    want[M // 2 : M - 1, 7] = False
    assert torch.equal(torch.isfinite(y), want)
    assert not bool(y[outside].any())


def every_code(product, x, M, G, N, K):
    """Every code under every scale byte, each alone in its weight row, against rows of
    ones: the product is the decoded weight, in bf16 with its subnormals, infinities
    past its range and NaN for MXFP8's NaN codes and scale byte 255."""
    bits = 4 if product == "mxfp4" else 8
    offsets = [round(i * M / G) for i in range(G + 1)]
    owner = torch.bucketize(torch.arange(M), torch.tensor(offsets[1:]), right=True).to(DEV)
    for base in range(0, 256 << bits, G * N):
        pair = (torch.arange(G * N) + base) % (256 << bits)
        code, scale = pair % (1 << bits), pair >> bits
        codes = torch.zeros(G * N, K, dtype=torch.uint8)
        scales = torch.full((G * N, K // 32), 127, dtype=torch.uint8)
        row, block = torch.arange(G * N), (pair * 5 + pair // 32) % (K // 32)
        codes[row, 32 * block + (pair * 7 + pair // 32) % 32] = code.to(torch.uint8)
        scales[row, block] = scale.to(torch.uint8)
        one = torch.zeros(G * N, 32, dtype=torch.uint8)
        one[:, 0] = code
        want = ref.decode(one, scale.to(torch.uint8)[:, None], product)[:, 0]
        want = torch.where(scale == 255, torch.nan, want).float().to(torch.bfloat16)
        packed = packing.pack_q(codes.view(G, N, K).to(DEV), bits)
        y = linear.mxfp_linear(x, packed, scales.view(G, N, -1).to(DEV), product, on(offsets),
                               validate=False)
        expect = want.view(G, N).to(DEV)[owner]
        same = (y == expect) | (torch.isnan(y) & torch.isnan(expect))
        assert bool(same.all()), (base, torch.nonzero(~same)[:4].tolist())


@pytest.mark.parametrize(PARAMS, MX_CASES)
def test_every_code_under_every_scale(product, off, rows, M, G, N, K):
    x = torch.ones(M, K + 16, dtype=torch.bfloat16, device=DEV)[:, off // 2 : off // 2 + K]
    assert choice(product, M, G, N, K, True, x.data_ptr(), 0, K + 16) == (
        rows, 32 if rows == 64 else 16, FEW)
    every_code(product, x, M, G, N, K)


@pytest.mark.parametrize("product", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("off,M,G,N,K,kind", [
    (0, 3, 2, 300, 96, DIRECT), (2, 3, 2, 300, 96, STAGED), (0, 700, 2, 520, 64, DIRECT),
    (2, 900, 2, 520, 64, STAGED), (0, 2100, 3, 4100, 32, DIRECT), (2, 2100, 3, 4100, 32, STAGED),
])
def test_every_code_under_every_scale_by_tiles(product, off, M, G, N, K, kind):
    x = torch.ones(M, K + 16, dtype=torch.bfloat16, device=DEV)[:, off // 2 : off // 2 + K]
    assert choice(product, M, G, N, K, True, x.data_ptr(), 0, K + 16)[2] == kind
    every_code(product, x, M, G, N, K)


@pytest.mark.parametrize(PARAMS, [c for c in CASES if c[2] == 16])
def test_rows_and_weights_beyond_32_bits(product, off, rows, M, G, N, K):
    """Rows and experts that lie more than 2^31 bytes apart each (packed words have no
    pitch: their rows only)."""
    p = Product(product, off, M, G, N, K, seed=3)
    size, e = p.dtype.itemsize, off // p.dtype.itemsize
    pitch = 2**31 // size + 16
    x = torch.empty((M - 1) * pitch + K + e, dtype=p.dtype, device=DEV)[e:].as_strided(
        (M, K), (pitch, 1))
    x.copy_(p.x)
    p.x = x
    if product in TYPES:
        far = 2**31 // size + N * K // 16 * 16
        w = torch.empty((G - 1) * far + N * K, dtype=p.dtype, device=DEV).as_strided(
            (G, N, K), (far, K, 1))
        w.copy_(p.w)
        p.w = w
    offsets = spans(M, G, 9)
    p.assert_choice(M, offsets, rows)
    p.check(p(on(offsets)), offsets)
