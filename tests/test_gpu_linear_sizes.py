"""Matrix products at the sizes that choose each kernel and tile, against float64
on the device.

The tolerance is that of the small products: n 2^-23 sum|terms| for a sum of n
terms in fp32, and half an ulp of the result's type (2^-8 relative for bf16, 2^-11
for f16, with half of its subnormal step). The int8 products' sums are exact.
"""

from __future__ import annotations

import pytest
import torch

from mlx_gptq import linear, packing
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


def close(got, want, mag, n, what):
    assert got.shape == want.shape, what
    d = (got.double() - want).abs()
    tol = (n + 8) * 2.0**-23 * mag + UNIT[got.dtype] * want.abs() * 1.01 + STEP[got.dtype]
    assert bool((d <= tol).all()), (what, float((d - tol).max()))


def counts_of(M, G, g):
    """M entries dealt unevenly to G groups, some of them empty."""
    p = torch.rand(G, generator=g) ** 3
    p[G // 3] = 0
    return torch.multinomial(p, M, replacement=True, generator=g).bincount(minlength=G).tolist()


def offsets_of(counts):
    return [0] + torch.tensor(counts).cumsum(0).tolist()


def randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


# entries, N, K, groups (0: one dense weight), gathered. The odd ones take the
# kernels whose rows are not 16 bytes apart.
SIZES = [
    (1, 1024, 2048, 0, False), (16, 512, 4096, 0, False), (24, 2048, 2048, 0, False),
    (48, 768, 1024, 0, True), (100, 4096, 512, 0, False), (256, 2048, 2048, 0, False),
    (700, 1000, 1024, 0, True), (2000, 2048, 520, 0, False), (4096, 4096, 264, 0, False),
    (3, 511, 2001, 0, False), (40, 2047, 1023, 0, True), (300, 1025, 1001, 0, False),
    (1500, 2047, 515, 0, True), (4000, 2049, 77, 0, False),
    (8, 1536, 1024, 64, True), (64, 768, 1024, 32, True), (512, 768, 1024, 32, True),
    (4096, 512, 1024, 60, True), (6000, 1408, 264, 8, False), (2048, 256, 128, 300, True),
    (64, 767, 1001, 32, True), (3000, 511, 999, 32, True), (5000, 1407, 129, 8, False),
    (256, 256, 1024, 0, False), (384, 512, 2048, 0, True), (384, 512, 4096, 0, False),
    (384, 512, 512, 0, False), (256, 255, 1023, 0, False), (128, 32767, 15, 8, False),
    (200, 32767, 17, 8, False), (8192, 128, 64, 256, False), (16384, 128, 64, 256, True),
    (16384, 64, 128, 256, False), (8192, 60, 100, 256, True), (384, 255, 1407, 0, False),
    (3000, 1536, 2048, 0, False), (6000, 2048, 1024, 0, True),
]


def case(M, N, K, G, gathered):
    cpu = torch.Generator().manual_seed(M + N + K + G)
    g = torch.Generator(DEV).manual_seed(M + 3 * N + 5 * K + G)
    off = offsets_of(counts_of(M, G, cpu)) if G else None
    T = max(M // 2, 1) if gathered else M
    idx = torch.randint(0, T, (M,), generator=cpu, dtype=torch.int32).to(DEV) if gathered else None
    return g, off, T, idx


def forward64(x, w, off, idx):
    xs = x.double() if idx is None else x.double()[idx.long()]
    if off is None:
        return xs @ w.double().T, xs.abs() @ w.double().abs().T
    y = torch.zeros(xs.shape[0], w.shape[1], dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(y)
    for g, (a, b) in enumerate(zip(off[:-1], off[1:])):
        y[a:b] = xs[a:b] @ w[g].double().T
        mag[a:b] = xs[a:b].abs() @ w[g].double().abs().T
    return y, mag


@pytest.mark.parametrize("M,N,K,G,gathered", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_forward(M, N, K, G, gathered, dtype):
    g, off, T, idx = case(M, N, K, G, gathered)
    x = randn(g, T, K, dtype=dtype)
    w = randn(g, *([G] if G else []), N, K, dtype=dtype, scale=0.1)
    y = linear.grouped_linear(x, w, off, idx)
    close(y, *forward64(x, w, off, idx), K, (M, N, K, G))


@pytest.mark.parametrize("M,N,K,G,gathered", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_dgrad(M, N, K, G, gathered, dtype):
    g, off, T, idx = case(M, N, K, G, gathered)
    dy = randn(g, M, N, dtype=dtype)
    w = randn(g, *([G] if G else []), N, K, dtype=dtype, scale=0.1)
    dx = linear.grouped_linear_dgrad(dy, w, off, idx, T)
    want, mag = forward64(dy, w.transpose(-1, -2).contiguous(), off, None)
    most = 1
    if idx is not None:
        most = int(idx.bincount().max())
        z = torch.zeros(T, K, dtype=torch.float64, device=DEV)
        want = z.index_add(0, idx.long(), want)
        mag = z.index_add(0, idx.long(), mag)
    close(dx, want, mag, N + most, (M, N, K, G))


@pytest.mark.parametrize("M,N,K,G,gathered", SIZES)
@pytest.mark.parametrize("dtype,out", [(torch.bfloat16, None), (torch.bfloat16, torch.float32),
                                       (torch.float16, None)])
def test_wgrad(M, N, K, G, gathered, dtype, out):
    g, off, T, idx = case(M, N, K, G, gathered)
    dy, x = randn(g, M, N, dtype=dtype, scale=0.1), randn(g, T, K, dtype=dtype)
    dw = linear.grouped_linear_wgrad(dy, x, off, idx, out_dtype=out)
    xs = x.double() if idx is None else x.double()[idx.long()]
    spans = [(0, M)] if off is None else list(zip(off[:-1], off[1:]))
    for i, (a, b) in enumerate(spans):
        d = dy[a:b].double().T.contiguous()
        close(dw if off is None else dw[i], d @ xs[a:b], d.abs() @ xs[a:b].abs(), b - a,
              (M, N, K, G, i))


@pytest.mark.parametrize("M,N,K,G,gathered", SIZES)
def test_int8(M, N, K, G, gathered):
    g, off, T, idx = case(M, N, K, G, gathered)
    gs = [G] if G else []
    q = torch.randint(-127, 128, (T, K), generator=g, dtype=torch.int8, device=DEV)
    w = torch.randint(-128, 128, (*gs, N, K), generator=g, dtype=torch.int8, device=DEV)
    s = torch.rand(T, generator=g, device=DEV) * 0.1 + 1e-3
    ws = torch.rand(*gs, N, generator=g, device=DEV) * 1e-2
    b = torch.randn(*gs, N, generator=g, device=DEV)
    y = linear.int8_linear(q, s, w, ws, b, torch.float32, off, idx)
    total = forward64(q, w, off, idx)[0]
    sx = (s if idx is None else s[idx.long()]).double()
    if off is None:
        scale, bias = ws.double().expand(M, N), b.double().expand(M, N)
    else:
        group = torch.arange(G, device=DEV).repeat_interleave(
            torch.tensor(off, device=DEV).diff())
        scale, bias = ws.double()[group], b.double()[group]
    prod = total * sx[:, None] * scale
    d = (y.double() - prod - bias).abs()
    assert bool((d <= 5 * 2.0**-24 * (prod.abs() + bias.abs())).all()), float(d.max())


@pytest.mark.parametrize("M,N,K,G,gathered", [s for s in SIZES if s[2] >= 512 or s[2] % 32 == 0])
@pytest.mark.parametrize("mode", ["mxfp4", "mxfp8"])
def test_mxfp(M, N, K, G, gathered, mode):
    K = K // 32 * 32
    g, off, T, idx = case(M, N, K, G, gathered)
    gs = [G] if G else []
    bits = 4 if mode == "mxfp4" else 8
    x = randn(g, T, K)
    codes = torch.randint(0, 1 << bits, (*gs, N, K), generator=g, dtype=torch.uint8, device=DEV)
    if bits == 8:
        codes = torch.where((codes & 127) == 127, 5, codes)  # no NaN codes
    scales = torch.randint(115, 131, (*gs, N, K // 32), generator=g, dtype=torch.uint8, device=DEV)
    y = linear.mxfp_linear(x, packing.pack_q(codes, bits), scales, mode, off, idx)
    w = ref.decode(codes.cpu(), scales.cpu(), mode).to(DEV)
    close(y, *forward64(x, w, off, idx), K, (M, N, K, G, mode))


@pytest.mark.parametrize("offsets", [[0, 300, 100, 400], [400, 300, 200, 0], [0, 400, 0, 400],
                                     [-7, 5000, -7, 10]])
def test_groups_that_overlap_stay_inside_the_list(offsets):
    """Unvalidated offsets that decrease: every call ends, and a weight gradient is
    the sum over what each group names."""
    g = torch.Generator(DEV).manual_seed(5)
    M, N, K = 400, 130, 264
    x, dy, w = randn(g, M, K), randn(g, M, N, scale=0.1), randn(g, 3, N, K, scale=0.1)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    assert linear.grouped_linear(x, w, off, validate=False).shape == (M, N)
    assert linear.grouped_linear_dgrad(dy, w, off, validate=False).shape == (M, K)
    dw = linear.grouped_linear_wgrad(dy, x, off, validate=False)
    at = [min(max(o, 0), M) for o in offsets]
    for i in range(3):
        a, b = at[i], max(at[i], at[i + 1])
        d = dy[a:b].double().T.contiguous()
        close(dw[i], d @ x[a:b].double(), d.abs() @ x[a:b].double().abs(), M, offsets)


def test_many_overlapping_groups():
    """Long groups that overlap add up to more than a list's worth of entries."""
    g = torch.Generator(DEV).manual_seed(6)
    M, N, K, G = 3000, 16, 24, 200
    x, dy = randn(g, M, K), randn(g, M, N, scale=0.1)
    off = torch.tensor([0, M] * (G // 2) + [0], dtype=torch.int32, device=DEV)
    dw = linear.grouped_linear_wgrad(dy, x, off, validate=False)
    d = dy.double().T.contiguous()
    for i in range(G):
        if i % 2:
            assert not bool(dw[i].any())
        else:
            close(dw[i], d @ x.double(), d.abs() @ x.double().abs(), M, i)


@pytest.mark.parametrize("off", [None, [0, 0, 0]])
def test_no_entries(off):
    gs = [] if off is None else [2]
    x, w = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), torch.ones(
        *gs, 40, 64, dtype=torch.bfloat16, device=DEV)
    dy = torch.empty(0, 40, dtype=torch.bfloat16, device=DEV)
    assert linear.grouped_linear(x, w, off).shape == (0, 40)
    assert linear.grouped_linear_dgrad(dy, w, off).shape == (0, 64)
    dw = linear.grouped_linear_wgrad(dy, x, off)
    assert dw.shape == (*gs, 40, 64) and not bool(dw.any())
    q, s = linear.quantize_rows_int8(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    y = linear.int8_linear(q, s, w.to(torch.int8), torch.ones(*gs, 40, device=DEV), offsets=off)
    assert y.shape == (0, 40)


@pytest.mark.parametrize("mode", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("M,N,K,G", [(3, 129, 544, 0), (70, 1000, 96, 0), (900, 515, 1056, 0),
                                     (3000, 1030, 288, 0), (500, 260, 160, 9)])
def test_mxfp_rows_and_words_off_every_boundary(M, N, K, G, mode):
    """Rows that start two bytes past a boundary, words that start four past one."""
    g, off, _, _ = case(M, N, K, G, False)
    gs = [G] if G else []
    bits = 4 if mode == "mxfp4" else 8
    x = randn(g, M, K + 3)[:, 1 : K + 1]
    codes = torch.randint(0, 127, (*gs, N, K), generator=g, dtype=torch.uint8, device=DEV) % (1 << bits)
    packed = packing.pack_q(codes, bits)
    words = torch.empty(packed.numel() + 1, dtype=packed.dtype, device=DEV)[1:].view(packed.shape)
    words.copy_(packed)
    flat = torch.randint(115, 131, (codes.numel() // 32 + 1,), generator=g, dtype=torch.uint8,
                         device=DEV)
    scales = flat[1:].view(*gs, N, K // 32)
    y = linear.mxfp_linear(x, words, scales, mode, off)
    w = ref.decode(codes.cpu(), scales.cpu(), mode).to(DEV)
    close(y, *forward64(x, w, off, None), K, (M, N, K, G, mode))
