"""Products with affine weights against float64.

Tolerance. A result is the sum over blocks of 32 of scale * sum(x q) + bias * sum(x), in
fp32: with m the sum of |x| (|q scale| + |bias|), every term passes through at most 32
additions of its block, two fused multiply-adds of each of the K / 32 blocks and the
additions of eight partial sums, each within 2^-23 of its operands' magnitudes (twice
2^-24, which also covers truncating adders): (K / 16 + 48) 2^-23 m, less than the bound
(K + 48) 2^-23 m used here. Rounding to the rows' type adds half a step: 2^-8 relative
for bf16, 2^-11 for f16 with half of its subnormal step, 2^-25. The tile kernel (many
rows) rounds q scale + bias to the rows' type before it multiplies, half a step of every
weight: UNIT sum|x| |q scale + bias| more, which `mag` is at least as large as.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from mlx_gptq import _native as nat
from mlx_gptq import gptq, grid, linear, packing
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25}


def weight(G, N, K, bits, group, params, seed=0):
    """(codes uint8 [G, N, K], scales, biases) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 2**bits, (G, N, K), generator=g, dtype=torch.uint8)
    s = (torch.rand(G, N, K // group, generator=g) + 0.3) * (2.0 / 2**bits) * K**-0.5
    b = -s * 2.0 ** (bits - 1) * (1 + 0.3 * torch.randn(G, N, K // group, generator=g))
    return q, s.to(TYPES[params]), b.to(TYPES[params])


def rows(T, K, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, K, generator=g).to(TYPES[dtype])


def close(got, want, mag, K, what=None, rounded=None):
    """rounded: sum|x| |w| where the kernel rounds the weights."""
    d = (got.cpu().double() - want).abs()
    tol = (K + 48) * 2.0**-23 * mag + UNIT[got.dtype] * want.abs() * 1.01 + STEP[got.dtype]
    if rounded is not None:
        tol = tol + 1.01 * UNIT[got.dtype] * rounded + STEP[got.dtype] * K * 8
    bad = ~(d <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((d - tol).max()),
                                 torch.nonzero(bad)[:4].tolist())


def product(x, q, s, b, bits, offsets=None, row_index=None, **kw):
    if offsets is None:
        q, s, b = q[0], s[0], b[0]
    words = packing.pack_q(q.to(DEV), bits)
    idx = None if row_index is None else row_index.to(DEV)
    return linear.affine_linear(x.to(DEV), words, s.to(DEV), b.to(DEV), bits, offsets, idx, **kw)


SINGLE, FEW, TILE, STAGED = range(4)


def kernel(x, words, bits, G, N, offsets, M=None):
    """mgq_affine_choice of a call on these device tensors."""
    out = (ctypes.c_int32 * 3)()
    nat.call("mgq_affine_choice", x.data_ptr(), x.stride(0) if x.shape[0] > 1 else x.shape[1],
             x.shape[0] if M is None else M, words.data_ptr(), bits, G, N, x.shape[1],
             int(offsets is not None), ctypes.addressof(out))
    return tuple(out)


def check(x, q, s, b, bits, offsets=None, row_index=None, what=None, words=None):
    """The product of these (x may be on the device) against float64; which kernel it took."""
    G, N, K = q.shape
    x = x.to(DEV)
    if words is None:
        words = packing.pack_q((q if offsets is not None else q[0]).to(DEV), bits)
    pick = (lambda t: t.to(DEV)) if offsets is not None else (lambda t: t[0].to(DEV))
    idx = None if row_index is None else row_index.to(DEV)
    y = linear.affine_linear(x, words, pick(s), pick(b), bits, offsets, idx)
    took = kernel(x, words, bits, G, N, offsets, y.shape[0])
    host = x.cpu()
    want, mag = ref.affine_forward(host, q, s, b, offsets, row_index)
    rounded = None
    if took[0] >= TILE:
        rounded = ref.forward(host, ref.affine(q, s, b)[0], offsets, row_index)[1]
    close(y, want, mag, K, what, rounded)
    return y, took


FORMS = [(bits, group, dtype, params) for bits in (2, 4, 8) for group in (32, 64, 128)
         for dtype in ("bf16", "f16") for params in ("bf16", "f16", "f32")]


@pytest.mark.parametrize("bits,group,dtype,params", FORMS)
def test_every_form(bits, group, dtype, params):
    """Every code, group size and type, in each kernel for few rows and in a tile."""
    N, K = 40, 3 * group + (128 if group < 128 else 0)
    q, s, b = weight(1, N, K, bits, group, params)
    for T in (1, 3, 5, 16, 30, 70, 300):
        check(rows(T, K, dtype), q, s, b, bits, what=T)


@pytest.mark.parametrize("bits", [2, 4, 8])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_codes_stand_in_their_places(bits, dtype):
    """Rows with a single one pick out single weights: every code of every place of a
    step. One product q s + b in fp32, so that a code off by one cannot hide."""
    K = 256
    q = torch.randint(0, 2**bits, (1, 19, K), generator=torch.Generator().manual_seed(4),
                      dtype=torch.uint8)
    q[0, 0] = (torch.arange(K) % 2**bits).to(torch.uint8)
    s, b = torch.ones(1, 19, K // 32), torch.zeros(1, 19, K // 32)
    x = torch.eye(K).to(TYPES[dtype])
    for T in (1, 4, 16, K):  # (whole numbers: the tile's rounding keeps them too)
        y = product(x[K - T:], q, s, b, bits)
        assert torch.equal(y.cpu().double(), q[0].double().T[K - T:])


SIZES = [(1, 1, 32), (1, 17, 32), (2, 16, 96), (4, 33, 1056), (5, 130, 160), (16, 257, 4096),
         (17, 48, 288), (33, 100, 544), (64, 1001, 736), (65, 64, 64), (129, 260, 416),
         (513, 300, 1120), (1, 50, 14336)]


@pytest.mark.parametrize("T,N,K", SIZES)
@pytest.mark.parametrize("bits", [4, 8])
def test_sizes(T, N, K, bits):
    q, s, b = weight(1, N, K, bits, 32, "bf16", seed=T)
    check(rows(T, K, "bf16"), q, s, b, bits)


# groups' counts, rows of x (0: not gathered), entries of no group in front and behind
LISTS = {
    "token": ([1, 1, 1, 1], 1, 0, 0),
    "few": ([3, 0, 1, 7, 0, 2, 16, 17], 11, 0, 0),
    "nothing": ([0, 0, 0], 9, 0, 0),
    "no_group": ([20, 0, 30], 25, 6, 9),
    "ragged": ([130, 1, 0, 64, 300], 0, 0, 3),
    "many": ([i % 4 for i in range(300)], 50, 0, 0),
    "large": ([700, 0, 300, 513], 400, 0, 0),
}


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("bits,group,dtype", [(4, 64, "bf16"), (8, 32, "f16"), (2, 128, "bf16")])
def test_groups(name, bits, group, dtype):
    counts, gathered, before, after = LISTS[name]
    G, N, K = len(counts), 72, 256
    M = before + sum(counts) + after
    T = gathered or M
    q, s, b = weight(G, N, K, bits, group, dtype, seed=7)
    x = rows(T, K, dtype)
    off = [before]
    for c in counts:
        off.append(off[-1] + c)
    idx = None
    if gathered:
        idx = torch.randint(0, T, (M,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    y, _ = check(x, q, s, b, bits, off, idx, name)
    if before:
        assert not bool(y[:before].any()) and not bool(y[off[-1]:].any())


@pytest.mark.parametrize("T", [2, 20, 200])
def test_strides_and_alignment(T):
    """Rows of a wider matrix that start at any element, words off 16-byte boundaries."""
    N, K, bits = 50, 192, 4
    q, s, b = weight(1, N, K, bits, 64, "bf16")
    wide = rows(T, K + 13, "bf16").to(DEV)
    flat = torch.empty(N * K // 8 + 1, dtype=torch.int32, device=DEV)
    words = flat[1:].view(N, K // 8)
    words.copy_(packing.pack_q(q[0].to(DEV), bits).view(torch.int32))
    for start in (0, 1, 5, 8):
        x = wide[:, start:start + K]
        check(x, q, s, b, bits, what=start, words=words)
    # scales and biases that are views, words given as uint32
    sb = torch.stack((s[0], b[0]), dim=-1).to(DEV)
    y = linear.affine_linear(x, words.view(torch.uint32), sb[..., 0], sb[..., 1], bits)
    assert torch.equal(y, linear.affine_linear(x, words, s[0].to(DEV), b[0].to(DEV), bits))


@pytest.mark.parametrize("T", [3, 40, 200])
def test_a_bias_far_from_its_scale(T):
    """Weights 100 +- 8 steps: the terms cancel in neither order of the sum."""
    q, s, b = weight(1, 33, 512, 4, 64, "f32")
    b = torch.full_like(b, 100.0)
    check(rows(T, 512, "bf16"), q, s, b, 4)


@pytest.mark.parametrize("T", [1, 20, 150])
def test_a_row_that_is_no_number_stays_alone(T):
    q, s, b = weight(1, 20, 96, 4, 32, "bf16")
    x = rows(T, 96, "bf16")
    x[T // 2, 7] = torch.nan
    y = product(x, q, s, b, 4).cpu()
    assert bool(y[T // 2].isnan().all())
    clean = x.clone()
    clean[T // 2] = 0
    keep = [t for t in range(T) if t != T // 2]
    assert torch.equal(y[keep], check(clean, q, s, b, 4)[0].cpu()[keep])
    s[0, 3, 1] = torch.nan  # and so does a weight row
    y = product(rows(T, 96, "bf16"), q, s, b, 4)
    assert y.isnan().all(dim=0).nonzero().flatten().tolist() == [3]


def test_the_solvers_results():
    """Round to nearest and GPTQ in the affine grid: their product with the packed codes
    is the product with what they call their dequantized weight."""
    g = torch.Generator().manual_seed(0)
    W = (torch.randn(2, 48, 128, generator=g) * 0.05).to(torch.bfloat16).to(DEV)
    x = torch.randn(9, 128, generator=g).to(torch.bfloat16).to(DEV)
    H = torch.eye(128, device=DEV).repeat(2, 1, 1)
    off = [0, 4, 9]
    for q, s, b, dq in (grid.rtn_quantize(W, 4, 64), gptq.solve_gptq(W, H, 4, 64, mode="affine")[:4]):
        y = linear.affine_linear(x, packing.pack_q(q, 4), s, b, 4, off)
        _, mag = ref.affine_forward(x.cpu(), q.cpu(), s.cpu(), b.cpu(), off)
        want, m = ref.forward(x.cpu(), dq.cpu(), off)
        # (dq itself is rounded to fp32 twice)
        close(y, want, mag + m, 128)


def test_host_tensors_and_gradients():
    q, s, b = weight(1, 20, 64, 4, 32, "bf16")
    x = rows(3, 64, "bf16")
    y = linear.affine_linear(x, packing.pack_q(q[0], 4), s[0], b[0], 4)
    assert y.device.type == "cpu"
    close(y, *ref.affine_forward(x, q, s, b), 64)
    leaf = x.to(DEV).requires_grad_()
    y = product(leaf, q, s, b, 4)
    with pytest.raises(NotImplementedError, match="affine_linear"):
        y.sum().backward()


@pytest.mark.parametrize("T", [1, 24, 300])
def test_captured_and_replayed(T):
    """New rows in the same buffers, through a graph on another stream."""
    q, s, b = weight(4, 64, 128, 4, 64, "bf16")
    words = packing.pack_q(q.to(DEV), 4)
    s_d, b_d = s.to(DEV), b.to(DEV)
    x = rows(T, 128, "bf16").to(DEV)
    off = torch.tensor([0, T // 3, T // 2, T // 2, T], dtype=torch.int32, device=DEV)
    call = lambda: linear.affine_linear(x, words, s_d, b_d, 4, off, validate=False)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call()
    for seed in (5, 6, 7):
        x.copy_(rows(T, 128, "bf16", seed))
        off.copy_(torch.tensor([0, seed % (T + 1), T, T, T], dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, call())


def test_offsets_out_of_range_are_clamped():
    q, s, b = weight(2, 24, 64, 4, 32, "bf16")
    x = rows(6, 64, "bf16")
    off = torch.tensor([-5, 3, 1000], dtype=torch.int32, device=DEV)
    idx = torch.tensor([0, 7, -2, 3, 5, 100], dtype=torch.int32)
    y = product(x, q, s, b, 4, off, idx, validate=False)
    close(y, *ref.affine_forward(x, q, s, b, [0, 3, 6], idx.clamp(0, 5)), 64)


# a call that reaches each form (M, N, K, G, bits, bytes that the rows are off 16)
REACHED = {
    (SINGLE, 0, 0): (1, 4096, 736, 0, 4, 0), (FEW, 1, 0): (32, 100, 32, 32, 4, 2),
    (FEW, 2, 0): (1, 16, 32, 0, 4, 2), (FEW, 3, 0): (600, 40, 512, 16, 2, 0),
    (FEW, 4, 0): (8, 6000, 512, 2, 4, 0), (FEW, 5, 0): (200, 40, 32, 0, 2, 0),
    (FEW, 6, 0): (600, 40, 32, 16, 8, 0), (FEW, 7, 0): (600, 40, 160, 16, 2, 2),
    (FEW, 8, 0): (200, 257, 512, 32, 4, 2), (FEW, 9, 0): (600, 257, 512, 32, 2, 2),
    (FEW, 10, 0): (300, 1001, 512, 16, 4, 2), (FEW, 11, 0): (40, 4096, 32, 16, 4, 2),
    (TILE, 64, 128): (300, 6000, 1024, 0, 8, 0), (TILE, 64, 256): (300, 6000, 32, 8, 8, 0),
    (TILE, 128, 256): (128, 6000, 32, 16, 4, 0), (TILE, 256, 256): (200, 6000, 32, 16, 8, 0),
    (STAGED, 64, 256): (300, 6000, 32, 8, 8, 2), (STAGED, 128, 256): (600, 4096, 32, 16, 8, 2),
}


@pytest.mark.parametrize("form", sorted(REACHED))
@pytest.mark.parametrize("dtype,params", [("bf16", "bf16"), ("f16", "f32")])
def test_every_kernel_is_reached(form, dtype, params):
    M, N, K, G, bits, off16 = REACHED[form]
    q, s, b = weight(max(G, 1), N, K, bits, 32, params, seed=M)
    store = torch.zeros(M * K + 8, dtype=TYPES[dtype], device=DEV)
    x = store[off16 // 2:off16 // 2 + M * K].view(M, K)
    x.copy_(rows(M, K, dtype))
    off = None
    if G:  # uneven groups, the third one empty where there is one
        cuts = torch.randint(0, M + 1, (G - 1,), generator=torch.Generator().manual_seed(2)).sort().values
        off = [0, *cuts.tolist(), M]
        if G > 3:
            off[3] = off[2]
    _, took = check(x, q, s, b, bits, off)
    assert took == form


@pytest.mark.parametrize("M", [1, 20, 300])
def test_far_rows_and_weights(M):
    """Rows, weights, scales and results whose places pass 2^32 bytes."""
    G, N, K, tail = 3, 1 << 20, 4096, 40
    T = (1 << 19) + 70000  # rows of 8 KiB
    g = torch.Generator().manual_seed(M)
    words = torch.zeros(G, N, K // 8, dtype=torch.int32, device=DEV)
    s = torch.zeros(G, N, K // 32, dtype=torch.float32, device=DEV)
    b = torch.zeros(G, N, K // 32, dtype=torch.float32, device=DEV)
    q, sl, bl = weight(1, tail, K, 4, 32, "f32")
    words[2, -tail:] = packing.pack_q(q[0].to(DEV), 4).view(torch.int32)
    s[2, -tail:], b[2, -tail:] = sl[0].to(DEV), bl[0].to(DEV)
    x = torch.zeros(T, K, dtype=torch.bfloat16, device=DEV)
    used = torch.randint(T - 60000, T, (M,), generator=g)
    used[-1] = T - 1
    x[used.to(DEV)] = rows(M, K, "bf16").to(DEV)
    idx = used.to(torch.int32).to(DEV)
    off = torch.tensor([0, 0, 0, M], dtype=torch.int32, device=DEV)
    y = linear.affine_linear(x, words, s, b, 4, off, idx)
    took = kernel(x, words, 4, G, N, off, M)
    few = x[used.to(DEV)].cpu()
    want, mag = ref.affine_forward(few, q, sl, bl)
    rounded = ref.forward(few, ref.affine(q, sl, bl)[0])[1] if took[0] >= TILE else None
    close(y[:, -tail:], want, mag, K, took, rounded)
    assert not bool(y[:, :-tail].any())


def test_the_choice_refuses_what_the_product_refuses():
    out = (ctypes.c_int32 * 3)()
    for args in ((3, 1, 16, 64), (4, 2, 16, 64), (4, 1, 1 << 31, 64), (4, 1, 16, 0)):
        bits, G, N, K = args
        with pytest.raises((ValueError, AssertionError)):
            nat.call("mgq_affine_choice", 16, 64, 4, 16, bits, G, N, K, 0, ctypes.addressof(out))
