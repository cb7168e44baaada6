"""Matrix products with dense, MXFP and int8 weights against float64.

Tolerances. A result is a sum of n products accumulated in fp32 in some order
and rounded once: it is within n 2^-23 sum|terms| (twice the bound of any order
of additions in round-to-nearest, which also covers truncating adders) plus half
an ulp of its type, 2^-8 relative for bf16 and 2^-11 for f16, plus half of f16's
subnormal step 2^-24.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from mlx_gptq import linear, packing
from oracle import linear_ref as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
STEP = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def close(got, want, mag, n, what):
    """got against want within the derived bound."""
    d = (got.cpu().double() - want).abs()
    tol = (n + 8) * 2.0**-23 * mag + UNIT[got.dtype] * want.abs() * 1.01 + STEP[got.dtype]
    bad = ~(d <= tol)
    assert not bool(bad.any()), (what, int(bad.sum()), float((d - tol).max()),
                                 torch.nonzero(bad)[:4].tolist())


def offsets_of(counts, start=0):
    return [start] + (start + np.cumsum(counts)).tolist()


# name: groups' counts, N, K, rows of x when gathered (0: no gather), entries
# before the first group, entries after the last
LISTS = {
    "one_token": ([1], 64, 64, 0, 0, 0),
    "one_of_everything": ([1], 1, 1, 0, 0, 0),
    "token_of_eight": ([1] * 8, 96, 160, 1, 0, 0),
    "few_each": ([3, 0, 1, 7, 0, 2, 16, 17], 257, 512, 11, 0, 0),
    "empty_ends": ([0, 0, 5, 40, 0], 130, 96, 0, 0, 0),
    "nothing": ([0, 0, 0], 40, 64, 9, 0, 0),
    "odd": ([33, 130, 0, 1, 64], 131, 77, 0, 0, 0),
    "odd_gather": ([33, 130, 0, 1, 64], 97, 251, 60, 0, 0),
    "no_group": ([20, 0, 30], 64, 128, 25, 6, 9),
    "tile_edges": ([128, 129, 127, 256, 1], 256, 320, 0, 0, 0),
    "long_rows": ([5, 70], 48, 4104, 0, 0, 0),
    "many_groups": ([i % 4 for i in range(300)], 40, 64, 50, 0, 0),
    "big": ([700, 0, 300, 513], 520, 776, 400, 0, 0),
    "wide": ([600], 1100, 264, 0, 0, 0),
    # groups long enough to be cut along their entries, few and many of them
    "heavy": ([3000, 10, 0, 1500], 136, 328, 700, 0, 0),
    "heavy_of_many": ([2500] + [i % 3 for i in range(70)] + [4100, 64, 65], 72, 264, 0, 3, 0),
    "mid": ([90, 0, 150, 111, 64], 320, 200, 300, 0, 0),
    "deep": ([300, 260, 1], 264, 1160, 0, 0, 5),
}


def make_list(name, dtype, seed=0):
    counts, N, K, gathered, before, after = LISTS[name]
    g = gen(sum(map(ord, name)) + seed)
    M = before + sum(counts) + after
    T = gathered or M
    x = randn(g, T, K, dtype=dtype)
    w = randn(g, len(counts), N, K, dtype=dtype, scale=0.1)
    idx = torch.randint(0, T, (M,), generator=g, dtype=torch.int32) if gathered else None
    dy = randn(g, M, N, dtype=dtype)
    return x, w, offsets_of(counts, before), idx, dy


def dev(t):
    return None if t is None else t.to(DEV)


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_forward(name, dt):
    x, w, off, idx, _ = make_list(name, HALF[dt])
    y = linear.grouped_linear(dev(x), dev(w), off, dev(idx))
    want, mag = ref.forward(x, w, off, idx)
    assert y.dtype == x.dtype and tuple(y.shape) == tuple(want.shape)
    close(y, want, mag, x.shape[1], name)


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_gradients(name, dt):
    x, w, off, idx, dy = make_list(name, HALF[dt], seed=1)
    dx = linear.grouped_linear_dgrad(dev(dy), dev(w), off, dev(idx), x.shape[0])
    want, mag = ref.dgrad(dy, w, off, idx, x.shape[0])
    reads = 1 if idx is None or not idx.numel() else int(torch.bincount(idx).max())
    assert tuple(dx.shape) == tuple(x.shape)
    close(dx, want, mag, w.shape[1] + reads, name)
    for out in (None, torch.float32):
        dw = linear.grouped_linear_wgrad(dev(dy), dev(x), off, dev(idx), out_dtype=out)
        want, mag = ref.wgrad(dy, x, off, idx)
        assert tuple(dw.shape) == tuple(w.shape)
        close(dw, want, mag, max(int(np.diff(off).max()), 1), name)


def test_gradient_is_the_functions_derivative():
    """Central differences of sum(c * y) in float64 against the gradients, along
    random directions; y is linear in x and in w, so the difference is exact up
    to float64 rounding and only the gradients' own rounding remains."""
    x, w, off, idx, c = make_list("few_each", torch.float16, seed=2)
    xg, wg = dev(x).requires_grad_(), dev(w).requires_grad_()
    y = linear.grouped_linear(xg, wg, off, dev(idx))
    y.backward(dev(c))
    for grad, which in ((xg.grad, 0), (wg.grad, 1)):
        base = [x.double(), w.double()]
        direction = torch.randn(base[which].shape, generator=gen(5), dtype=torch.float64)
        vals = []
        for h in (1e-3, -1e-3):
            moved = [b.clone() for b in base]
            moved[which] += h * direction
            vals.append(float((c.double() * ref.forward(moved[0], moved[1], off, idx)[0]).sum()))
        numeric = (vals[0] - vals[1]) / 2e-3
        analytic = float((grad.cpu().double() * direction).sum())
        # each gradient entry is within 2^-11 relative (half an ulp of f16) and
        # its fp32 sum within the bound of `close`
        gm = grad.cpu().double().abs()
        if which == 0:
            _, mag = ref.dgrad(c, w, off, idx, x.shape[0])
        else:
            _, mag = ref.wgrad(c, x, off, idx)
        tol = float(((2.0**-11 * gm + 600 * 2.0**-23 * mag + 2.0**-25) * direction.abs()).sum())
        assert abs(numeric - analytic) <= tol + 1e-6 * abs(numeric), (which, numeric, analytic, tol)


def test_autograd_gives_the_explicit_gradients():
    x, w, off, idx, dy = make_list("big", torch.bfloat16, seed=3)
    xg, wg = dev(x).requires_grad_(), dev(w).requires_grad_()
    y = linear.grouped_linear(xg, wg, torch.tensor(off, device=DEV), dev(idx), validate=False)
    y.backward(dev(dy))
    assert torch.equal(xg.grad, linear.grouped_linear_dgrad(dev(dy), dev(w), off, dev(idx), len(x)))
    assert torch.equal(wg.grad, linear.grouped_linear_wgrad(dev(dy), dev(x), off, dev(idx)))
    # only one of the two
    xg2 = dev(x).requires_grad_()
    linear.grouped_linear(xg2, dev(w), off, dev(idx)).backward(dev(dy))
    assert torch.equal(xg2.grad, xg.grad)


def test_a_row_read_by_many_entries_sums_in_order():
    """One row read by every entry (more than the slots of a row), and rows read
    by 0, 1, 15, 16 and 17 entries; the same bits on every call."""
    g = gen(9)
    counts = [0, 1, 15, 16, 17, 300]
    idx = torch.repeat_interleave(torch.arange(6), torch.tensor(counts))
    idx = idx[torch.randperm(len(idx), generator=g)].to(torch.int32)
    w = randn(g, 1, 72, 1100, dtype=torch.bfloat16, scale=0.1)
    dy = randn(g, len(idx), 72, dtype=torch.bfloat16)
    off = [0, len(idx)]
    want, mag = ref.dgrad(dy, w, off, idx, 6)
    first = linear.grouped_linear_dgrad(dev(dy), dev(w), off, dev(idx), 6)
    close(first, want, mag, 72 + 300, "many reads")
    for _ in range(3):
        assert torch.equal(first, linear.grouped_linear_dgrad(dev(dy), dev(w), off, dev(idx), 6))


MX_LISTS = ["one_token", "token_of_eight", "empty_ends", "nothing", "no_group", "tile_edges",
            "few_each", "many_groups", "big", "mid", "deep"]


def mx_case(name, mode, K=None):
    counts, N, K0, gathered, before, after = LISTS[name]
    K = K or K0
    g = gen(sum(map(ord, name)) + 77)
    M = before + sum(counts) + after
    T = gathered or M
    x = randn(g, T, K, dtype=torch.bfloat16)
    codes = torch.randint(0, 16 if mode == "mxfp4" else 256, (len(counts), N, K), generator=g)
    if mode == "mxfp8":
        codes = torch.where((codes & 127) == 127, 5, codes)  # no NaN codes
    scales = torch.randint(115, 131, (len(counts), N, K // 32), generator=g).to(torch.uint8)
    idx = torch.randint(0, T, (M,), generator=g, dtype=torch.int32) if gathered else None
    return x, codes.to(torch.uint8), scales, offsets_of(counts, before), idx


@pytest.mark.parametrize("name", MX_LISTS)
@pytest.mark.parametrize("mode", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("K", [None, 32, 352])
def test_mxfp(name, mode, K):
    if K is None and LISTS[name][2] % 32:
        K = LISTS[name][2] // 32 * 32
    x, q, s, off, idx = mx_case(name, mode, K)
    packed = packing.pack_q(q.to(DEV), 4 if mode == "mxfp4" else 8)
    y = linear.mxfp_linear(dev(x), packed, dev(s), mode, off, dev(idx))
    want, mag = ref.forward(x, ref.decode(q, s, mode), off, idx)
    close(y, want, mag, x.shape[1], name)


@pytest.mark.parametrize("mode", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("rows", [1, 200])
def test_mxfp_dense_every_code_and_scale(mode, rows):
    """Every code at every scale byte from 1 to 246 (448 stays finite), each alone in its sum: the
    product with a one-hot row is the decoded weight itself."""
    n = 16 if mode == "mxfp4" else 256
    codes = torch.arange(n, dtype=torch.uint8)
    if mode == "mxfp8":
        codes = codes[(codes.long() & 127) != 127]
    s = torch.arange(1, 247, dtype=torch.uint8)
    K = 32 * ((len(codes) + 31) // 32)
    q = torch.zeros(len(s), K, dtype=torch.uint8)
    q[:, : len(codes)] = codes
    sc = s[:, None].expand(len(s), K // 32).contiguous()
    x = torch.zeros(rows, K, dtype=torch.bfloat16)
    want = ref.decode(q, sc, mode)  # [246, K]
    packed = packing.pack_q(q.to(DEV), 4 if mode == "mxfp4" else 8)
    for k0 in range(0, len(codes), rows):
        x.zero_()
        for i in range(min(rows, len(codes) - k0)):
            x[i, k0 + i] = 1.0
        y = linear.mxfp_linear(dev(x), packed, dev(sc), mode).cpu().double()
        for i in range(min(rows, len(codes) - k0)):
            w = want[:, k0 + i].to(torch.bfloat16).double()  # exact above 2^-133
            big = want[:, k0 + i].abs() >= 2.0**-126
            assert torch.equal(y[i][big], w[big])
        if rows == 1 and k0 >= 40:
            break


def test_mxfp_equals_the_solvers_dequantized_weights():
    """The codes of the framework's own round-to-nearest, packed, against the
    dense product with its dequantized weights (exact in bf16): the same bits
    in both operators' sums are not promised, the bound of the sums is."""
    from mlx_gptq import grid

    g = gen(21)
    W = randn(g, 3, 160, 256, dtype=torch.bfloat16, scale=0.02)
    x = randn(g, 50, 256, dtype=torch.bfloat16)
    off = [0, 20, 20, 50]
    for mode, bits in (("mxfp4", 4), ("mxfp8", 8)):
        q, s, _, dq = grid.rtn_quantize_mxfp(dev(W), mode)
        assert torch.equal(dq.to(torch.bfloat16).float(), dq)
        y = linear.mxfp_linear(dev(x), packing.pack_q(q, bits), s, mode, off)
        want, mag = ref.forward(x, dq.cpu(), off)
        close(y, want, mag, 256, mode)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (7, 33), (300, 1000), (5, 5121), (3, 20000)])
def test_quantize_rows(shape, dt):
    x = randn(gen(shape[1]), *shape, dtype=dt)
    x[0] = x[0] * 3
    if shape[0] > 2:
        x[1] = 0
    q, s = linear.quantize_rows_int8(dev(x))
    wq, ws = ref.quantize_rows(x)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), wq)


def test_quantize_rows_extremes():
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[1.0, -2.0, 0.5, 0.0], [float("nan"), 1, 2, 3], [float("inf"), 1, 2, 3],
                      [-float("inf"), float("nan"), 0, 0], [0, -0.0, 0, 0], [big, -big, 1, 0],
                      [1e-45, 0, -1e-45, 0], [1e-38, 2e-38, -3e-39, 1e-40],
                      [127.0, 0.5, 1.5, -2.5]])
    q, s = linear.quantize_rows_int8(dev(x))
    wq, ws = ref.quantize_rows(x)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(ws))
    ok = ~torch.isnan(ws)
    assert torch.equal(s.cpu()[ok], ws[ok]) and torch.equal(q.cpu(), wq.clamp(-127, 127))
    assert q.cpu()[8].tolist() == [127, 0, 2, -2]  # ties to even


def test_quantize_rows_strides_and_leading_dims():
    x = randn(gen(3), 4, 6, 50, dtype=torch.bfloat16)
    q, s = linear.quantize_rows_int8(dev(x))
    wq, ws = ref.quantize_rows(x)
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    wide = dev(randn(gen(4), 40, 90, dtype=torch.float16))
    for v in (wide[:, 3:72], wide.t(), wide[::2, :64], wide[:, ::3]):
        q, s = linear.quantize_rows_int8(v)
        wq, ws = ref.quantize_rows(v.cpu())
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    q, s = linear.quantize_rows_int8(wide[:0])
    assert tuple(q.shape) == (0, 90) and tuple(s.shape) == (0,)


def int8_inputs(name, seed=0, dense=False):
    counts, N, K, gathered, before, after = LISTS[name]
    g = gen(sum(map(ord, name)) + seed + 500)
    M = before + sum(counts) + after
    T = gathered or M
    q = torch.randint(-127, 128, (T, K), generator=g, dtype=torch.int8)
    s = torch.rand(T, generator=g) * 0.1 + 1e-3
    w = torch.randint(-128, 128, (len(counts), N, K), generator=g, dtype=torch.int8)
    ws = torch.rand(len(counts), N, generator=g) * 1e-2
    b = torch.randn(len(counts), N, generator=g)
    idx = torch.randint(0, T, (M,), generator=g, dtype=torch.int32) if gathered else None
    return q, s, w, ws, b, offsets_of(counts, before), idx


def close_int8(got, y, prod, bias, what):
    """The integer sum is exact; its rounding to fp32, two products and a sum
    are each within 2^-24 relative of what they give. A value past f16's range
    is an infinity."""
    tol = 4 * 2.0**-24 * (prod + bias) + UNIT[got.dtype] * y.abs() * 1.01 + STEP[got.dtype]
    over = torch.isinf(y.to(got.dtype))
    d = torch.where(over, (got.cpu().double() != y.to(got.dtype).double()).double() * torch.inf,
                    (got.cpu().double() - y).abs()).nan_to_num(0.0, posinf=torch.inf)
    assert bool((d <= tol).all()), (what, float((d - tol).max()))


@pytest.mark.parametrize("name", sorted(LISTS))
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_int8(name, out):
    q, s, w, ws, b, off, idx = int8_inputs(name)
    for bias in (None, b):
        y = linear.int8_linear(dev(q), dev(s), dev(w), dev(ws), dev(bias), out, off, dev(idx))
        want, prod, bm = ref.int8_forward(q, s, w, ws, bias, off, idx)
        assert y.dtype == out
        close_int8(y, want, prod, bm, name)


@pytest.mark.parametrize("M,N,K", [(1, 300, 4096), (17, 129, 65), (513, 260, 1000), (2, 16, 131071),
                                   (300, 512, 1024)])
def test_int8_dense(M, N, K):
    g = gen(M + N + K)
    q = torch.full((M, K), -128, dtype=torch.int8) if K > 100000 else torch.randint(
        -128, 128, (M, K), generator=g, dtype=torch.int8)
    w = torch.full((N, K), -128, dtype=torch.int8) if K > 100000 else torch.randint(
        -128, 128, (N, K), generator=g, dtype=torch.int8)
    s, ws = torch.rand(M, generator=g), torch.rand(N, generator=g) * 1e-4
    y = linear.int8_linear(dev(q), dev(s), dev(w), dev(ws), out_dtype=torch.float32)
    want, prod, bm = ref.int8_forward(q, s, w, ws)
    close_int8(y, want, prod, bm, "dense")
    y = linear.int8_linear(dev(q), dev(s), dev(w), dev(ws), out_dtype=torch.float16)
    close_int8(y, want, prod, bm, "dense f16")


@pytest.mark.parametrize("M,N,K", [(1, 200, 512), (5, 64, 96), (300, 260, 320), (700, 96, 1000),
                                   (4000, 264, 136)])
def test_dense_forms(M, N, K):
    g = gen(M * N)
    x, w = randn(g, M, K, dtype=torch.bfloat16), randn(g, N, K, dtype=torch.bfloat16, scale=0.1)
    dy = randn(g, M, N, dtype=torch.bfloat16)
    close(linear.grouped_linear(dev(x), dev(w)), *ref.forward(x, w), K, "dense")
    close(linear.grouped_linear_dgrad(dev(dy), dev(w)), *ref.dgrad(dy, w), N, "dense dgrad")
    close(linear.grouped_linear_wgrad(dev(dy), dev(x)), *ref.wgrad(dy, x), M, "dense wgrad")


@pytest.mark.parametrize("off", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("K", [64, 72, 200])
def test_strides_and_alignment(off, K):
    """Views with a pitch of their own and a start off every boundary, a
    transposed and a broadcast weight, expanded rows."""
    g = gen(off + K)
    x = randn(g, 90, 300, dtype=torch.bfloat16)
    w = randn(g, 3, 70, 300, dtype=torch.bfloat16, scale=0.1)
    dy = randn(g, 90, 120, dtype=torch.bfloat16)
    lists = [0, 30, 31, 90]
    xd, wd, dyd = dev(x)[:, off : off + K], dev(w)[:, :, off : off + K], dev(dy)[:, off : off + 70]
    xc, wc, dyc = x[:, off : off + K], w[:, :, off : off + K], dy[:, off : off + 70]
    close(linear.grouped_linear(xd, wd, lists), *ref.forward(xc, wc, lists), K, "views")
    close(linear.grouped_linear_dgrad(dyd, wd, lists), *ref.dgrad(dyc, wc, lists), 70, "dgrad views")
    close(linear.grouped_linear_wgrad(dyd, xd, lists), *ref.wgrad(dyc, xc, lists), 59, "wgrad views")
    wt = randn(g, 3, K, 70, dtype=torch.bfloat16, scale=0.1)
    close(linear.grouped_linear(xd, dev(wt).transpose(1, 2), lists),
          *ref.forward(xc, wt.transpose(1, 2), lists), K, "transposed weight")
    one = randn(g, 1, 70, K, dtype=torch.bfloat16, scale=0.1)
    close(linear.grouped_linear(xd, dev(one).expand(3, -1, -1), lists),
          *ref.forward(xc, one.expand(3, -1, -1), lists), K, "one weight for all")
    row = randn(g, 1, K, dtype=torch.bfloat16)
    close(linear.grouped_linear(dev(row).expand(90, -1), wd, lists),
          *ref.forward(row.expand(90, -1), wc, lists), K, "expanded row")
    q = torch.randint(-127, 128, (90, 300), generator=g, dtype=torch.int8)
    w8 = torch.randint(-127, 128, (3, 70, 300), generator=g, dtype=torch.int8)
    s, ws = torch.rand(90, generator=g), torch.rand(3, 70, generator=g)
    y = linear.int8_linear(dev(q)[:, off : off + K], dev(s), dev(w8)[:, :, off : off + K], dev(ws),
                           offsets=lists)
    close_int8(y, *ref.int8_forward(q[:, off : off + K], s, w8[:, :, off : off + K], ws,
                                    offsets=lists), "int8 views")
    xm = dev(x)[:, off : off + 64]
    codes = torch.randint(0, 16, (3, 70, 64), generator=g, dtype=torch.uint8)
    sc = torch.randint(120, 130, (3, 70, 2), generator=g).to(torch.uint8)
    y = linear.mxfp_linear(xm, packing.pack_q(codes.to(DEV), 4), dev(sc), "mxfp4", lists)
    close(y, *ref.forward(x[:, off : off + 64], ref.decode(codes, sc, "mxfp4"), lists), 64, "mx views")


@pytest.mark.parametrize("M", [9, 300])
def test_non_finite_values_stay_in_their_rows(M):
    """A NaN or an infinity reaches the results that read it and no other: not
    the neighbours of a tile, not another group, not zero rows of no group."""
    g = gen(M)
    x, w = randn(g, M, 100, dtype=torch.bfloat16), randn(g, 3, 70, 100, dtype=torch.bfloat16)
    off = [2, M // 2, M // 2, M - 2]
    x[0, 3] = float("nan")  # no group
    x[3, 5] = float("nan")
    x[M - 3, 99] = float("inf")
    x[M - 1] = float("inf")  # no group
    w[2, 7, 0] = float("nan")
    w[1] = float("nan")  # a group without entries
    y = linear.grouped_linear(dev(x), dev(w), off).cpu()
    ok = torch.isfinite(y)
    want = torch.ones_like(ok)
    want[3] = False
    want[M - 3] = False
    want[M // 2 : M - 2, 7] = False
    assert torch.equal(ok, want)
    assert bool((y[:2] == 0).all()) and bool((y[M - 2 :] == 0).all())
    dy = randn(g, M, 70, dtype=torch.bfloat16)
    dy[0] = float("nan")
    dy[M - 3, 4] = float("nan")
    dw = linear.grouped_linear_wgrad(dev(dy), dev(x), off).cpu()
    ok = torch.isfinite(dw)
    want = torch.ones_like(ok)
    want[0, :, 5] = False  # x[3, 5]
    want[2, 4, :] = False  # dy[M - 3, 4]
    want[2, :, 99] = False  # x[M - 3, 99]
    assert torch.equal(ok, want) and bool((dw[1] == 0).all())
    dx = linear.grouped_linear_dgrad(dev(dy), dev(w), off).cpu()
    ok = torch.isfinite(dx)
    want = torch.ones_like(ok)
    want[M - 3] = False
    want[M // 2 : M - 2, 0] = False  # w[2, 7, 0]
    assert torch.equal(ok, want) and bool((dx[:2] == 0).all()) and bool((dx[M - 2 :] == 0).all())
    q, s = linear.quantize_rows_int8(dev(x))
    w8 = torch.randint(-127, 128, (3, 70, 100), generator=g, dtype=torch.int8)
    y = linear.int8_linear(q, s, dev(w8), torch.ones(3, 70, device=DEV), offsets=off).cpu()
    bad = torch.isnan(y).all(dim=1)
    assert bad.nonzero().flatten().tolist() == [3, M - 3] and not bool(torch.isnan(y[~bad]).any())


def test_offsets_and_indexes_that_lie_are_not_followed():
    """Unvalidated lists with entries outside their ranges: the call returns, and
    what the clamped list defines is right."""
    g = gen(31)
    x, w = randn(g, 40, 64, dtype=torch.bfloat16), randn(g, 2, 48, 64, dtype=torch.bfloat16)
    off = torch.tensor([-5, 12, 9000], dtype=torch.int32)
    idx = torch.randint(0, 40, (30,), generator=g, dtype=torch.int32)
    idx[3], idx[7] = -9, 2**30
    want, mag = ref.forward(x, w, [0, 12, 30], idx.clamp(0, 39))
    y = linear.grouped_linear(dev(x), dev(w), dev(off), dev(idx), validate=False)
    close(y, want, mag, 64, "clamped")
    dy = randn(g, 30, 48, dtype=torch.bfloat16)
    dw = linear.grouped_linear_wgrad(dev(dy), dev(x), dev(off), dev(idx), validate=False)
    close(dw, *ref.wgrad(dy, x, [0, 12, 30], idx.clamp(0, 39)), 30, "clamped wgrad")
    dx = linear.grouped_linear_dgrad(dev(dy), dev(w), dev(off), dev(idx), 40, validate=False)
    close(dx, *ref.dgrad(dy, w, [0, 12, 30], idx.clamp(0, 39), 40), 100, "clamped dgrad")


def test_offsets_beyond_32_bits():
    """Rows and weights that lie more than 2^32 bytes apart."""
    g = gen(41)
    pitch = (3 << 30) // 40
    pitch -= pitch % 8
    store = torch.empty(40 * pitch + 72 * 128, dtype=torch.bfloat16, device=DEV)
    x = randn(g, 40, 128, dtype=torch.bfloat16)
    xd = store.as_strided((40, 128), (pitch, 1))
    xd.copy_(x)
    w = randn(g, 3, 72, 128, dtype=torch.bfloat16, scale=0.1)
    off, idx = [0, 10, 30, 60], torch.randint(0, 40, (60,), generator=g, dtype=torch.int32)
    dy = randn(g, 60, 72, dtype=torch.bfloat16)
    for i in (None, idx):
        o = off if i is not None else [0, 10, 30, 40]
        close(linear.grouped_linear(xd, dev(w), o, dev(i)), *ref.forward(x, w, o, i), 128, "far rows")
        d = dy[: o[-1]]
        close(linear.grouped_linear_wgrad(dev(d), xd, o, dev(i)), *ref.wgrad(d, x, o, i), 30, "far")
    del xd
    wd = store.as_strided((3, 72, 128), (20 * pitch - 8, 128, 1))
    wd.copy_(w)
    close(linear.grouped_linear(dev(x), wd, off, dev(idx)), *ref.forward(x, w, off, idx), 128, "far w")
    close(linear.grouped_linear_dgrad(dev(dy), wd, off), *ref.dgrad(dy, w, off), 72, "far w dgrad")


def test_on_a_stream_of_its_own_and_captured():
    """The call runs on the current stream, and a captured graph of the
    unvalidated calls gives on every replay what the eager calls give, with new
    contents in the same tensors."""
    x, w, off, idx, dy = make_list("few_each", torch.bfloat16, seed=7)
    xd, wd, dyd = dev(x), dev(w), dev(dy)
    offd, idxd = torch.tensor(off, dtype=torch.int32, device=DEV), dev(idx)
    sc = torch.rand(w.shape[0], w.shape[1], device=DEV)
    w8 = torch.randint(-127, 128, w.shape, dtype=torch.int8, device=DEV)

    def calls():
        q, s = linear.quantize_rows_int8(xd)
        return (linear.grouped_linear(xd, wd, offd, idxd, validate=False),
                linear.grouped_linear_dgrad(dyd, wd, offd, idxd, x.shape[0], validate=False),
                linear.grouped_linear_wgrad(dyd, xd, offd, idxd, validate=False),
                linear.int8_linear(q, s, w8, sc, offsets=offd, row_index=idxd, validate=False))

    want = calls()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = calls()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for seed in range(4):
        xd.copy_(randn(gen(seed + 60), *x.shape, dtype=torch.bfloat16))
        dyd.copy_(randn(gen(seed + 70), *dy.shape, dtype=torch.bfloat16))
        idxd.copy_(torch.randint(0, x.shape[0], idx.shape, generator=gen(seed + 80), dtype=torch.int32))
        want = calls()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, out)), seed


def test_host_tensors_and_host_results():
    x, w, off, idx, dy = make_list("few_each", torch.bfloat16, seed=8)
    y = linear.grouped_linear(x, w, off, idx)
    assert y.device.type == "cpu"
    assert torch.equal(y, linear.grouped_linear(dev(x), dev(w), off, dev(idx)).cpu())
