"""float64 restatement of the matrix products of mlx_gptq.linear, on the CPU.

Every function also returns the sum of the terms' magnitudes, from which the
tests derive how far a sum in fp32 may be off.
"""

from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def spans(offsets, groups, entries):
    """(group, first entry, end) of every group."""
    if offsets is None:
        return [(0, 0, entries)]
    off = [int(v) for v in offsets]
    return [(g, off[g], off[g + 1]) for g in range(groups)]


def rows_of(x, row_index):
    return x.double() if row_index is None else x.double()[row_index.long()]


def forward(x, weight, offsets=None, row_index=None):
    """y[t] = x[row_index[t]] @ weight[g].T; entries of no group are zero."""
    w = weight.double()
    w = w.unsqueeze(0) if w.dim() == 2 else w
    xs = rows_of(x, row_index)
    y = torch.zeros(xs.shape[0], w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for g, a, b in spans(offsets, w.shape[0], xs.shape[0]):
        y[a:b] = xs[a:b] @ w[g].T
        mag[a:b] = xs[a:b].abs() @ w[g].abs().T
    return y, mag


def dgrad(dy, weight, offsets=None, row_index=None, n_rows=None):
    w = weight.double()
    w = w.unsqueeze(0) if w.dim() == 2 else w
    dxl = torch.zeros(dy.shape[0], w.shape[2], dtype=torch.float64)
    mag = torch.zeros_like(dxl)
    for g, a, b in spans(offsets, w.shape[0], dy.shape[0]):
        dxl[a:b] = dy[a:b].double() @ w[g]
        mag[a:b] = dy[a:b].double().abs() @ w[g].abs()
    if row_index is None:
        return dxl, mag
    out = torch.zeros(n_rows, w.shape[2], dtype=torch.float64)
    m = torch.zeros_like(out)
    out.index_add_(0, row_index.long(), dxl)
    m.index_add_(0, row_index.long(), mag)
    return out, m


def wgrad(dy, x, offsets=None, row_index=None):
    xs = rows_of(x, row_index)
    groups = 1 if offsets is None else len(offsets) - 1
    dw = torch.zeros(groups, dy.shape[1], x.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for g, a, b in spans(offsets, groups, xs.shape[0]):
        dw[g] = dy[a:b].double().T @ xs[a:b]
        mag[g] = dy[a:b].double().abs().T @ xs[a:b].abs()
    return (dw[0], mag[0]) if offsets is None else (dw, mag)


def decode(q, scales, mode):
    """Codes [..., K] and E8M0 bytes [..., K / 32] -> float64 weights."""
    q = q.long()
    if mode == "mxfp4":
        v = E2M1[q & 7] * torch.where(q >= 8, -1.0, 1.0).double()
    else:
        e, m = (q >> 3) & 15, (q & 7).double()
        v = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2((e - 7).double()))
        v = torch.where((q & 127) == 127, torch.nan, v) * torch.where(q >= 128, -1.0, 1.0).double()
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, dim=-1)


def affine(q, scales, biases):
    """Codes [..., K], scales and biases [..., K / group] -> (float64 weights, the
    magnitudes |q scale| + |bias| of their two terms)."""
    group = q.shape[-1] // scales.shape[-1]
    s, b = (t.double().repeat_interleave(group, dim=-1) for t in (scales, biases))
    return q.double() * s + b, q.double() * s.abs() + b.abs()


def affine_forward(x, q, scales, biases, offsets=None, row_index=None):
    """(y, the sum of |x| (|q scale| + |bias|))."""
    w, m = affine(q, scales, biases)
    return (forward(x, w, offsets, row_index)[0],
            forward(x.double().abs(), m, offsets, row_index)[0])


def quantize_rows(x):
    """(codes, scales) with the quotients rounded to fp32 as defined."""
    f = x.double()
    s = (f.abs().amax(dim=-1) / 127).float()
    ratio = torch.where(s[..., None] > 0, f / s.double()[..., None], 0.0).float()
    q = torch.round(ratio)
    bad = ~torch.isfinite(f).all(dim=-1)
    s = torch.where(bad, torch.nan, s)
    q = torch.where(bad[..., None], 0.0, q)
    return q.to(torch.int8), s


def int8_forward(q, s, weight, w_scale, bias=None, offsets=None, row_index=None):
    """(y, |product|, |bias|); the integer sum is exact in float64."""
    w = weight if weight.dim() == 3 else weight.unsqueeze(0)
    ws = w_scale.double() if weight.dim() == 3 else w_scale.double().unsqueeze(0)
    xs = rows_of(q, row_index)
    ss = rows_of(s, row_index)
    y = torch.zeros(xs.shape[0], w.shape[1], dtype=torch.float64)
    bm = torch.zeros_like(y)
    for g, a, b in spans(offsets, w.shape[0], xs.shape[0]):
        y[a:b] = (xs[a:b] @ w[g].double().T) * ss[a:b, None] * ws[g]
        if bias is not None:
            bm[a:b] = (bias if bias.dim() == 1 else bias[g]).double()
    return y + bm, y.abs(), bm.abs()
