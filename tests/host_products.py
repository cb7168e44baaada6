"""The C entries of the matrix products computed on the CPU from the same
arguments, so that what mlx_gptq.linear does around its launches (autograd, lists,
devices) runs without a GPU. Pointers are followed as the kernels follow them."""

from __future__ import annotations

import ctypes

import torch

from mlx_gptq import _native as nat
from mlx_gptq import linear

TYPES = {nat.DTYPE_F32: torch.float32, nat.DTYPE_BF16: torch.bfloat16, nat.DTYPE_F16: torch.float16}


def at(ptr, dtype, *shape, strides=None):
    """The tensor at `ptr` (row-major unless `strides` are given)."""
    if 0 in shape:
        return torch.empty(shape, dtype=dtype)
    if strides is None:
        strides, n = [], 1
        for s in reversed(shape):
            strides.insert(0, n)
            n *= s
    count = 1 + sum((s - 1) * st for s, st in zip(shape, strides))
    size = count * torch.empty(0, dtype=dtype).element_size()
    buf = (ctypes.c_char * size).from_address(ptr)
    return torch.frombuffer(buf, dtype=dtype).as_strided(shape, strides)


def _lists(off, idx, G, M, n_rows):
    rows = torch.arange(M) if idx is None else at(idx, torch.int32, M).long().clamp(0, n_rows - 1)
    if off is None:
        return rows, [(0, 0, M)]
    o = at(off, torch.int32, G + 1).clamp(0, M).tolist()
    return rows, [(g, o[g], max(o[g], o[g + 1])) for g in range(G)]


def grouped_linear(X, dtype, n_rows, ldx, idx, M, W, G, N, K, ldw, wg, off, Y, stream):
    dt = TYPES[dtype]
    rows, spans = _lists(off, idx, G, M, n_rows)
    x = at(X, dt, n_rows, K, strides=(ldx, 1)).float()[rows]
    w = at(W, dt, G, N, K, strides=(wg, ldw, 1)).float()
    y = at(Y, dt, M, N)
    y.zero_()
    for g, a, b in spans:
        y[a:b] = (x[a:b] @ w[g].T).to(dt)


def grouped_dgrad(dY, dtype, M, lddy, W, G, N, K, ldw, wg, off, dX, out_dtype, stream):
    dt = TYPES[dtype]
    dy = at(dY, dt, M, N, strides=(lddy, 1)).float()
    w = at(W, dt, G, N, K, strides=(wg, ldw, 1)).float()
    dx = at(dX, TYPES[out_dtype], M, K)
    dx.zero_()
    for g, a, b in _lists(off, None, G, M, M)[1]:
        dx[a:b] = (dy[a:b] @ w[g]).to(dx.dtype)


def grouped_wgrad(dY, dtype, M, lddy, X, n_rows, ldx, idx, G, N, K, off, dW, out_dtype, ws, size,
                  stream):
    dt = TYPES[dtype]
    rows, spans = _lists(off, idx, G, M, n_rows)
    dy = at(dY, dt, M, N, strides=(lddy, 1)).float()
    x = at(X, dt, n_rows, K, strides=(ldx, 1)).float()[rows]
    dw = at(dW, TYPES[out_dtype], G, N, K)
    for g, a, b in spans:
        dw[g] = (dy[a:b].T @ x[a:b]).to(dw.dtype)


def rows_sum(src, idx, M, n_rows, cols, out, dtype, ws, size, stream):
    rows = at(idx, torch.int32, M).long().clamp(0, n_rows - 1)
    total = torch.zeros(n_rows, cols).index_add_(0, rows, at(src, torch.float32, M, cols))
    at(out, TYPES[dtype], n_rows, cols).copy_(total)


def mxfp_linear(X, n_rows, ldx, idx, M, words, scales, mode, G, N, K, off, Y, stream):
    at(Y, torch.bfloat16, M, N).fill_(1.0)


def quantize_rows_int8(X, dtype, rows, cols, ldx, q, scales, stream):
    x = at(X, TYPES[dtype], rows, cols, strides=(ldx, 1)).float()
    s = x.abs().amax(dim=1) / 127
    at(scales, torch.float32, rows).copy_(s)
    at(q, torch.int8, rows, cols).copy_(torch.round(x / s[:, None]).nan_to_num())


def int8_linear(X, xs, n_rows, ldx, idx, M, W, ws, bias, G, N, K, ldw, wg, off, Y, dtype, stream):
    at(Y, TYPES[dtype], M, N).fill_(1.0)


def install(monkeypatch, device=torch.device("cpu")):
    """mlx_gptq.linear on host tensors; returns the list of calls made."""
    calls = []

    def launch(device, name, *args):
        calls.append(name)
        globals()[name.removeprefix("mgq_")](*args, 0)

    monkeypatch.setattr(linear, "_device", lambda *tensors: device)
    monkeypatch.setattr(nat, "launch", launch)
    return calls
