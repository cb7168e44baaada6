"""Which kernel a product takes (the host's choice; nothing is launched)."""

from __future__ import annotations

import ctypes

import torch

from mlx_gptq import _native as nat

PRODUCTS = {"bf16": 0, "f16": 1, "int8": 2, "mxfp4": 3, "mxfp8": 4, "dgrad_bf16": 5, "dgrad_f16": 6}
NAMES = {torch.bfloat16: "bf16", torch.float16: "f16", torch.int8: "int8"}
FEW, DIRECT, STAGED = 0, 1, 2


def choice(product, M, G, N, K, grouped, x=0, w=0, ldx=None, ldw=None):
    """(rows, columns, kind); x and w are the operands' addresses, pitches default to
    contiguous rows."""
    tile = (ctypes.c_int32 * 3)()
    width = N if product.startswith("dgrad") else K
    ldx, ldw = ldx or max(width, 1), ldw or max(K, 1)
    nat.call("mgq_linear_choice", PRODUCTS[product], x, ldx, M, w, G, N, K, ldw, N * ldw,
             int(grouped), ctypes.addressof(tile))
    return tuple(tile)


def of_call(product, M, x, weight, offsets):
    """The choice of linear's call on these tensors (rows x; mxfp: words `weight`)."""
    w = weight if weight.dim() == 3 else weight.unsqueeze(0)
    K = x.shape[1]
    ldw = w.stride(1) if w.dtype != torch.int32 else K
    return choice(product, M, w.shape[0], w.shape[1], K, offsets is not None, x.data_ptr(),
                  w.data_ptr(), x.stride(0) if x.shape[0] > 1 else K, ldw)
