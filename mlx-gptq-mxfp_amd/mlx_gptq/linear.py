"""Matrix products with dense, MXFP, affine and int8 weights on MI355X.

What the solver's codes are multiplied with: the products of a calibration
forward, a fine-tuning step or a serving program, for one weight or for every
expert of a routed layer at once. The reference leaves these to torch and MLX;
the kernels are csrc/linear*.hip and csrc/affine_linear.hip.

* ``grouped_linear`` (bf16 or f16 weights, differentiable) with its two
  gradients ``grouped_linear_dgrad`` and ``grouped_linear_wgrad``;
* ``mxfp_linear``: the same product with packed MXFP4 / MXFP8 weights, decoded
  inside the kernel;
* ``affine_linear``: the same with packed 2-, 4- or 8-bit codes and a scale and a
  bias for each group of 32, 64 or 128 values (MLX's affine grid);
* ``quantize_rows_int8`` and ``int8_linear``: rows quantized to 8-bit integers
  with a scale each, and their product with 8-bit weights that have a scale for
  each output channel.

Groups. The rows are a list of entries in the experts' order: expert g owns
entries ``offsets[g]:offsets[g + 1]``, as ``capture.RoutedStash.plan`` lays
them out. With ``row_index`` entry t reads row ``row_index[t]`` of ``x`` (the
gather is part of the product; nothing is copied), without it row t. Entries
that belong to no group give zero rows. ``offsets=None`` is one dense weight
(without its leading dimension). Offsets on the device stay there: with
``validate=False`` no call waits for the device, so a decoding loop can be
captured in a graph. Offsets and indexes outside their ranges are clamped by the
kernels, never followed; ``validate`` raises for them, and for offsets that decrease
(unvalidated, those leave rows of the result unwritten). Only ``grouped_linear``
is differentiable. The other calls run on tensors that require a gradient, but a
backward that reaches their results raises, as forward-mode tangents do in every call.

Work is enqueued on the current stream of the tensors' device. Host tensors are
staged through the current HIP device, as in the other modules.
"""

from __future__ import annotations

import functools
import operator

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _native as nat

_MX_MODES = {"mxfp4": (4, nat.MODE_MXFP4), "mxfp8": (8, nat.MODE_MXFP8)}  # bits, code
_AFFINE_BITS = (2, 4, 8)
_AFFINE_GROUPS = (32, 64, 128)
_HALF = (torch.bfloat16, torch.float16)
_FLOATS = (torch.float32, *_HALF)
_WORDS = (torch.int32, torch.uint32)


# A single token's product takes a few microseconds, which the calls below reach
# only if the host side of one takes no longer: contiguous device tensors pass with
# one comparison each.


def _pitched(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """`t` on `dev` with contiguous rows that do not overlap (a copy if need be)."""
    if t.device != dev:
        t = t.to(dev)
    if not t.is_contiguous() and (
            t.stride(-1) != 1 or (t.shape[-2] > 1 and t.stride(-2) < t.shape[-1])):
        t = t.contiguous()
    return t


def _dense(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """`t` on `dev`, contiguous."""
    return t if t.device == dev and t.is_contiguous() else nat.on_device(t, dev)


def _device(*tensors: torch.Tensor) -> torch.device:
    return tensors[0].device if tensors[0].is_cuda else nat.device_for(*tensors)


def _home(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """The result on the caller's device."""
    return t if like.is_cuda else t.to(like.device)


def _ld(t: torch.Tensor) -> int:
    """Row pitch in elements (a single row's stride says nothing)."""
    shape = t.shape
    return t.stride(-2) if shape[-2] > 1 else max(shape[-1], 1)


def _weight3(fn: str, weight: torch.Tensor, offsets) -> torch.Tensor:
    """The weight as [G, N, K]; dense weights are [N, K]."""
    if offsets is None:
        if weight.dim() != 2:
            raise ValueError(f"{fn}: without offsets the weight is [N, K] (got {tuple(weight.shape)})")
        return weight.unsqueeze(0)
    if weight.dim() != 3:
        raise ValueError(f"{fn}: with offsets the weight is [G, N, K] (got {tuple(weight.shape)})")
    return weight


def _rows2(fn: str, name: str, x: torch.Tensor) -> None:
    if x.dim() != 2:
        raise ValueError(f"{fn}: {name} must be a matrix (got {tuple(x.shape)})")


def _integers(t: torch.Tensor) -> bool:
    dt = t.dtype
    return dt is torch.int32 or not (dt.is_floating_point or dt.is_complex or dt is torch.bool)


def _int32(t: torch.Tensor) -> torch.Tensor:
    """`t` in 32 bits. What lies past them stays out of range, as the kernels' clamps
    expect it."""
    if t.dtype is torch.int32:
        return t
    if t.dtype in (torch.int64, torch.uint64, torch.uint32):
        wide = t.to(torch.int64)
        if t.dtype is torch.uint64:  # (2^63 and more read as negative numbers)
            wide = wide.masked_fill(wide < 0, 2**31 - 1)
        t = wide.clamp(-(2**31), 2**31 - 1)
    return t.to(torch.int32)


def _list(fn: str, offsets, row_index, groups: int, n_rows: int, dev: torch.device, validate: bool):
    """(offsets int32 on dev | None, row_index int32 on dev | None, entries)."""
    if row_index is not None:
        if row_index.dim() != 1 or not _integers(row_index):
            raise ValueError(f"{fn}: row_index must be a list of integers")
        if validate and row_index.numel():
            lo, hi = torch.aminmax(row_index)
            if int(lo) < 0 or int(hi) >= n_rows:
                raise IndexError(f"{fn}: row_index outside [0, {n_rows})")
        row_index = _dense(_int32(row_index), dev)
    entries = n_rows if row_index is None else row_index.numel()
    if offsets is None:
        return None, row_index, entries
    if not isinstance(offsets, torch.Tensor):
        host = np.asarray(offsets)
        whole = host.dtype.kind != "f" or bool(np.all(host == np.floor(host)))
        offsets = torch.from_numpy(host.astype(np.int64) if whole else np.array(host, dtype=np.float64))
    if offsets.dim() != 1 or offsets.numel() != groups + 1 or not _integers(offsets):
        raise ValueError(f"{fn}: offsets must hold {groups + 1} integers for {groups} groups")
    if validate or not offsets.is_cuda:
        o = offsets.detach().cpu().numpy()
        if np.any(np.diff(o) < 0) or o[0] < 0:
            raise ValueError(f"{fn}: offsets must be non-negative and non-decreasing")
        if o[-1] > entries:
            raise ValueError(f"{fn}: offsets exceed the {entries} list entries")
    return _dense(_int32(offsets), dev), row_index, entries


def _check_half(fn: str, a: torch.Tensor, b: torch.Tensor) -> None:
    dt = a.dtype
    if dt not in _HALF or b.dtype != dt:
        raise TypeError(f"{fn}: expects bfloat16 or float16 tensors of one type "
                        f"(got {dt}, {b.dtype})")


def _tracked(fn: str, *tensors: torch.Tensor) -> bool:
    """Whether autograd would follow a result of `tensors`. Forward-mode tangents are
    refused (outside their levels that costs one comparison)."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{fn} has no forward-mode derivative")
    for t in tensors:
        if t.requires_grad:
            return torch.is_grad_enabled()
    return False


class _NoGradient(torch.autograd.Function):
    """A result that has no gradient, handed on with a backward that raises, where the
    plain result would read as a constant."""

    @staticmethod
    def forward(ctx, fn, out, *inputs):
        ctx.fn = fn
        return out.detach()

    @staticmethod
    def backward(ctx, dy):
        raise NotImplementedError(f"{ctx.fn} has no gradient: detach its inputs, or call it under "
                                  "torch.no_grad()")


def _forward(x, weight, offsets, row_index, validate):
    """(y, offsets, row_index), the lists as the product ran on them."""
    fn = "grouped_linear"
    _check_half(fn, x, weight)
    _rows2(fn, "x", x)
    w = _weight3(fn, weight, offsets)
    G, N, K = w.shape
    if x.shape[1] != K:
        raise AssertionError(f"{fn}: x has {x.shape[1]} columns, the weight {K}")
    dev = _device(x, weight)
    xd, wd = _pitched(x, dev), _pitched(w, dev)
    off, idx, M = _list(fn, offsets, row_index, G, int(x.shape[0]), dev, validate)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    if M and N:
        nat.launch(dev, "mgq_grouped_linear", xd.data_ptr(), nat.dtype_code(x.dtype), xd.shape[0],
                   _ld(xd), nat.ptr(idx), M, wd.data_ptr(), G, N, K, _ld(wd), wd.stride(0),
                   nat.ptr(off), y.data_ptr())
    return _home(y, x), off, idx


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, offsets, row_index, validate):
        y, offsets, row_index = _forward(x, weight, offsets, row_index, validate)
        # the lists are saved like the operands, so that a routing buffer that is
        # written again before the backward is an error there (routing made in
        # inference mode has no version to check: a copy is saved)
        lists = (t.clone() if t is not None and t.is_inference() else t for t in (offsets, row_index))
        # (each operand only for the other one's gradient)
        needs_x, needs_weight = ctx.needs_input_grad[:2]
        ctx.n_rows, ctx.weight_device = x.shape[0], weight.device
        ctx.save_for_backward(x if needs_weight else None, weight if needs_x else None, *lists)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, offsets, row_index = ctx.saved_tensors
        dx = dw = None
        if ctx.needs_input_grad[0]:
            dx = grouped_linear_dgrad(dy, weight, offsets, row_index, ctx.n_rows, validate=False)
        if ctx.needs_input_grad[1]:
            dw = grouped_linear_wgrad(dy, x, offsets, row_index, validate=False).to(ctx.weight_device)
        return dx, dw, None, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets=None,
                   row_index: torch.Tensor | None = None, validate: bool = True) -> torch.Tensor:
    """y[t] = x[row_index[t]] @ weight[g].T for the entries t of every group g.

    x: [T, K] bf16 or f16, weight: [G, N, K] of the same type (any row pitch),
    offsets: G + 1 integers (a device tensor or any host sequence) ->
    [entries, N]. fp32 sums, rounded once. Differentiable in x and weight: the
    gradients are ``grouped_linear_dgrad`` and ``grouped_linear_wgrad`` on the
    lists of the forward (autograd refuses a backward after int32 lists on the
    device, or the tensors they are views of, were written again). The gradients
    have none themselves: a second derivative raises.
    """
    if _tracked("grouped_linear", x, weight):
        return _GroupedLinear.apply(x, weight, offsets, row_index, validate)
    return _forward(x, weight, offsets, row_index, validate)[0]


def grouped_linear_dgrad(dy: torch.Tensor, weight: torch.Tensor, offsets=None,
                         row_index: torch.Tensor | None = None, n_rows: int | None = None,
                         validate: bool = True) -> torch.Tensor:
    """Gradient of ``grouped_linear`` with respect to x: [n_rows, K].

    dy: [entries, N]. With ``row_index``, row r is the sum over the entries that
    read it, in fp32 and in the entries' order, rounded once (``n_rows`` is
    required; rows that no entry reads are zero).
    """
    fn = "grouped_linear_dgrad"
    tracked = _tracked(fn, dy, weight)
    _check_half(fn, dy, weight)
    _rows2(fn, "dy", dy)
    w = _weight3(fn, weight, offsets)
    G, N, K = w.shape
    if dy.shape[1] != N:
        raise AssertionError(f"{fn}: dy has {dy.shape[1]} columns, the weight {N} rows")
    if row_index is not None and n_rows is None:
        raise ValueError(f"{fn}: n_rows is required with row_index")
    dev = _device(dy, weight)
    dyd, wd = _pitched(dy, dev), _pitched(w, dev)
    M = int(dy.shape[0])
    off, idx, entries = _list(fn, offsets, row_index, G, M if row_index is None else int(n_rows),
                              dev, validate)
    if entries != M:
        raise ValueError(f"{fn}: dy has {M} rows, row_index {entries} entries")
    gathered = idx is not None
    out_type = torch.float32 if gathered else dy.dtype
    dx = torch.empty(M, K, dtype=out_type, device=dev)
    if M and K and N:
        nat.launch(dev, "mgq_grouped_dgrad", dyd.data_ptr(), nat.dtype_code(dy.dtype), M, _ld(dyd),
                   wd.data_ptr(), G, N, K, _ld(wd), wd.stride(0), nat.ptr(off), dx.data_ptr(),
                   nat.dtype_code(out_type))
    elif N == 0:
        dx.zero_()
    if gathered:
        out = torch.empty(int(n_rows), K, dtype=dy.dtype, device=dev)
        if out.numel():
            ws = torch.empty(nat.load().mgq_rows_sum_workspace_size(M, int(n_rows)),
                             dtype=torch.uint8, device=dev)
            nat.launch(dev, "mgq_rows_sum", dx.data_ptr(), idx.data_ptr(), M, int(n_rows), K,
                       out.data_ptr(), nat.dtype_code(out.dtype), ws.data_ptr(), ws.numel())
        dx = out
    dx = _home(dx, dy)
    return _NoGradient.apply(fn, dx, dy, weight) if tracked else dx


def grouped_linear_wgrad(dy: torch.Tensor, x: torch.Tensor, offsets=None,
                         row_index: torch.Tensor | None = None, validate: bool = True,
                         out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of ``grouped_linear`` with respect to the weight: [G, N, K]
    ([N, K] without offsets), of dy's type or ``out_dtype=torch.float32``.

    dy: [entries, N], x: [T, K]. fp32 sums over a group's entries, rounded
    once; zeros for a group without entries. At most 4096 groups. A call takes up
    to 0.75 GiB of workspace for the partial results of long groups.
    """
    fn = "grouped_linear_wgrad"
    tracked = _tracked(fn, dy, x)
    _check_half(fn, dy, x)
    _rows2(fn, "dy", dy)
    _rows2(fn, "x", x)
    out_dtype = dy.dtype if out_dtype is None else out_dtype
    if out_dtype not in (dy.dtype, torch.float32):
        raise TypeError(f"{fn}: the result is {dy.dtype} or float32 (got {out_dtype})")
    dev = _device(dy, x)
    dyd, xd = _pitched(dy, dev), _pitched(x, dev)
    G = 1 if offsets is None else len(offsets) - 1
    if G < 1:
        raise ValueError(f"{fn}: offsets must hold at least two integers")
    off, idx, M = _list(fn, offsets, row_index, G, int(x.shape[0]), dev, validate)
    if dy.shape[0] != M:
        raise ValueError(f"{fn}: dy has {dy.shape[0]} rows, the list {M} entries")
    N, K = int(dy.shape[1]), int(x.shape[1])
    dw = torch.empty(G, N, K, dtype=out_dtype, device=dev)
    if N and K:
        size = nat.load().mgq_grouped_wgrad_workspace_size(M, G, N, K)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        nat.launch(dev, "mgq_grouped_wgrad", dyd.data_ptr(), nat.dtype_code(dy.dtype), M, _ld(dyd),
                   xd.data_ptr(), xd.shape[0], _ld(xd), nat.ptr(idx), G, N, K, nat.ptr(off),
                   dw.data_ptr(), nat.dtype_code(out_dtype), nat.ptr(ws), size)
    if offsets is None:
        dw = dw[0]
    dw = _home(dw, dy)
    return _NoGradient.apply(fn, dw, dy, x) if tracked else dw


def check_mxfp(fn: str, cols: int, mode: str, packed: torch.Tensor, scales: torch.Tensor) -> None:
    """The tensors of an MXFP weight [..., N, cols]."""
    if packed.dtype not in _WORDS or scales.dtype is not torch.uint8:
        raise TypeError(f"{fn}: expects 32-bit words and uint8 scales "
                        f"(got {packed.dtype} and {scales.dtype})")
    *lead, words = packed.shape
    K = words * 32 // _MX_MODES[mode][0]
    if cols != K or K % 32:
        raise AssertionError(f"{fn}: x has {cols} columns, the words hold {K} (a multiple of 32)")
    if scales.shape != (*lead, K // 32):
        raise AssertionError(f"{fn}: scales must be {(*lead, K // 32)} (got {tuple(scales.shape)})")


def mxfp_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, mode: str,
                offsets=None, row_index: torch.Tensor | None = None,
                validate: bool = True) -> torch.Tensor:
    """``grouped_linear`` with MXFP4 or MXFP8 weights.

    x: [T, K] bf16, packed: [G, N, K * bits / 32] words as ``packing.pack_q``
    (or the solver's ``packed_out``) lays them out, scales: uint8
    [G, N, K / 32] E8M0 bytes; without offsets both lack the leading G.
    -> bf16 [entries, N]. The decoded weights are exact in bf16, the sums fp32.
    """
    fn = "mxfp_linear"
    tracked = _tracked(fn, x)
    if mode not in _MX_MODES:
        raise ValueError(f"not a microscaling mode: {mode}")
    code = _MX_MODES[mode][1]
    if x.dtype is not torch.bfloat16:
        raise TypeError(f"{fn}: expects bfloat16 rows (got {x.dtype})")
    _rows2(fn, "x", x)
    w, s = _weight3(fn, packed, offsets), _weight3(fn, scales, offsets)
    K = int(x.shape[1])
    check_mxfp(fn, K, mode, w, s)
    G, N, _ = w.shape
    dev = _device(x, packed, scales)
    xd = _pitched(x, dev)
    wd, sd = _dense(w, dev), _dense(s, dev)
    off, idx, M = _list(fn, offsets, row_index, G, int(x.shape[0]), dev, validate)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    if M and N:
        nat.launch(dev, "mgq_mxfp_linear", xd.data_ptr(), xd.shape[0], _ld(xd), nat.ptr(idx), M,
                   wd.data_ptr(), sd.data_ptr(), code, G, N, K, nat.ptr(off), y.data_ptr())
    y = _home(y, x)
    return _NoGradient.apply(fn, y, x) if tracked else y


@functools.lru_cache(maxsize=1024)
def affine_dims(fn: str, cols: int, bits: int, words: torch.Size, word_type: torch.dtype,
                scales: torch.Size, scale_type: torch.dtype, biases: torch.Size,
                bias_type: torch.dtype, grouped: bool) -> tuple[int, int, int]:
    """(groups, rows, group size) of an affine weight for rows of `cols`, its tensors'
    shapes and types checked. (Remembered by these: a single token's product takes about
    as long as the checks.)"""
    if bits not in _AFFINE_BITS:
        raise ValueError(f"{fn}: bits must be one of {_AFFINE_BITS} (got {bits})")
    if word_type not in _WORDS:
        raise TypeError(f"{fn}: expects 32-bit words (got {word_type})")
    if scale_type not in _FLOATS or bias_type != scale_type:
        raise TypeError(f"{fn}: scales and biases must be float32, bfloat16 or float16 of one type "
                        f"(got {scale_type} and {bias_type})")
    if len(words) != 2 + grouped:
        with_, dims = ("with", "[G, N, K]") if grouped else ("without", "[N, K]")
        raise ValueError(f"{fn}: {with_} offsets the weight is {dims} (got words {tuple(words)})")
    if not cols or cols * bits != words[-1] * 32:
        raise AssertionError(f"{fn}: x has {cols} columns, the words hold {words[-1] * 32 // bits}")
    n = scales[-1] if scales else 0
    group = cols // n if n and cols % n == 0 else 0
    if group not in _AFFINE_GROUPS:
        raise ValueError(f"{fn}: groups of 32, 64 or 128 values (got {n} scales for {cols})")
    if scales[:-1] != words[:-1] or biases != scales:
        raise AssertionError(f"{fn}: scales and biases must be {(*words[:-1], n)} "
                             f"(got {tuple(scales)} and {tuple(biases)})")
    return (words[0] if grouped else 1), words[-2], group


def affine_linear(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor,
                  bits: int, offsets=None, row_index: torch.Tensor | None = None,
                  validate: bool = True) -> torch.Tensor:
    """``grouped_linear`` with affine weights w = q * scale + bias.

    x: [T, K] bf16 or f16, packed: [G, N, K * bits / 32] words as ``packing.pack_q``
    lays them out (bits 2, 4 or 8), scales and biases: [G, N, K / group] float32,
    bf16 or f16, as ``gptq.solve_gptq`` and ``grid.rtn_quantize`` return them, for
    groups of 32, 64 or 128 values; without offsets all three lack the leading G.
    -> [entries, N] of x's type. fp32 sums, rounded once. For few rows (up to some 128 a
    group, as measured) the weights are not rounded, as q * scale and bias enter the sum
    apart; for more they are rounded to x's type, like a dense weight of it (in float16 a
    weight past 65504 is then infinite). For few rows a row that holds an infinity, or
    values beyond 1e34, may give results that are no numbers where the product with the
    decoded weight would be infinite.
    """
    fn = "affine_linear"
    tracked = _tracked(fn, x, scales, biases)
    if x.dtype not in _HALF:
        raise TypeError(f"{fn}: expects bfloat16 or float16 rows (got {x.dtype})")
    _rows2(fn, "x", x)
    T, K = x.shape
    st = scales.dtype
    bits = operator.index(bits)
    G, N, group = affine_dims(fn, K, bits, packed.shape, packed.dtype, scales.shape, st, biases.shape,
                              biases.dtype, offsets is not None)
    dev = _device(x, packed, scales)
    xd = _pitched(x, dev)
    wd, sd, bd = _dense(packed, dev), _dense(scales, dev), _dense(biases, dev)
    off = idx = None
    M = T
    if offsets is not None or row_index is not None:
        off, idx, M = _list(fn, offsets, row_index, G, T, dev, validate)
    y = torch.empty(M, N, dtype=x.dtype, device=dev)
    if M and N:
        nat.launch(dev, "mgq_affine_linear", xd.data_ptr(), nat.dtype_code(x.dtype), T, _ld(xd),
                   None if idx is None else idx.data_ptr(), M, wd.data_ptr(), sd.data_ptr(),
                   bd.data_ptr(), nat.dtype_code(st), bits, group, G, N, K,
                   None if off is None else off.data_ptr(), y.data_ptr())
    y = _home(y, x)
    return _NoGradient.apply(fn, y, x, scales, biases) if tracked else y


def quantize_rows_int8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows as 8-bit integers with a scale each: (q int8 [..., K], scales f32
    [...]), scale = max|row| / 127, q = round-half-even(row / scale).

    A zero row has scale 0 and zero codes. A row that holds a NaN or an infinity
    has scale NaN and zero codes, so products with it are NaN.
    """
    tracked = _tracked("quantize_rows_int8", x)
    if x.dtype not in _FLOATS:
        raise TypeError(f"quantize_rows_int8: expects float32, bfloat16 or float16 (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"quantize_rows_int8: rows of no elements ({tuple(x.shape)})")
    dev = _device(x)
    rows = _pitched(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]), dev)
    q = torch.empty(x.shape, dtype=torch.int8, device=dev)
    s = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    if rows.shape[0]:
        nat.launch(dev, "mgq_quantize_rows_int8", rows.data_ptr(), nat.dtype_code(x.dtype),
                   rows.shape[0], rows.shape[1], _ld(rows), q.data_ptr(), s.data_ptr())
    q, s = _home(q, x), _home(s, x)
    return q, _NoGradient.apply("quantize_rows_int8", s, x) if tracked else s


def int8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor,
                w_scale: torch.Tensor, bias: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16, offsets=None,
                row_index: torch.Tensor | None = None, validate: bool = True) -> torch.Tensor:
    """y[t, n] = (x[r] . weight[g, n]) * x_scale[r] * w_scale[g, n] (+ bias[g, n]).

    x: int8 [T, K] with x_scale f32 [T] (``quantize_rows_int8``), weight: int8
    [G, N, K] with w_scale f32 [G, N], bias f32 [G, N]; without offsets the
    weight's tensors lack the leading G. -> ``out_dtype`` [entries, N]. The sum
    is exact (int32, K <= 131071), the scaling fp32, rounded once. Entries of no
    group are zero, without bias.
    """
    fn = "int8_linear"
    scaling = (x_scale, w_scale) if bias is None else (x_scale, w_scale, bias)
    tracked = _tracked(fn, *scaling)
    if x.dtype is not torch.int8 or weight.dtype is not torch.int8:
        raise TypeError(f"{fn}: expects int8 rows and weights (got {x.dtype} and {weight.dtype})")
    for t in scaling:
        if t.dtype is not torch.float32:
            raise TypeError(f"{fn}: x_scale, w_scale and bias must be float32 (got {t.dtype})")
    if out_dtype not in _FLOATS:
        raise TypeError(f"{fn}: the result is float32, bfloat16 or float16 (got {out_dtype})")
    _rows2(fn, "x", x)
    w = _weight3(fn, weight, offsets)
    G, N, K = w.shape
    if x.shape[1] != K:
        raise AssertionError(f"{fn}: x has {x.shape[1]} columns, the weight {K}")
    per_channel = (N,) if offsets is None else (G, N)
    if x_scale.shape != (x.shape[0],) or w_scale.shape != per_channel or (
            bias is not None and bias.shape != per_channel):
        raise AssertionError(f"{fn}: x_scale must be {(int(x.shape[0]),)}, w_scale and bias "
                             f"{per_channel}")
    dev = _device(x, weight)
    xd, wd = _pitched(x, dev), _pitched(w, dev)
    xs, ws = _dense(x_scale, dev), _dense(w_scale, dev)
    b = None if bias is None else _dense(bias, dev)
    off, idx, M = _list(fn, offsets, row_index, G, int(x.shape[0]), dev, validate)
    y = torch.empty(M, N, dtype=out_dtype, device=dev)
    if M and N:
        nat.launch(dev, "mgq_int8_linear", xd.data_ptr(), xs.data_ptr(), xd.shape[0], _ld(xd),
                   nat.ptr(idx), M, wd.data_ptr(), ws.data_ptr(), nat.ptr(b), G, N, K, _ld(wd),
                   wd.stride(0), nat.ptr(off), y.data_ptr(), nat.dtype_code(out_dtype))
    y = _home(y, x)
    return _NoGradient.apply(fn, y, *scaling) if tracked else y
