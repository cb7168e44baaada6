"""The MLP of a routed layer's experts, on the grouped products of linear.py.

``ExpertMLP`` computes what a transformers fused-expert module computes
(``forward(hidden_states, top_k_index, top_k_weights)``: gate/up projection,
SiLU(gate) * up, down projection, sum over a row's experts with the router's
weights), every expert in one product instead of the eager loop over experts,
with weights that are

* ``"dense"``: bf16 or f16, differentiable (a fine-tuning step of the experts, or
  the forward that feeds a calibration's next layer);
* ``"mxfp4"`` / ``"mxfp8"``: the solver's or ``grid.rtn_quantize_mxfp``'s codes,
  packed;
* ``"affine"``: 2-, 4- or 8-bit codes of the affine grid, packed, with a scale and a
  bias for each group;
* ``"int8"``: 8-bit weights with a scale for each output channel, rows quantized
  to 8 bits on the way into each product.

Only dense experts are differentiable; in the other formats a backward that reaches
the rows raises.

``top_k_softmax`` is the router's choice that both take, with its gradient.

``ExpertMLP.decode`` is the same layer for up to 64 rows in two launches, where
``forward`` sorts the assignments and takes about 25.

No call waits for the device: the routing stays there.
"""

from __future__ import annotations

import ctypes
import operator
import weakref
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import _native as nat
from . import grid, linear, packing


MAX_TOP_K = 16
MAX_EXPERTS = 1024


def _check_logits(fn: str, logits: torch.Tensor, k: int) -> None:
    if logits.dtype not in linear._FLOATS:
        raise TypeError(f"{fn}: expects float32, bfloat16 or float16 logits (got {logits.dtype})")
    linear._rows2(fn, "logits", logits)
    E = logits.shape[1]
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_TOP_K):
        raise ValueError(f"{fn}: 1 to {MAX_TOP_K} of up to {MAX_EXPERTS} experts (got {k} of {E})")


def _choose(logits: torch.Tensor, k: int, renormalize: bool):
    dev = linear._device(logits)
    x = linear._pitched(logits, dev)
    T, E = x.shape
    index = torch.empty(T, k, dtype=torch.int64, device=dev)
    weights = torch.empty(T, k, dtype=torch.float32, device=dev)
    if T:
        nat.launch(dev, "mgq_top_k_softmax", x.data_ptr(), nat.dtype_code(x.dtype), T, E,
                   linear._ld(x), k, int(renormalize), index.data_ptr(), weights.data_ptr())
    return linear._home(index, logits), linear._home(weights, logits)


class _TopKSoftmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize):
        index, weights = _choose(logits, k, renormalize)
        ctx.renormalize = renormalize
        ctx.save_for_backward(logits, index)
        ctx.mark_non_differentiable(index)
        return index, weights

    @staticmethod
    def backward(ctx, _, dw):
        logits, index = ctx.saved_tensors
        return top_k_softmax_grad(dw, logits, index, ctx.renormalize), None, None


def top_k_softmax(logits: torch.Tensor, k: int,
                  renormalize: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """The router's choice: (index int64 [T, k], weights float32 [T, k]).

    The k largest logits of each row in descending order, the lower index first among
    equal ones (a NaN counts as the largest), and the softmax's weights of these: over
    the chosen (``renormalize``) or over all experts. logits: [T, E] float32, bf16 or
    f16, E up to 1024, k up to 16. Logits of -infinity mask experts out: they are never
    chosen, and where a row has fewer than k others the index is -1 (which ``route``,
    ``ExpertMLP.forward`` and ``.decode`` take as no expert) and the weight 0.

    The weights are differentiable in the logits (``top_k_softmax_grad``, which has no
    derivative itself). Nothing waits for the device.
    """
    k = operator.index(k)
    _check_logits("top_k_softmax", logits, k)
    if linear._tracked("top_k_softmax", logits):
        return _TopKSoftmax.apply(logits, k, bool(renormalize))
    return _choose(logits, k, renormalize)


def top_k_softmax_grad(dw: torch.Tensor, logits: torch.Tensor, index: torch.Tensor,
                       renormalize: bool = True) -> torch.Tensor:
    """Gradient of ``top_k_softmax``'s weights with respect to the logits: [T, E] of
    their type, computed in fp32 and rounded once. dw: [T, k], index: the choice."""
    fn = "top_k_softmax_grad"
    tracked = linear._tracked(fn, dw, logits)
    if index.dim() != 2 or not linear._integers(index):
        raise ValueError(f"{fn}: index must be integers [T, k] (got {tuple(index.shape)})")
    _check_logits(fn, logits, int(index.shape[1]))
    T, E = logits.shape
    k = index.shape[1]
    if index.shape[0] != T or dw.shape != index.shape or not dw.dtype.is_floating_point:
        raise ValueError(f"{fn}: dw and index must be {(T, k)} "
                         f"(got {tuple(dw.shape)} and {tuple(index.shape)})")
    dev = linear._device(logits, dw)
    x = linear._pitched(logits, dev)
    d, i = linear._dense(dw.float(), dev), linear._dense(index.to(torch.int64), dev)
    out = torch.empty(T, E, dtype=x.dtype, device=dev)
    if T:
        nat.launch(dev, "mgq_top_k_softmax_grad", d.data_ptr(), x.data_ptr(), nat.dtype_code(x.dtype),
                   T, E, linear._ld(x), i.data_ptr(), k, int(renormalize), out.data_ptr())
    out = linear._home(out, logits)
    return linear._NoGradient.apply(fn, out, dw, logits) if tracked else out


@dataclass
class Routing:
    """A batch's assignments in the experts' order."""

    offsets: torch.Tensor    # int32 [E + 1]: expert e owns entries offsets[e]:offsets[e + 1]
    row_index: torch.Tensor  # int32 [T * k]: the row each entry reads
    entry: torch.Tensor      # int64 [T * k]: where assignment (row, j) stands in the list


def route(top_k_index: torch.Tensor, num_experts: int) -> Routing:
    """The list that the grouped products take, from the router's choice
    ``top_k_index`` [T, k]. Assignments keep the rows' order inside an expert;
    ids outside [0, num_experts) belong to no expert and come last."""
    if top_k_index.dim() != 2 or top_k_index.dtype.is_floating_point:
        raise ValueError(f"route: top_k_index must be integers [T, k] (got {tuple(top_k_index.shape)})")
    T, k = top_k_index.shape
    e = top_k_index.reshape(-1).to(torch.int64)
    e = torch.where((e >= 0) & (e < num_experts), e, num_experts)
    e_sorted, order = torch.sort(e, stable=True)
    bounds = torch.arange(num_experts + 1, device=e.device)
    offsets = torch.searchsorted(e_sorted, bounds).to(torch.int32)
    entry = torch.empty_like(order)
    entry[order] = torch.arange(T * k, device=e.device)
    row_index = torch.div(order, max(k, 1), rounding_mode="floor").to(torch.int32)
    return Routing(offsets, row_index, entry)


class _DecodeWeights:
    """What ExpertMLP.decode passes of its weights. It keeps none of the layer's tensors
    alive; copies (of host weights, or of ones whose rows do not lie one after the other)
    are its own, and such a description serves one call only."""

    def __init__(self, cols, dtype, device, inner, up, down, given, passed):
        self.cols, self.dtype, self.device, self.inner = cols, dtype, device, inner
        self.type_code = nat.dtype_code(dtype)
        self.up, self.down = up, down
        self.up_ptr, self.down_ptr = ctypes.addressof(up), ctypes.addressof(down)
        self.in_place = [t.data_ptr() for t in passed] == [t.data_ptr() for t in given]
        self.copies = () if self.in_place else passed
        self.layout = [(weakref.ref(t), t.data_ptr(), t.dtype, t.shape, t.stride()) for t in given]
        self._sizes: dict[tuple[int, int], int] = {}

    def current(self, now) -> bool:
        """Whether the layer's tensors, `now`, are those described, where they were: one may
        have taken another's place on the layer, or in a list of them that stayed."""
        if len(now) != len(self.layout):
            return False
        for t, (old, ptr, dtype, shape, stride) in zip(now, self.layout):
            if (old() is not t or t.data_ptr() != ptr or t.dtype is not dtype or t.shape != shape
                    or t.stride() != stride):
                return False
        return True

    def workspace(self, T: int, k: int) -> int:
        try:
            return self._sizes[T, k]
        except KeyError:
            size = nat.load().mgq_experts_decode_workspace_size(T, k, self.cols, self.inner)
            self._sizes[T, k] = size
            return size


class ExpertMLP:
    """Experts gate_up [E, 2 I, H] and down [E, H, I] in one of the formats.

    ``gate_up`` and ``down`` are the weight itself (dense), a pair: packed words
    and E8M0 scale bytes (mxfp4, mxfp8), int8 weights and fp32 channel scales
    (int8), or packed words, scales and biases (affine), as linear.py takes them.
    """

    MODES = ("dense", "mxfp4", "mxfp8", "int8")  # one grid each
    GRID_MODES = ("affine",)                      # `bits` and a group size choose the grid

    _described: _DecodeWeights | None = None

    def __init__(self, gate_up, down, mode: str = "dense"):
        if mode not in self.MODES + self.GRID_MODES:
            raise ValueError(f"unsupported expert mode: {mode} "
                             f"({', '.join(self.MODES + self.GRID_MODES)})")
        self.mode = mode
        self.gate_up, self.down = gate_up, down
        first = gate_up if mode == "dense" else gate_up[0]
        if first.dim() != 3 or first.shape[1] % 2:
            raise ValueError(f"ExpertMLP: gate_up must be [E, 2 I, H] (got {tuple(first.shape)})")
        self.num_experts = int(first.shape[0])

    def __getstate__(self):
        # (addresses of this process's tensors: a copy describes its own)
        return {name: value for name, value in self.__dict__.items() if name != "_described"}

    @classmethod
    def from_weights(cls, gate_up: torch.Tensor, down: torch.Tensor, mode: str = "dense",
                     bits: int = 4, group_size: int = 64):
        """Weights [E, out, in] rounded to the nearest in `mode`, without
        calibration. ``bits`` and ``group_size`` are the affine grid's."""
        if mode == "dense":
            return cls(gate_up, down)
        return cls(*(cls._nearest(w, mode, bits, group_size) for w in (gate_up, down)), mode)

    @classmethod
    def from_codes(cls, gate_up, down, mode: str, bits: int | None = None):
        """The solver's results: (q uint8 [E, out, in], scale bytes [E, out, in /
        32]) of each parameter, as ``gptq.solve_gptq`` returns them first and
        second; affine codes of ``bits`` bits (4 unless given) with scales and
        biases, which it returns second and third."""
        if mode not in ("mxfp4", "mxfp8", "affine"):
            raise ValueError(f"not a grid of the solver: {mode}")
        default = grid.mode_defaults(mode)[1]
        if mode != "affine" and bits not in (None, default):
            raise ValueError(f"{mode} codes have {default} bits (got {bits})")
        given = 3 if mode == "affine" else 2
        if len(gate_up) != given or len(down) != given:
            raise ValueError(f"from_codes: {mode} weights are codes and scales"
                             + (" and biases" if given == 3 else "")
                             + f" (got {len(gate_up)} and {len(down)} tensors)")
        return cls(*((packing.pack_q(w[0], bits or default), *w[1:]) for w in (gate_up, down)), mode)

    @staticmethod
    def _nearest(w: torch.Tensor, mode: str, bits: int, group_size: int):
        if mode == "int8":
            return linear.quantize_rows_int8(w.detach())
        if mode == "affine":
            q, s, b, _ = grid.rtn_quantize(w, bits, group_size, storage_dtype=w.dtype)
            return packing.pack_q(q, bits), s, b
        q, s, _, _ = grid.rtn_quantize_mxfp(w, mode)
        return packing.pack_q(q, grid.mode_defaults(mode)[1]), s

    def _product(self, x, weight, offsets, row_index=None, cols=None):
        """x times a weight, whose rows have `cols` values (as many as x unless given)."""
        if self.mode == "dense":
            return linear.grouped_linear(x, weight, offsets, row_index, validate=False)
        if self.mode == "int8":
            q, s = linear.quantize_rows_int8(x)
            return linear.int8_linear(q, s, *weight, out_dtype=x.dtype, offsets=offsets,
                                      row_index=row_index, validate=False)
        if self.mode == "affine":
            bits = 32 * weight[0].shape[-1] // max(x.shape[1] if cols is None else cols, 1)
            return linear.affine_linear(x, *weight, bits, offsets, row_index, validate=False)
        return linear.mxfp_linear(x, *weight, self.mode, offsets, row_index, validate=False)

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                top_k_weights: torch.Tensor) -> torch.Tensor:
        """[T, H] -> [T, H]. The activation and the sum over a row's experts are
        formed in fp32 and rounded to the rows' type. Assignments to no expert add
        nothing, whatever their weight is."""
        T, k = top_k_index.shape
        r = route(top_k_index, self.num_experts)
        # (each weight's rows are as long as the other one says)
        up_rows, down_rows = ((w if self.mode == "dense" else w[0]).shape[1]
                              for w in (self.gate_up, self.down))
        gate, up = self._product(hidden_states, self.gate_up, r.offsets, r.row_index,
                                 down_rows).chunk(2, dim=-1)
        act = (F.silu(gate.float()) * up.float()).to(hidden_states.dtype)
        y = self._product(act, self.down, r.offsets, cols=up_rows // 2)
        y = y[r.entry].view(T, k, y.shape[1]).float()
        # (a row whose experts are all masked may come with weights of NaN)
        dropped = (r.entry >= r.offsets[-1]).view(T, k)
        weights = top_k_weights.float().masked_fill(dropped, 0.0)
        return (y * weights.unsqueeze(-1)).sum(1).to(hidden_states.dtype)

    __call__ = forward

    def _decode_weight(self, weight, out_rows: int, cols: int, dtype: torch.dtype,
                       dev: torch.device):
        """(nat.Weight, its tensors) for rows of `cols` of `dtype`."""
        fn, E = "ExpertMLP.decode", self.num_experts
        if self.mode == "dense":
            if weight.dtype != dtype:
                raise TypeError(f"{fn}: expects rows of the weights' type (got {dtype} and {weight.dtype})")
            if weight.shape != (E, out_rows, cols):
                raise AssertionError(f"{fn}: expects weights {(E, out_rows, cols)} "
                                     f"(got {tuple(weight.shape)})")
            w = linear._pitched(weight, dev)
            return nat.Weight(w.data_ptr(), None, None, linear._ld(w), w.stride(0), 0,
                              nat.WEIGHT_DENSE, 0), (w,)
        bits = 32 * weight[0].shape[-1] // max(cols, 1)
        if weight[0].shape[:-1] != (E, out_rows):
            raise AssertionError(f"{fn}: expects weights {(E, out_rows, cols)} "
                                 f"(words {tuple(weight[0].shape)})")
        params = 0
        if self.mode == "affine":
            packed, scales, biases = weight
            group = linear.affine_dims(fn, cols, bits, packed.shape, packed.dtype, scales.shape,
                                       scales.dtype, biases.shape, biases.dtype, True)[2]
            code = {2: nat.WEIGHT_AFFINE2, 4: nat.WEIGHT_AFFINE4, 8: nat.WEIGHT_AFFINE8}[bits]
            params = nat.dtype_code(scales.dtype)
        else:
            linear.check_mxfp(fn, cols, self.mode, *weight)
            group, code = 32, nat.WEIGHT_MXFP4 if self.mode == "mxfp4" else nat.WEIGHT_MXFP8
        t = tuple(linear._dense(w, dev) for w in weight)
        return nat.Weight(t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr() if len(t) > 2 else None,
                          0, 0, group, code, params), t

    def _tensors(self) -> tuple[torch.Tensor, ...]:
        """Those of gate_up, then those of down."""
        gate_up, down = self.gate_up, self.down
        return (gate_up, down) if self.mode == "dense" else (*gate_up, *down)

    def _decode_weights(self, cols: int, dtype: torch.dtype, dev: torch.device, given=None):
        """Both weights as mgq_experts_decode takes them: described once, and again for
        other rows or when a tensor is no longer the one described. The caller holds
        `given` (``_tensors``) until they are launched: the description does not."""
        given = self._tensors() if given is None else given
        d = self._described
        if (d is not None and d.cols == cols and d.dtype is dtype and d.device == dev
                and d.current(given)):
            return d
        # (before new copies are made, and if an error follows)
        self._described = None
        half = len(given) // 2
        gate_up, down = given if self.mode == "dense" else (given[:half], given[half:])
        inner = given[0].shape[1] // 2
        up, up_tensors = self._decode_weight(gate_up, 2 * inner, cols, dtype, dev)
        dn, dn_tensors = self._decode_weight(down, cols, inner, dtype, dev)
        d = _DecodeWeights(cols, dtype, dev, inner, up, dn, given, up_tensors + dn_tensors)
        self._described = d if d.in_place else None
        return d

    def decode(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
               top_k_weights: torch.Tensor) -> torch.Tensor:
        """``forward`` for up to 64 rows with up to 16 experts each, in two launches that
        read the weights of the rows' experts once. [T, H] -> [T, H].

        For up to 8 rows the activation keeps twice the bits of the rows' type, for more it
        is rounded to it; everything else is fp32 until the result is rounded once
        (``forward`` also rounds between its products, so the two agree within the type's
        precision only). Assignments to no expert add nothing. The
        order of the sums depends on the sizes and the routing alone. int8 experts, whose
        rows are quantized for each product, have ``forward`` only. Not differentiable.
        """
        fn = "ExpertMLP.decode"
        if self.mode == "int8":
            raise ValueError(f"{fn}: int8 experts are not supported, use forward")
        x = hidden_states
        given = self._tensors()
        if self.mode == "dense":
            floats = given
        else:
            floats = (*given[1:3], *given[4:]) if self.mode == "affine" else ()
        tracked = linear._tracked(fn, x, top_k_weights, *floats)
        if x.dtype not in linear._HALF or (self.mode[:2] == "mx" and x.dtype is not torch.bfloat16):
            raise TypeError(f"{fn}: expects bfloat16 rows, or float16 ones without MXFP weights "
                            f"(got {x.dtype})")
        linear._rows2(fn, "hidden_states", x)
        T, H = x.shape
        if top_k_index.dim() != 2 or top_k_index.shape[0] != T or not linear._integers(top_k_index):
            raise ValueError(f"{fn}: top_k_index must be integers [{T}, k] "
                             f"(got {tuple(top_k_index.shape)})")
        k = top_k_index.shape[1]
        if top_k_weights.shape != top_k_index.shape or not top_k_weights.dtype.is_floating_point:
            raise ValueError(f"{fn}: top_k_weights must be numbers {(T, k)} "
                             f"(got {tuple(top_k_weights.shape)})")
        if T > 64 or not 1 <= k <= 16:
            raise ValueError(f"{fn}: up to 64 rows with 1 to 16 experts each (got {(T, k)}); "
                             "forward takes any number")
        dev = linear._device(x, *given)
        d = self._decode_weights(H, x.dtype, dev, given)
        xd = linear._pitched(x, dev)
        index = top_k_index
        if index.dtype is not torch.int64:
            index = linear._int32(index)
        index = linear._dense(index, dev)
        weights = top_k_weights if top_k_weights.dtype is torch.float32 else top_k_weights.float()
        weights = linear._dense(weights, dev)
        out = torch.empty(T, H, dtype=x.dtype, device=dev)
        if T and H:
            size = d.workspace(T, k)
            ws = torch.empty(size, dtype=torch.uint8, device=dev)
            nat.launch(dev, "mgq_experts_decode", xd.data_ptr(), d.type_code, T, linear._ld(xd),
                       index.data_ptr(), 64 if index.dtype is torch.int64 else 32, weights.data_ptr(),
                       k, self.num_experts, H, d.inner, d.up_ptr, d.down_ptr, out.data_ptr(),
                       ws.data_ptr(), size)
        out = linear._home(out, x)
        return linear._NoGradient.apply(fn, out, x, top_k_weights, *floats) if tracked else out
