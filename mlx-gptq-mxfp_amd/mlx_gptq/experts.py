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
* ``"int8"``: 8-bit weights with a scale for each output channel, rows quantized
  to 8 bits on the way into each product.

Only dense experts are differentiable; in the other formats a backward that reaches
the rows raises.

No call waits for the device: the routing stays there.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import grid, linear, packing


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


class ExpertMLP:
    """Experts gate_up [E, 2 I, H] and down [E, H, I] in one of the formats.

    ``gate_up`` and ``down`` are the weight itself (dense) or a pair: packed words
    and E8M0 scale bytes (mxfp4, mxfp8), int8 weights and fp32 channel scales
    (int8), as linear.py takes them.
    """

    MODES = ("dense", "mxfp4", "mxfp8", "int8")

    def __init__(self, gate_up, down, mode: str = "dense"):
        if mode not in self.MODES:
            raise ValueError(f"unsupported expert mode: {mode} ({', '.join(self.MODES)})")
        self.mode = mode
        self.gate_up, self.down = gate_up, down
        first = gate_up if mode == "dense" else gate_up[0]
        if first.dim() != 3 or first.shape[1] % 2:
            raise ValueError(f"ExpertMLP: gate_up must be [E, 2 I, H] (got {tuple(first.shape)})")
        self.num_experts = int(first.shape[0])

    @classmethod
    def from_weights(cls, gate_up: torch.Tensor, down: torch.Tensor, mode: str = "dense"):
        """Weights [E, out, in] rounded to the nearest in `mode`, without
        calibration."""
        if mode == "dense":
            return cls(gate_up, down)
        return cls(cls._nearest(gate_up, mode), cls._nearest(down, mode), mode)

    @classmethod
    def from_codes(cls, gate_up, down, mode: str):
        """The solver's results: (q uint8 [E, out, in], scale bytes [E, out, in /
        32]) of each parameter, as ``gptq.solve_gptq`` returns them first and
        second."""
        if mode not in ("mxfp4", "mxfp8"):
            raise ValueError(f"not a microscaling mode: {mode}")
        bits = grid.mode_defaults(mode)[1]
        return cls(*((packing.pack_q(q, bits), s) for q, s in (gate_up, down)), mode)

    @staticmethod
    def _nearest(w: torch.Tensor, mode: str):
        if mode == "int8":
            return linear.quantize_rows_int8(w.detach())
        q, s, _, _ = grid.rtn_quantize_mxfp(w, mode)
        return packing.pack_q(q, grid.mode_defaults(mode)[1]), s

    def _product(self, x, weight, offsets, row_index=None):
        if self.mode == "dense":
            return linear.grouped_linear(x, weight, offsets, row_index, validate=False)
        if self.mode == "int8":
            q, s = linear.quantize_rows_int8(x)
            return linear.int8_linear(q, s, *weight, out_dtype=x.dtype, offsets=offsets,
                                      row_index=row_index, validate=False)
        return linear.mxfp_linear(x, *weight, self.mode, offsets, row_index, validate=False)

    def forward(self, hidden_states: torch.Tensor, top_k_index: torch.Tensor,
                top_k_weights: torch.Tensor) -> torch.Tensor:
        """[T, H] -> [T, H]. The activation and the sum over a row's experts are
        formed in fp32 and rounded to the rows' type. Assignments to no expert add
        nothing, whatever their weight is."""
        T, k = top_k_index.shape
        r = route(top_k_index, self.num_experts)
        gate, up = self._product(hidden_states, self.gate_up, r.offsets, r.row_index).chunk(2, dim=-1)
        act = (F.silu(gate.float()) * up.float()).to(hidden_states.dtype)
        y = self._product(act, self.down, r.offsets)
        y = y[r.entry].view(T, k, y.shape[1]).float()
        # (a row whose experts are all masked may come with weights of NaN)
        dropped = (r.entry >= r.offsets[-1]).view(T, k)
        weights = top_k_weights.float().masked_fill(dropped, 0.0)
        return (y * weights.unsqueeze(-1)).sum(1).to(hidden_states.dtype)

    __call__ = forward
