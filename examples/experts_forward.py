"""A routed layer from calibration to its quantized forward.

Captures the inputs of a fused-expert module, solves its two parameters with
GPTQ on the MXFP4 grid, and runs the module's forward on the packed codes, for a
single token in two launches; beside it the same forward with dense, MXFP8, affine
and int8 weights rounded to the nearest, and one fine-tuning step of the dense
experts. The router's choice comes with its gradient. Random weights and rows.

    python examples/experts_forward.py [--tokens 512] [--device cuda:0]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "mlx-gptq-mxfp_amd"))

from mlx_gptq import capture, gptq, grid  # noqa: E402
from mlx_gptq.experts import ExpertMLP, route, top_k_softmax  # noqa: E402


def relative(y: torch.Tensor, ref: torch.Tensor) -> float:
    return float((y.float() - ref.float()).norm() / ref.float().norm())


def main(argv=None) -> dict[str, float]:
    ap = argparse.ArgumentParser(description=__doc__)
    ap.add_argument("--experts", type=int, default=16)
    ap.add_argument("--hidden", type=int, default=512)
    ap.add_argument("--inter", type=int, default=256)
    ap.add_argument("--tokens", type=int, default=512)
    ap.add_argument("--top-k", type=int, default=4)
    ap.add_argument("--device", default="cuda:0")
    args = ap.parse_args(argv)
    E, H, I, T, k = args.experts, args.hidden, args.inter, args.tokens, args.top_k
    dev = torch.device(args.device)
    g = torch.Generator().manual_seed(3)

    def rand(*shape, scale):
        return (torch.randn(*shape, generator=g) * scale).to(dev, torch.bfloat16)

    gate_up, down = rand(E, 2 * I, H, scale=H**-0.5), rand(E, H, I, scale=I**-0.5)
    x = rand(T, H, scale=1.0)
    score = torch.randn(T, E, generator=g).to(dev)
    index, weights = top_k_softmax(score, k, renormalize=False)

    dense = ExpertMLP(gate_up, down)
    y = dense(x, index, weights)

    # calibration: the block input with its routing, and the down inputs as the
    # dense forward makes them
    r = route(index, E)
    inputs = capture.RoutedStash("gate_up", H, E)
    inputs.add_routed(x, index)
    gate, up = dense._product(x, gate_up, r.offsets, r.row_index).chunk(2, dim=-1)
    act = (F.silu(gate.float()) * up.float()).to(x.dtype)
    codes = []
    for w, hess in ((gate_up, inputs.hessians()), (down, capture.grouped_hessian(act, r.offsets))):
        q, s, _, _, _ = gptq.solve_gptq(w, hess, 4, 32, mode="mxfp4")
        codes.append((q, s))

    errors = {"mxfp4 solved": relative(ExpertMLP.from_codes(*codes, "mxfp4")(x, index, weights), y)}
    for mode in ("mxfp4", "mxfp8", "int8", "affine"):
        errors[f"{mode} nearest"] = relative(
            ExpertMLP.from_weights(gate_up, down, mode)(x, index, weights), y)
        if mode in ("mxfp4", "mxfp8"):  # of the weights themselves
            errors[f"{mode} weights"] = max(
                relative(grid.rtn_quantize_mxfp(w, mode)[3], w) for w in (gate_up, down))
    one = ExpertMLP.from_codes(*codes, "mxfp4").decode(x[:1], index[:1], weights[:1])  # a single token
    errors["single token"] = relative(one, y[:1])
    for name, e in errors.items():
        print(f"{name:16s} relative error {e:.4f}")

    # one step of fine-tuning: both gradients through the grouped products, into
    # fp32 master weights
    params = [gate_up.float().requires_grad_(), down.float().requires_grad_()]
    target = 1.5 * y.float()
    losses = []
    for _ in range(2):
        out = ExpertMLP(*(p.to(torch.bfloat16) for p in params))(x, index, weights)
        loss = (out.float() - target).square().mean()
        losses.append(float(loss.detach()))
        loss.backward()
        with torch.no_grad():
            for p in params:
                p -= 0.002 * p.grad * (p.norm() / p.grad.norm())
                p.grad = None
    print(f"loss {losses[0]:.6f} -> {losses[1]:.6f}")
    errors["loss before"], errors["loss after"] = losses
    return errors


if __name__ == "__main__":
    main()
