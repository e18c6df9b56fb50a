"""Fit a gated residual trunk to the manufactured Poisson solution: the trunk's operators and the
multi-tensor AdamW step as they are used together, the whole iteration in one CUDA graph.

    python -m fused_hoad.fit_trunk [--points 65536] [--width 64] [--hidden 256] [--blocks 4]
                                   [--steps 300] [--dtype float32|bfloat16] [--state-bits 32|8]

Prints the error before and after and the time of a step. Needs a B200.
"""

from __future__ import annotations

import argparse

import torch
from torch import Tensor

from fused_hoad.blocks import GatedResidualTrunk
from fused_hoad.optim import AdamW
from fused_hoad.problem import manufactured_solution, uniform_points
from fused_hoad.training import cuda_graph_step


def fit_trunk(
    *,
    points: int = 65536,
    width: int = 64,
    hidden: int = 256,
    blocks: int = 4,
    steps: int = 300,
    lr: float = 2e-3,
    dtype: torch.dtype = torch.float32,
    state_bits: int = 32,
    seed: int = 0,
) -> tuple[GatedResidualTrunk, float, float, float]:
    """``(trunk, mean squared error before, after, milliseconds a step)`` of ``steps`` AdamW
    steps (at least 3, which warm up the graph) on uniform points."""
    if steps < 3:
        raise ValueError("steps must be at least 3")
    torch.manual_seed(seed)
    model = GatedResidualTrunk(2, width, hidden, blocks).to("cuda", dtype)
    x = uniform_points(points).cuda()
    want = manufactured_solution(x)
    inputs = x.to(dtype)

    def loss_fn() -> Tensor:
        return (model(inputs).float() - want).square().mean()

    with torch.no_grad():
        before = float(loss_fn())
    step = cuda_graph_step(loss_fn, AdamW(model.parameters(), lr=lr, state_bits=state_bits))
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(steps - 3):
        step()
    end.record()
    end.synchronize()
    with torch.no_grad():
        after = float(loss_fn())
    return model, before, after, start.elapsed_time(end) / max(1, steps - 3)


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("points", 65536), ("width", 64), ("hidden", 256), ("blocks", 4),
                          ("steps", 300)):
        parser.add_argument(f"--{name}", type=int, default=default)
    parser.add_argument("--lr", type=float, default=2e-3)
    parser.add_argument("--dtype", choices=("float32", "bfloat16"), default="float32")
    parser.add_argument("--state-bits", type=int, choices=(32, 8), default=32)
    args = vars(parser.parse_args())
    args["dtype"] = getattr(torch, args["dtype"])
    _, before, after, ms = fit_trunk(**args)
    print(f"mean squared error {before:.3e} -> {after:.3e}, {ms:.3f} ms a step")


if __name__ == "__main__":
    main()
