"""The operators of deep gated residual trunks, and a small trunk built from them.

``gated_feed_forward`` and ``residual_norm`` are differentiable and run on the sm_100a kernels
of the compiled extension, forward and backward; ``rms_norm`` is the entry norm of a stack.
float32 and bfloat16. There is no CPU or PyTorch fallback. The reference's networks are plain
``Linear, activation`` stacks (its ``src/fused_hoad/models.py:15-26``); these blocks are what a
deeper trunk for the same problems is made of.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from fused_hoad._extension import load_extension
from fused_hoad.problem import ACTIVATIONS


def gated_feed_forward(
    x: Tensor,
    w_gate: Tensor,
    w_up: Tensor,
    w_down: Tensor,
    b_gate: Tensor | None = None,
    b_up: Tensor | None = None,
    b_down: Tensor | None = None,
    activation: str = "silu",
) -> Tensor:
    """``(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down``, ``[..., out]``.

    ``x`` is ``[..., width]``, ``w_gate`` and ``w_up`` ``[hidden, width]``, ``w_down``
    ``[out, hidden]``, all float32 or all bfloat16; ``activation`` ``"silu"`` or ``"tanh"``.
    Rows may have any stride (a slice of a larger tensor is not copied). Sums are held in 32
    bits. In bfloat16 the gated product, and in the backward the gradients of the two
    projections, are rounded to bfloat16 as operands of the next matrix product. Differentiable
    once, in reverse (``create_graph`` and forward-mode tangents raise).
    """
    return load_extension().gated_feed_forward(
        x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation
    )


def _norm(residual, branch, pre_weight, post_weight, gate, residual_scale, eps):
    tensor = isinstance(residual_scale, Tensor)
    return load_extension().residual_norm(
        residual, branch, pre_weight, post_weight, gate, residual_scale if tensor else None,
        1.0 if tensor else float(residual_scale), eps
    )


def residual_norm(
    residual: Tensor,
    branch: Tensor,
    pre_weight: Tensor,
    post_weight: Tensor | None = None,
    gate: Tensor | None = None,
    residual_scale: Tensor | float = 1.0,
    eps: float = 1e-6,
) -> tuple[Tensor, Tensor]:
    """The norms after one block and before the next, with the gate and the residual scale.

    ``total = residual_scale * residual + gate * (rms(branch) * post_weight)`` and
    ``normed = rms(total) * pre_weight``, ``rms(v) = v / sqrt(mean(v^2) + eps)`` over the last
    dimension; returns ``(total, normed)``: the residual stream and the next block's input.
    Without ``post_weight`` the branch is not normed; without ``gate`` it is not gated.

    ``branch`` has the shape of ``residual``. ``gate`` has shape ``[width]`` (a learned gate per
    channel), the shape of ``residual``, or that shape with ones in its last leading dimensions
    (``[batch, 1, width]``: a gate for each sample). ``residual_scale`` is a number or a float32
    tensor with one element, which then gets a gradient. ``residual`` and ``total`` may be
    float32 where everything else is bfloat16. Sums and norms are held in 32 bits, and the
    norm is that of the unrounded total. Differentiable once, in reverse.
    """
    if branch is None:
        raise ValueError("residual_norm needs a branch; rms_norm is the norm alone")
    total, normed = _norm(residual, branch, pre_weight, post_weight, gate, residual_scale, eps)
    return total, normed


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in the weight's type."""
    return _norm(x, None, weight, None, None, 1.0, eps)[0]


class _Float32Parameters(nn.ParameterList):
    """Parameters that stay float32 when their module's type is changed."""

    def _apply(self, fn, recurse=True):
        def move(t: Tensor) -> Tensor:
            moved = fn(t)
            return moved if moved.dtype == t.dtype else t.to(moved.device)

        return super()._apply(move, recurse)


class GatedResidualTrunk(nn.Module):
    """A deep trunk for point-wise problems: ``Linear``, ``blocks`` gated feed-forward blocks
    with norms before and after, a gate per channel and a learned residual scale, a last norm
    and a ``Linear``. ``[..., input_dim] -> [..., output_dim]``, float32 or bfloat16.

    The gates start at ``gate_init``, so that a deep trunk starts near its first layer. The residual
    scales stay float32 whatever the trunk's type: they stay near 1, where bfloat16's steps are
    larger than an optimizer's.
    """

    def __init__(
        self,
        input_dim: int = 2,
        width: int = 64,
        hidden: int = 256,
        blocks: int = 4,
        output_dim: int = 1,
        *,
        activation: str = "tanh",
        bias: bool = True,
        gate_init: float = 0.5,
        eps: float = 1e-6,
    ) -> None:
        super().__init__()
        for name, value in (("input_dim", input_dim), ("width", width), ("hidden", hidden),
                            ("blocks", blocks), ("output_dim", output_dim)):
            if value < 1:
                raise ValueError(f"{name} must be positive")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
        self.activation, self.eps = activation, float(eps)
        self.encode = nn.Linear(input_dim, width)
        self.entry = nn.Parameter(torch.ones(width))
        self.gate = nn.ModuleList(nn.Linear(width, hidden, bias=bias) for _ in range(blocks))
        self.up = nn.ModuleList(nn.Linear(width, hidden, bias=bias) for _ in range(blocks))
        self.down = nn.ModuleList(nn.Linear(hidden, width, bias=bias) for _ in range(blocks))
        self.post = nn.ParameterList(torch.ones(width) for _ in range(blocks))
        self.channel_gate = nn.ParameterList(torch.full((width,), gate_init) for _ in range(blocks))
        self.pre = nn.ParameterList(torch.ones(width) for _ in range(blocks))
        self.scale = _Float32Parameters(torch.ones(1) for _ in range(blocks))
        self.decode = nn.Linear(width, output_dim)

    def forward(self, x: Tensor) -> Tensor:
        stream = self.encode(x)
        normed = rms_norm(stream, self.entry, self.eps)
        for k in range(len(self.gate)):
            branch = gated_feed_forward(
                normed, self.gate[k].weight, self.up[k].weight, self.down[k].weight,
                self.gate[k].bias, self.up[k].bias, self.down[k].bias, self.activation,
            )
            stream, normed = residual_norm(
                stream, branch, self.pre[k], self.post[k], self.channel_gate[k], self.scale[k],
                self.eps,
            )
        return self.decode(normed)
