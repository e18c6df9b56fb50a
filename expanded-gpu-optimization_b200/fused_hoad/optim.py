"""AdamW over many tensors in one kernel, with 32-bit or 8-bit states.

``adamw_step`` is the step on lists of tensors; ``AdamW`` is the optimizer around it
(``torch.optim.AdamW``'s arguments and state names). The step counter lives on the device, so a
step can be captured in a CUDA graph (:func:`fused_hoad.cuda_graph_step`). ``PoissonTrainer``
keeps its own Adam inside its update kernel; this one is for models of many parameters.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch
from torch import Tensor

from fused_hoad._extension import load_extension

# Consecutive values that share one scale of an 8-bit state (FHB_ADAMW_BLOCK of the C ABI).
ADAMW_BLOCK = 256


def adamw_step(
    params: Sequence[Tensor],
    grads: Sequence[Tensor],
    exp_avgs: Sequence[Tensor],
    exp_avg_sqs: Sequence[Tensor],
    step: Tensor,
    *,
    lr: float = 1e-3,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    exp_avg_scales: Sequence[Tensor] | None = None,
    exp_avg_sq_scales: Sequence[Tensor] | None = None,
) -> None:
    """One AdamW step, in place, on every tensor of ``params`` (float32 or bfloat16 each).

    32-bit states: ``exp_avgs`` and ``exp_avg_sqs`` are float32. 8-bit states: they are
    ``torch.float8_e4m3fn`` codes of m and of sqrt(v) in units of a float32 scale for each
    ``ADAMW_BLOCK`` consecutive values, and the two lists of scales are given (see
    :func:`decode_states`). ``step`` is a CUDA int64 tensor with the number of steps taken so
    far; the call advances it on the stream. All tensors are contiguous and on one device.
    """
    load_extension().adamw_step(
        list(params), list(grads), list(exp_avgs), list(exp_avg_sqs),
        None if exp_avg_scales is None else list(exp_avg_scales),
        None if exp_avg_sq_scales is None else list(exp_avg_sq_scales),
        step, lr, betas[0], betas[1], eps, weight_decay,
    )


def decode_states(
    exp_avg: Tensor, exp_avg_sq: Tensor, exp_avg_scale: Tensor, exp_avg_sq_scale: Tensor
) -> tuple[Tensor, Tensor]:
    """The float32 moments ``(m, v)`` that a parameter's 8-bit states stand for."""

    def values(codes: Tensor, scale: Tensor) -> Tensor:
        spread = scale.repeat_interleave(ADAMW_BLOCK)[: codes.numel()]
        return codes.float() * spread.view(codes.shape)

    return values(exp_avg, exp_avg_scale), values(exp_avg_sq, exp_avg_sq_scale).square()


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on the multi-tensor kernel: one launch for many parameters.

    ``state_bits`` 32 keeps float32 moments (8 bytes a parameter), 8 keeps e4m3 codes with one
    scale for each 256 values (2.03 bytes a parameter). Parameters are float32 or bfloat16,
    contiguous, and all on one CUDA device; those without a gradient are skipped. Every parameter
    counts its own steps, on the device; those of a group that have had their gradients in the
    same steps share a counter and a launch. A step with new parameters, or with fewer than share
    a counter, is taken once before one like it is captured in a CUDA graph.
    """

    def __init__(
        self,
        params,
        lr: float = 1e-3,
        betas: tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 1e-2,
        *,
        state_bits: int = 32,
    ) -> None:
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        if not lr >= 0.0:
            raise ValueError("lr must be >= 0")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError("betas must be in [0, 1)")
        if not eps >= 0.0:
            raise ValueError("eps must be >= 0")
        if not weight_decay >= 0.0:
            raise ValueError("weight_decay must be >= 0")
        defaults = dict(lr=float(lr), betas=(float(betas[0]), float(betas[1])), eps=float(eps),
                        weight_decay=float(weight_decay), state_bits=state_bits, capturable=True)
        super().__init__(params, defaults)

    def _new_state(self, p: Tensor, state_bits: int, step: Tensor) -> dict:
        state = self.state[p]
        state["step"] = step
        if state_bits == 32:
            state["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            state["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            blocks = -(-p.numel() // ADAMW_BLOCK)
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(p, dtype=torch.float8_e4m3fn)
                state[name + "_scale"] = torch.zeros(blocks, device=p.device)
        return state

    def _by_counter(self, group: dict) -> list[tuple[list[Tensor], list[Tensor], list[dict]]]:
        """(parameters, gradients, states) for each step counter that parameters with a gradient
        share. Those that share one with a parameter that has none now get one of their own."""
        shared: dict[int, tuple[list[Tensor], list[Tensor], list[dict]]] = {}
        idle = set()
        fresh = None
        for p in group["params"]:
            state, grad = self.state.get(p), p.grad
            if grad is None:
                if state:
                    idle.add(id(state["step"]))
                continue
            if not state:
                if fresh is None:
                    _refuse_capture(p)
                    fresh = torch.zeros(1, dtype=torch.int64, device=p.device)
                state = self._new_state(p, group["state_bits"], fresh)
            key = id(state["step"])
            if key not in shared:
                shared[key] = ([], [], [])
            params, grads, states = shared[key]
            params.append(p)
            grads.append(grad.contiguous())
            states.append(state)
        for key in idle & shared.keys():
            params, _, states = shared[key]
            _refuse_capture(params[0])
            own = states[0]["step"].clone()
            for state in states:
                state["step"] = own
        return list(shared.values())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for params, grads, states in self._by_counter(group):
                scales = {}
                if group["state_bits"] == 8:
                    scales = {"exp_avg_scales": [s["exp_avg_scale"] for s in states],
                              "exp_avg_sq_scales": [s["exp_avg_sq_scale"] for s in states]}
                adamw_step(
                    params, grads, [s["exp_avg"] for s in states],
                    [s["exp_avg_sq"] for s in states], states[0]["step"], lr=group["lr"],
                    betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                    **scales,
                )
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As ``torch.optim.Optimizer.load_state_dict``; the moments keep their own types (that
        method would cast floating-point state to the parameter's type). Takes the states of
        ``torch.optim.AdamW`` too (without ``amsgrad`` and ``maximize``), and those with one
        counter for a group. Waits for the device to read the counters."""
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("amsgrad and maximize are not supported")
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        for group, saved_group in zip(self.param_groups, state_dict["param_groups"]):
            of_group = group.pop("step", None)
            group.setdefault("state_bits", 32)
            counters: dict[int, Tensor] = {}
            for p, index in zip(group["params"], saved_group["params"]):
                if not saved.get(index):
                    continue
                state = {}
                for name, value in saved[index].items():
                    if isinstance(value, Tensor):
                        moment = group["state_bits"] == 32 and name in ("exp_avg", "exp_avg_sq")
                        value = value.to(p.device, torch.float32 if moment else None, copy=True)
                    state[name] = value
                count = int(state.get("step", of_group))
                if count not in counters:
                    counters[count] = torch.full((1,), count, dtype=torch.int64, device=p.device)
                state["step"] = counters[count]
                self.state[p] = state


def _refuse_capture(p: Tensor) -> None:
    """What is made while a graph is captured would be made anew by every replay."""
    if p.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the optimizer's states are made by a step before the captured one")
