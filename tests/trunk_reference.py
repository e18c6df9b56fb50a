"""Plain 64-bit forms of the gated residual trunk's operators, and how far the kernels may be.

An error is measured against the *size* of the value: what it would be if its terms had not
cancelled (for a sum, the root of the sum of their squares, since their roundings have random
signs; for a difference, the sum of the magnitudes), or the value itself where that is larger.
Tolerances are relative to it and follow from the number formats:

* float32: a sum of K terms rounded K times at 2^-24 with random signs is off by about
  sqrt(K) 2^-24; two such sums in a row and their elementwise steps stay below
  (8 + 2 sqrt(K)) 2^-24.
* bfloat16: every rounding is at most 2^-9. An output has its own, and at most one operand
  rounded before it (h, or the gradients of the two projections): 3 * 2^-9 leaves one more for
  the 32-bit parts.
* in the 2-norm of the tensor; single values: 8 times that, against the larger of the value's
  size and the tensor's rms size.
"""

from __future__ import annotations

import math

import torch


def tolerance(dtype: torch.dtype, terms: int) -> float:
    if dtype == torch.bfloat16:
        return 3 * 2.0**-9
    return (8 + 2 * math.sqrt(terms)) * 2.0**-24


def assert_near(got, want, tol: float, what: str, size=None) -> None:
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.numel():
        return
    got, want = got.detach().double(), want.detach().double()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    size = want.abs() if size is None else torch.maximum(want.abs(), size.detach().double())
    rms = size.square().mean().sqrt()
    off = (got - want).abs()
    if not rms > 0:
        assert not off.any(), f"{what}: not zero"
        return
    norm = float(off.square().mean().sqrt() / rms)
    assert norm <= tol, f"{what}: {norm:.3e} off in norm, {tol:.3e} allowed"
    single = float((off / torch.maximum(size, rms)).max())
    assert single <= 8 * tol, f"{what}: a value {single:.3e} off, {8 * tol:.3e} allowed"


def ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu"):
    g, u = x @ w_gate.T, x @ w_up.T
    if b_gate is not None:
        g = g + b_gate
    if b_up is not None:
        u = u + b_up
    a = torch.tanh(g) if activation == "tanh" else g * torch.sigmoid(g)
    y = (a * u) @ w_down.T
    return y if b_down is None else y + b_down


def ffn_gradients(grad, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
    """By the formulas, for rows of x: dx, dWg, dWu, dWd, dbg, dbu, dbd."""
    g, u = x @ w_gate.T, x @ w_up.T
    g = g if b_gate is None else g + b_gate
    u = u if b_up is None else u + b_up
    if activation == "tanh":
        a = torch.tanh(g)
        slope = 1 - a * a
    else:
        s = torch.sigmoid(g)
        a, slope = g * s, s * (1 + g * (1 - s))
    dh = grad @ w_down
    du, dg = dh * a, dh * u * slope
    return (dg @ w_gate + du @ w_up, dg.T @ x, du.T @ x, grad.T @ (a * u), dg.sum(0), du.sum(0),
            grad.sum(0))


def ffn_sizes(grad, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation):
    """The sizes of y and of the seven gradients."""
    def root(a, b):
        return (a.square() @ b.square()).sqrt()

    g, u = x @ w_gate.T, x @ w_up.T
    g = g if b_gate is None else g + b_gate
    u = u if b_up is None else u + b_up
    if activation == "tanh":
        a = torch.tanh(g)
        slope = 1 - a * a
    else:
        s = torch.sigmoid(g)
        a, slope = g * s, s * (1 + g * (1 - s))
    dh = root(grad, w_down)
    du, dg = dh * a.abs(), dh * (u * slope).abs()
    y = root(a * u, w_down.T)
    if b_down is not None:
        y = y + b_down.abs()
    return y, ((root(dg, w_gate).square() + root(du, w_up).square()).sqrt(), root(dg.T, x),
               root(du.T, x), root(grad.T, a * u), dg.norm(dim=0), du.norm(dim=0),
               grad.norm(dim=0))


def norm(residual, branch, pre_weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    def rms(v):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)

    total = scale * residual
    if branch is not None:
        z = branch if post_weight is None else rms(branch) * post_weight
        total = total + (z if gate is None else gate * z)
    return total, rms(total) * pre_weight


def norm_sizes(residual, branch, pre_weight, post_weight, gate, scale, d_total, d_normed,
               eps=1e-6):
    """The sizes of (total, normed) and of the gradients of the six arguments (None where an
    argument is). A total that nearly cancels has a larger relative error, and with it
    everything that is divided by its norm: `worse` is by how much."""
    def mean(v):
        return v.mean(-1, keepdim=True)

    inv_b = 1 / torch.sqrt(mean(branch.square()) + eps)
    b_hat = branch * inv_b
    z = branch if post_weight is None else b_hat * post_weight
    c = torch.ones_like(z) if gate is None else gate.expand_as(z)
    total = scale * residual + c * z
    s_total = (scale * residual).abs() + (c * z).abs()
    root = torch.sqrt(mean(total.square()) + eps)
    worse = torch.sqrt(mean(s_total.square()) + eps) / root
    t_hat = total / root
    s_hat = worse * t_hat.abs() + s_total / root
    q = (d_normed * pre_weight).abs()
    s_dt = d_total.abs() + worse / root * (q + s_hat * mean(q * s_hat))
    rows = tuple(range(total.dim() - 1))

    def sum_like(v, like):  # root of the sum of squares over the dimensions that `like` lacks
        v = v.square()
        if like.dim() < v.dim():
            v = v.sum(tuple(range(v.dim() - like.dim())))
        for d in range(like.dim()):
            if like.shape[d] == 1 and v.shape[d] != 1:
                v = v.sum(d, keepdim=True)
        return v.sqrt()

    s_z = s_dt * c.abs()
    s_branch = s_z
    if post_weight is not None:
        p = s_z * post_weight.abs()
        s_branch = inv_b * (p + b_hat.abs() * mean(p * b_hat.abs()))
    return (s_total, s_hat * pre_weight.abs()), (
        abs(scale) * s_dt, s_branch, sum_like(d_normed * s_hat, pre_weight),
        None if post_weight is None else sum_like(s_z * b_hat, post_weight),
        None if gate is None else sum_like(s_dt * z, gate),
        (s_dt * residual).norm().reshape(1))
