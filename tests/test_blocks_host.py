"""Refusals of the gated residual trunk's operators, which need no GPU, and the 64-bit forms
that the GPU tests compare with, checked against differences."""

from __future__ import annotations

import ctypes

import pytest
import torch

import fused_hoad
import trunk_reference
from fused_hoad import _native

GOOD, BAD = 4096, 4097  # stand-in addresses: never dereferenced, the checks return first


def ffn_problem(**change):
    fields = dict(tokens=4, width=8, hidden=16, out_width=8, dtype=0, activation=1, x=GOOD,
                  w_gate=GOOD, w_up=GOOD, w_down=GOOD, x_stride=8, w_gate_stride=8,
                  w_up_stride=8, w_down_stride=16)
    return _native.FfnProblem(**{**fields, **change})


def norm_problem(**change):
    fields = dict(rows=4, width=8, residual_dtype=0, dtype=0, residual=GOOD, branch=GOOD,
                  pre_weight=GOOD, residual_stride=8, branch_stride=8, gate_rows=4,
                  residual_scale=1.0, eps=1e-6)
    return _native.NormProblem(**{**fields, **change})


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), 1), (dict(activation=5), 1), (dict(tokens=-1), 1), (dict(width=0), 1),
    (dict(hidden=0), 1), (dict(out_width=0), 1), (dict(x=None), 1), (dict(w_gate=None), 1),
    (dict(w_up=None), 1), (dict(w_down=None), 1), (dict(x_stride=7), 1),
    (dict(w_down_stride=8), 1), (dict(x=BAD), 2), (dict(w_up=BAD), 2), (dict(b_gate=BAD), 2),
    (dict(width=1 << 23, x_stride=1 << 23, w_gate_stride=1 << 23, w_up_stride=1 << 23), 6),
    (dict(tokens=1 << 40), 6),
])
def test_ffn_refusals(change, code):
    lib, p = _native.library(), ffn_problem(**change)
    grads = _native.FfnGrads()
    assert lib.fhb_ffn_forward(ctypes.byref(p), GOOD, None, GOOD, 1 << 20, None) == code
    assert lib.fhb_ffn_backward(ctypes.byref(p), GOOD, 8, GOOD, ctypes.byref(grads), GOOD,
                                1 << 20, None) == code


def test_ffn_refusals_of_outputs():
    lib, p, grads = _native.library(), ffn_problem(), _native.FfnGrads()
    r = ctypes.byref
    assert lib.fhb_ffn_forward(None, GOOD, None, GOOD, 1 << 20, None) == 1
    assert lib.fhb_ffn_forward(r(p), None, None, GOOD, 1 << 20, None) == 1
    assert lib.fhb_ffn_forward(r(p), BAD, None, GOOD, 1 << 20, None) == 2
    assert lib.fhb_ffn_forward(r(p), GOOD, GOOD + 4, GOOD, 1 << 20, None) == 2
    assert lib.fhb_ffn_forward(r(ffn_problem(tokens=0, x=None)), None, None, None, 0, None) == 0
    assert lib.fhb_ffn_backward(r(p), None, 8, GOOD, r(grads), GOOD, 1 << 20, None) == 1
    assert lib.fhb_ffn_backward(r(p), GOOD, 7, GOOD, r(grads), GOOD, 1 << 20, None) == 1
    assert lib.fhb_ffn_backward(r(p), GOOD, 8, None, r(grads), GOOD, 1 << 20, None) == 1
    assert lib.fhb_ffn_backward(r(p), GOOD, 8, GOOD, None, GOOD, 1 << 20, None) == 1
    bad = _native.FfnGrads(w_up=BAD)
    assert lib.fhb_ffn_backward(r(p), GOOD, 8, GOOD, r(bad), GOOD, 1 << 20, None) == 2
    assert lib.fhb_ffn_saved_bytes(r(p)) > 0
    assert lib.fhb_ffn_saved_bytes(r(ffn_problem(hidden=0))) == 0


@pytest.mark.parametrize("change,code", [
    (dict(dtype=3), 1), (dict(residual_dtype=-1), 1), (dict(residual_dtype=1), 1),
    (dict(rows=-1), 1), (dict(width=0), 1), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(residual=None), 1), (dict(pre_weight=None), 1), (dict(branch=None, gate=GOOD), 1),
    (dict(branch=None, post_weight=GOOD), 1), (dict(gate=GOOD, gate_rows=0), 1),
    (dict(residual_stride=4), 1), (dict(branch_stride=4), 1), (dict(residual=BAD), 2),
    (dict(branch=BAD), 2), (dict(gate=BAD), 2), (dict(residual_scale_ptr=BAD), 2),
    (dict(width=1 << 23, residual_stride=1 << 23, branch_stride=1 << 23), 6),
])
def test_norm_refusals(change, code):
    lib, p, grads = _native.library(), norm_problem(**change), _native.NormGrads()
    r = ctypes.byref
    assert lib.fhb_residual_norm(r(p), GOOD, GOOD, GOOD, None) == code
    assert lib.fhb_residual_norm_backward(r(p), GOOD, 8, GOOD, 8, GOOD, r(grads), GOOD, 1 << 20,
                                          None) == code


def test_norm_refusals_of_outputs():
    lib, p, r = _native.library(), norm_problem(), ctypes.byref
    assert lib.fhb_residual_norm(r(p), GOOD, None, GOOD, None) == 1
    assert lib.fhb_residual_norm(r(p), BAD, GOOD, GOOD, None) == 2
    assert lib.fhb_residual_norm(r(norm_problem(rows=0, residual=None)), None, None, None, None) == 0
    none = _native.NormGrads()
    assert lib.fhb_residual_norm_backward(r(p), GOOD, 8, GOOD, 8, None, r(none), GOOD, 64, None) == 1
    gate = _native.NormGrads(gate=GOOD)  # no gate was given
    assert lib.fhb_residual_norm_backward(r(p), GOOD, 8, GOOD, 8, GOOD, r(gate), GOOD, 64, None) == 1
    assert lib.fhb_residual_norm_backward(r(p), GOOD, 4, GOOD, 8, GOOD, r(none), GOOD, 64, None) == 1


def test_adamw_refusals():
    lib, r = _native.library(), ctypes.byref

    def call(bits=32, n=1, step=GOOD, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, decay=0.0, **change):
        fields = dict(param=GOOD, grad=GOOD, exp_avg=GOOD, exp_avg_sq=GOOD, exp_avg_scale=GOOD,
                      exp_avg_sq_scale=GOOD, count=8, dtype=0)
        t = _native.AdamwTensor(**{**fields, **change})
        return lib.fhb_adamw_step(r(t), n, bits, step, lr, b1, b2, eps, decay, None)

    nan = float("nan")
    for bad in (dict(bits=16), dict(n=-1), dict(step=None), dict(lr=-1.0), dict(lr=nan),
                dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(decay=-1.0), dict(count=-1),
                dict(dtype=7), dict(param=None), dict(grad=None), dict(exp_avg=None),
                dict(bits=8, exp_avg_sq=None), dict(bits=8, exp_avg_scale=None)):
        assert call(**bad) == 1, bad
    for bad in (dict(step=4100), dict(param=BAD), dict(exp_avg=4098), dict(bits=8, exp_avg_scale=4098)):
        assert call(**bad) == 2, bad
    assert lib.fhb_adamw_step(None, 1, 32, GOOD, 1e-3, 0.9, 0.99, 1e-8, 0.0, None) == 1


def test_python_refusals():
    x = torch.zeros(2, 4)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        fused_hoad.gated_feed_forward(x, x, x, x)
    with pytest.raises(RuntimeError, match="activation must be"):
        fused_hoad.gated_feed_forward(x, x, x, x, activation="relu")
    with pytest.raises(RuntimeError, match="residual must be a CUDA tensor"):
        fused_hoad.residual_norm(x, x, x[0])
    with pytest.raises(ValueError, match="needs a branch"):
        fused_hoad.residual_norm(x, None, x[0])
    with pytest.raises(RuntimeError, match="step must be a CUDA int64 tensor"):
        fused_hoad.adamw_step([], [], [], [], torch.zeros(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="same length"):
        fused_hoad.adamw_step([x], [], [], [], torch.zeros(1, dtype=torch.int64))
    w = [torch.nn.Parameter(x)]
    for bad in (dict(state_bits=4), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            fused_hoad.AdamW(w, **bad)
    for bad in (dict(width=0), dict(blocks=0), dict(activation="relu")):
        with pytest.raises(ValueError):
            fused_hoad.GatedResidualTrunk(**bad)


@pytest.mark.gpu
def test_python_refusals_of_shapes_and_types():
    x, w, d = (torch.zeros(s, device="cuda") for s in ((3, 4), (6, 4), (5, 6)))
    ffn = fused_hoad.gated_feed_forward
    for args, message in [
        ((x.half(), w, w, d), "float32 or bfloat16"), ((x, w.bfloat16(), w, d), "type of x"),
        ((x, w[:, :3], w, d), "w_gate must have shape"), ((x, w, w[:5], d), "w_up must have shape"),
        ((x, w, w, d[:, :5]), "w_down must have shape"), ((x, w, w, w.T), None),
        ((x, w, w, d, x[0]), "b_gate must have shape"), ((x, w.cpu(), w, d), "CUDA tensor"),
        ((x[:, :0], w[:, :0], w[:, :0], d), "width of at least 1"),
    ]:
        if message is None:
            ffn(*args)
            continue
        with pytest.raises(RuntimeError, match=message):
            ffn(*args)
    r, c = torch.zeros(2, 3, 4, device="cuda"), torch.ones(4, device="cuda")
    for args, kwargs, message in [
        ((r, r[0], c), {}, "shape of residual"), ((r, r, c[:3]), {}, "pre_weight must have shape"),
        ((r, r.bfloat16(), c), {}, "type of pre_weight"),
        ((r.bfloat16(), r, c), {}, "goes with bfloat16"),
        ((r, r, c), dict(gate=torch.zeros(1, 3, 4, device="cuda")), "gate must have shape"),
        ((r, r, c), dict(gate=torch.zeros(2, 4, device="cuda")), "gate must have shape"),
        ((r, r, c), dict(residual_scale=torch.zeros(1)), "residual_scale must be"),
        ((r, r, c), dict(eps=-1.0), "eps must be"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            fused_hoad.residual_norm(*args, **kwargs)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    for lists, message in [
        (([x], [x[:2]], [x], [x]), "grads"), (([x], [x], [x.bfloat16()], [x]), "exp_avgs"),
        (([x.T], [x], [x], [x]), "params"), (([x.half()], [x], [x], [x]), "float32 or bfloat16"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            fused_hoad.adamw_step(*lists, step)


@pytest.mark.parametrize("activation", ["tanh", "silu"])
def test_reference_gradients_against_differences(activation):
    g = torch.Generator().manual_seed(0)
    shapes = [(5, 3), (7, 3), (7, 3), (4, 7), (7,), (7,), (4,)]
    tensors = [torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in shapes]
    grad = torch.randn(5, 4, generator=g, dtype=torch.float64)
    assert torch.autograd.gradcheck(
        lambda *t: trunk_reference.ffn(*t, activation=activation), tensors)
    auto = torch.autograd.grad(trunk_reference.ffn(*tensors, activation=activation), tensors, grad)
    for a, b in zip(auto, trunk_reference.ffn_gradients(grad, *tensors, activation)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    rows = [torch.randn(4, 6, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2)]
    weights = [torch.randn(6, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(3)]
    scale = torch.tensor([0.7], dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(trunk_reference.norm, (*rows, *weights, scale))


@pytest.mark.gpu
def test_messages_with_numbers():
    """A refusal that names a size is an exception like any other (also the flat Adam's)."""
    p = torch.zeros(8, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="grad must have 8 values"):
        fused_hoad.load_extension().adam_step(p, p[:4], p, p, step, 1e-3, 0.9, 0.999, 1e-8)


@pytest.mark.gpu
def test_differentiable_once():
    """Recording a graph of a backward is refused: it would be cut off there."""
    x, w, d = (torch.randn(s, device="cuda", requires_grad=True) for s in ((3, 8), (16, 8), (8, 16)))
    y = fused_hoad.gated_feed_forward(x, w, w, d)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(y.sum(), x, create_graph=True, retain_graph=True)
    (gradient,) = torch.autograd.grad(y.sum(), x)
    assert not gradient.requires_grad
    scale = torch.ones(8, device="cuda", requires_grad=True)
    total, normed = fused_hoad.residual_norm(x, x, scale)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad((total.sum() + normed.square().sum()), scale, create_graph=True)


@pytest.mark.gpu
def test_inputs_used_twice_and_saved_inputs_changed():
    x, w, d = (torch.randn(s, device="cuda", requires_grad=True) for s in ((5, 8), (16, 8), (8, 16)))
    (twice,) = torch.autograd.grad(fused_hoad.gated_feed_forward(x, w, w, d).sum(), [w])
    v = w.detach().clone().requires_grad_()
    parts = torch.autograd.grad(fused_hoad.gated_feed_forward(x, w, v, d).sum(), [w, v])
    assert torch.allclose(twice, parts[0] + parts[1], rtol=1e-6, atol=1e-6)
    y = fused_hoad.gated_feed_forward(x, w, w, d)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
