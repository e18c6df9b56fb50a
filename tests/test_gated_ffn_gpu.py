"""The gated feed-forward block against its formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

import fused_hoad
from trunk_reference import assert_near, ffn, ffn_gradients, ffn_sizes, tolerance

pytestmark = pytest.mark.gpu
NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
TYPES = [torch.float32, torch.bfloat16]


def make(tokens, width, hidden, out, dtype, bias, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    tensors = [normal(tokens, width), normal(hidden, width, std=width**-0.5),
               normal(hidden, width, std=width**-0.5), normal(out, hidden, std=hidden**-0.5)]
    tensors += [normal(hidden, std=0.3), normal(hidden, std=0.3), normal(out, std=0.3)] if bias \
        else [None] * 3
    return tensors, normal(tokens, out)


def wide(tensors):
    return [None if t is None else t.double() for t in tensors]


def check(tensors, grad, activation):
    """Forward without and with gradients, and every gradient, against 64 bits."""
    dtype = tensors[0].dtype
    width, hidden = tensors[1].shape[1], tensors[1].shape[0]
    want = ffn(*wide(tensors), activation)
    tol = tolerance(dtype, max(width, hidden))
    y_size, sizes = ffn_sizes(grad.double(), *wide(tensors), activation)
    with torch.no_grad():
        assert_near(fused_hoad.gated_feed_forward(*tensors, activation), want, tol, "y", y_size)
    leaves = [None if t is None else t.detach().requires_grad_() for t in tensors]
    y = fused_hoad.gated_feed_forward(*leaves, activation)
    assert y.dtype == dtype
    assert_near(y, want, tol, "y with gradients", y_size)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], grad)
    wanted = ffn_gradients(grad.double(), *wide(tensors), activation)
    got = iter(grads)
    rows = max(1, tensors[0].shape[0])
    for name, t, w, size in zip(NAMES, tensors, wanted, sizes):
        if t is None:
            continue
        terms = 2 * hidden if name == "x" else rows
        assert_near(next(got), w, tolerance(dtype, max(terms, width, hidden)), "d_" + name, size)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 2, 7, 8, 9, 16, 17, 33, 64, 127, 128, 129, 257, 1000])
def test_token_counts(tokens, dtype):
    tensors, grad = make(tokens, 96, 160, 96, dtype, bias=False, seed=tokens)
    check(tensors, grad, "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("width,hidden,out", [
    (1, 1, 1), (2, 64, 1), (64, 256, 64), (31, 33, 29), (64, 65, 63), (201, 533, 201),
    (72, 8, 264), (8, 1000, 8), (256, 136, 520), (1032, 64, 24),
])
def test_sizes(width, hidden, out, bias, dtype):
    tensors, grad = make(130, width, hidden, out, dtype, bias, seed=width)
    check(tensors, grad, "tanh" if bias else "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,width,hidden", [
    (1, 1024, 4096), (3, 1023, 2047), (48, 1024, 1408), (300, 512, 1411), (2500, 384, 768),
    (9000, 64, 128),
])
def test_larger(tokens, width, hidden, dtype):
    tensors, grad = make(tokens, width, hidden, width, dtype, bias=True, seed=5)
    check(tensors, grad, "silu")


@pytest.mark.parametrize("dtype", TYPES)
def test_no_tokens(dtype):
    tensors, grad = make(0, 40, 24, 40, dtype, bias=True)
    leaves = [t.requires_grad_() for t in tensors]
    y = fused_hoad.gated_feed_forward(*leaves)
    assert y.shape == (0, 40)
    for t, g in zip(leaves, torch.autograd.grad(y, leaves, grad)):
        assert g.shape == t.shape and not g.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [5, 200])
def test_strides_and_offsets(tokens, dtype):
    """Slices with odd offsets and row strides, transposed weights, leading dimensions."""
    (x, wg, wu, wd, bg, bu, bd), grad = make(tokens, 48, 80, 48, dtype, bias=True)

    def inside(t, before, after):  # the same values as a slice of a larger tensor of NaN
        big = torch.full((t.shape[0], t.shape[1] + before + after), float("nan"), device="cuda",
                         dtype=dtype)
        view = big[:, before:before + t.shape[1]]
        view.copy_(t)
        return view

    both = torch.cat([wg, wu])
    for args, g in [
        ((inside(x, 1, 2), inside(wg, 3, 0), inside(wu, 8, 8), inside(wd, 0, 1)), inside(grad, 5, 6)),
        ((inside(x, 8, 8), *both.chunk(2), wd.T.contiguous().T), inside(grad, 8, 0)),
        ((x.T.contiguous().T, wg.T.contiguous().T, wu, wd), grad.T.contiguous().T),
    ]:
        check([*args, bg, bu, bd], g, "silu")
    deep = x.view(1, tokens, 1, 48).requires_grad_()
    y = fused_hoad.gated_feed_forward(deep, wg, wu, wd, bg, bu, bd)
    assert y.shape == (1, tokens, 1, 48)
    (dx,) = torch.autograd.grad(y.sum(), deep)  # the gradient of a sum is an expanded scalar
    want = ffn_gradients(torch.ones(tokens, 48, device="cuda", dtype=torch.float64),
                         *wide([x, wg, wu, wd, bg, bu, bd]), "silu")[0]
    assert_near(dx.view(tokens, 48), want, tolerance(dtype, 160), "d_x of a sum")


@pytest.mark.parametrize("activation", ["tanh", "silu"])
def test_gradient_against_differences(activation):
    """Directional differences of a float32 call: the truncation error of a step e is e^2 f'''/6
    and the rounding error 2^-22 |f| / e: both below 2e-3 of |f'| at e = 2^-6 for values near 1."""
    tensors, grad = make(40, 24, 56, 24, torch.float32, bias=True, seed=3)
    leaves = [t.detach().requires_grad_() for t in tensors]
    grads = torch.autograd.grad(fused_hoad.gated_feed_forward(*leaves, activation), leaves, grad)
    e = 2.0**-6
    for k, (t, g) in enumerate(zip(tensors, grads)):
        v = torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(k),
                        device="cuda")
        v /= v.norm()
        ends = []
        for sign in (1, -1):
            moved = list(tensors)
            moved[k] = t + sign * e * v
            with torch.no_grad():
                y = fused_hoad.gated_feed_forward(*moved, activation)
            ends.append(float((y.double() * grad.double()).sum()))
        slope = (ends[0] - ends[1]) / (2 * e)
        assert abs(slope - float((g.double() * v.double()).sum())) <= 5e-3 * float(g.norm()), NAMES[k]


@pytest.mark.parametrize("dtype", TYPES)
def test_only_asked_gradients_and_repeatability(dtype):
    tensors, grad = make(700, 64, 200, 64, dtype, bias=True)
    leaves = [t.detach().requires_grad_() for t in tensors]
    full = torch.autograd.grad(fused_hoad.gated_feed_forward(*leaves), leaves, grad)
    again = torch.autograd.grad(fused_hoad.gated_feed_forward(*leaves), leaves, grad)
    for a, b in zip(full, again):
        assert torch.equal(a, b)
    for k in range(7):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate(tensors)]
        (g,) = torch.autograd.grad(fused_hoad.gated_feed_forward(*some), [some[k]], grad)
        assert torch.equal(g, full[k]), NAMES[k]


def test_large_and_extreme_values():
    """Saturated activations, and rows of zeros, tiny and huge values next to ordinary ones."""
    tensors, grad = make(64, 64, 96, 64, torch.float32, bias=True)
    tensors[0][3] = 0.0
    tensors[0][5] *= 1e6
    tensors[0][7] *= 1e-20
    for activation in ("silu", "tanh"):
        with torch.no_grad():
            y = fused_hoad.gated_feed_forward(*tensors, activation)
        want = ffn(*wide(tensors), activation)
        for row in range(64):  # each row to its own size
            assert_near(y[row], want[row], 2 * tolerance(torch.float32, 96), f"row {row}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [2, 150])
def test_not_a_number_stays_in_its_row(tokens, dtype):
    tensors, _ = make(tokens, 64, 64, 64, dtype, bias=False)
    tensors[0][1, 9] = float("nan")
    with torch.no_grad():
        y = fused_hoad.gated_feed_forward(*tensors)
    bad = torch.isnan(y).all(1)
    assert bad[1] and torch.isfinite(y[~bad]).all() and int(bad.sum()) == 1


def test_other_stream_and_graph():
    tensors, _ = make(300, 64, 128, 64, torch.bfloat16, bias=True)
    with torch.no_grad():
        want = fused_hoad.gated_feed_forward(*tensors)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            side = fused_hoad.gated_feed_forward(*tensors)
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(side, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fused_hoad.gated_feed_forward(*tensors)
        tensors[0].mul_(0.5)
        graph.replay()
        assert torch.equal(y, fused_hoad.gated_feed_forward(*tensors))
    assert fused_hoad.read_device_status(0) == 0
