"""The norms with gate and residual scale against their formulas in 64 bits."""

from __future__ import annotations

import pytest
import torch

import fused_hoad
from trunk_reference import assert_near, norm, norm_sizes, tolerance

pytestmark = pytest.mark.gpu
TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
         (torch.bfloat16, torch.bfloat16)]
NAMES = ("residual", "branch", "pre_weight", "post_weight", "gate", "residual_scale")


def make(shape, types, gate, post, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide, narrow = types
    width = shape[-1]

    def normal(*s, mean=0.0, std=1.0, dtype=narrow):
        return (mean + std * torch.randn(*s, generator=g, device="cuda")).to(dtype)

    gate_shape = {"none": None, "channel": (width,), "full": shape,
                  "sample": (shape[0],) + (1,) * (len(shape) - 2) + (width,)}[gate]
    return [normal(*shape, dtype=wide), normal(*shape, std=0.7), normal(width, mean=1.0, std=0.2),
            normal(width, mean=1.0, std=0.2) if post else None,
            normal(*gate_shape, mean=0.5, std=0.3) if gate_shape else None,
            normal(1, mean=0.9, std=0.1, dtype=torch.float32)], \
        [normal(*shape, mean=0.3, dtype=wide), normal(*shape)]


def check(tensors, upstream):
    given = [k for k, t in enumerate(tensors) if t is not None]
    exact = [None if t is None else t.detach().double().requires_grad_() for t in tensors]
    want = norm(*exact)
    out_sizes, sizes = norm_sizes(*[None if t is None else t.detach() for t in exact],
                                  *[u.double() for u in upstream])
    shape = tensors[0].shape
    rows = max(1, tensors[0].numel() // shape[-1])
    with torch.no_grad():
        plain = fused_hoad.residual_norm(*tensors)
    leaves = [None if t is None else t.detach().requires_grad_() for t in tensors]
    got = fused_hoad.residual_norm(*leaves)
    for outs in (plain, got):
        for o, w, name, k in zip(outs, want, ("total", "normed"), (0, 1)):
            assert o.dtype == tensors[k].dtype
            assert_near(o, w, tolerance(o.dtype, shape[-1]), name, out_sizes[k])
    grads = torch.autograd.grad(got, [leaves[k] for k in given], upstream)
    wanted = torch.autograd.grad(want, [exact[k] for k in given], [u.double() for u in upstream])
    for k, g, w in zip(given, grads, wanted):
        assert g.dtype == tensors[k].dtype and g.shape == tensors[k].shape
        terms = rows * shape[-1] if NAMES[k] == "residual_scale" else max(rows, shape[-1])
        assert_near(g, w, tolerance(g.dtype, terms), "d_" + NAMES[k], sizes[k])


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("rows", [1, 2, 31, 64, 1000])
@pytest.mark.parametrize("width", [1, 2, 7, 32, 64, 65, 128, 201, 512, 777, 2048, 4099, 8192])
def test_sizes(rows, width, types):
    check(*make((rows, width), types, "channel", post=True, seed=width))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "sample", "full"])
@pytest.mark.parametrize("shape", [(3, 37, 64), (16, 70, 96), (40, 5, 33), (700, 1, 40), (5, 3, 2, 24)])
def test_gates(shape, gate, post, types):
    check(*make(shape, types, gate, post, seed=shape[0]))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", [(30000, 64), (4, 3000, 256), (2000, 2056), (70, 20000)])
def test_larger(shape, types):
    check(*make(shape, types, "sample", post=True, seed=1))


@pytest.mark.parametrize("types", TYPES)
def test_strides(types):
    tensors, upstream = make((50, 96), types, "channel", post=True)

    def inside(t, before, after):
        big = torch.full((50, 96 + before + after), float("nan"), device="cuda", dtype=t.dtype)
        view = big[:, before:before + 96]
        view.copy_(t)
        return view

    check([inside(tensors[0], 1, 1), inside(tensors[1], 3, 2), *tensors[2:]],
          [inside(upstream[0], 1, 0), inside(upstream[1], 5, 0)])
    check([inside(tensors[0], 8, 8), inside(tensors[1], 8, 0), *tensors[2:]],
          [inside(upstream[0], 16, 0), upstream[1].T.contiguous().T])
    check([tensors[0].T.contiguous().T, *tensors[1:]], upstream)


@pytest.mark.parametrize("types", TYPES)
def test_one_output_used(types):
    """A gradient through only one of the two outputs."""
    tensors, upstream = make((9, 64), types, "channel", post=True)
    for used in (0, 1):
        leaves = [t.detach().requires_grad_() for t in tensors]
        out = fused_hoad.residual_norm(*leaves)[used]
        grads = torch.autograd.grad(out, leaves, upstream[used], allow_unused=True)
        exact = [t.double().requires_grad_() for t in tensors]
        wanted = torch.autograd.grad(norm(*exact)[used], exact, upstream[used].double(),
                                     allow_unused=True)
        alone = [u.double() if k == used else torch.zeros_like(u).double()
                 for k, u in enumerate(upstream)]
        _, sizes = norm_sizes(*[t.detach() for t in exact], *alone)
        for name, g, w, size in zip(NAMES, grads, wanted, sizes):
            w = torch.zeros_like(g) if w is None else w
            assert_near(g, w, tolerance(g.dtype, 576), "d_" + name, size)


@pytest.mark.parametrize("types", TYPES)
def test_rms_norm(types):
    (x, *_), (grad, _) = make((70, 130), types, "none", post=False)
    weight = torch.linspace(0.5, 1.5, 130, device="cuda").to(types[1])
    leaves = [x.requires_grad_(), weight.requires_grad_()]
    y = fused_hoad.rms_norm(*leaves)
    exact = [t.detach().double().requires_grad_() for t in leaves]
    want = norm(exact[0], None, exact[1])[1]
    assert_near(y, want.detach(), tolerance(types[1], 130), "y")
    grads = torch.autograd.grad(y, leaves, grad.to(types[1]))
    wanted = torch.autograd.grad(want, exact, grad.to(types[1]).double())
    for g, w in zip(grads, wanted):
        assert_near(g, w, tolerance(g.dtype, 130), "gradient")


@pytest.mark.parametrize("types", TYPES)
def test_no_rows_and_empty_rows(types):
    tensors, upstream = make((0, 48), types, "channel", post=True)
    leaves = [t.requires_grad_() for t in tensors]
    out = fused_hoad.residual_norm(*leaves)
    grads = torch.autograd.grad(out, leaves, upstream)
    assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, leaves))
    # rows of zeros: eps alone under the root, nothing divided by zero
    tensors, upstream = make((6, 48), types, "channel", post=True)
    tensors[0][2] = 0
    tensors[1][2] = 0
    tensors[1][4] = 0
    check(tensors, upstream)


def test_number_as_scale_and_repeatability():
    tensors, upstream = make((900, 160), TYPES[1], "sample", post=True)
    leaves = [t.detach().requires_grad_() for t in tensors]
    runs = []
    for _ in range(2):
        out = fused_hoad.residual_norm(*leaves)
        runs.append([*out, *torch.autograd.grad(out, leaves, upstream)])
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    number = fused_hoad.residual_norm(*tensors[:5], float(tensors[5]))
    for a, b in zip(runs[0], number):
        assert torch.equal(a, b)


def test_not_a_number_stays_in_its_row():
    tensors, upstream = make((12, 64), TYPES[0], "full", post=True)
    tensors[1][3, 5] = float("nan")
    tensors[0][7, 1] = float("inf")
    leaves = [t.detach().requires_grad_() for t in tensors]
    out = fused_hoad.residual_norm(*leaves)
    grads = torch.autograd.grad(out, leaves, upstream)
    clean = [r for r in range(12) if r not in (3, 7)]
    for t in (*out, grads[0], grads[1], grads[4]):
        assert torch.isfinite(t[clean]).all()
    assert torch.isnan(out[1][3]).all()


def test_gradient_against_differences():
    """Directional differences in float32 at a step of 2^-6 (see the feed-forward block's)."""
    tensors, upstream = make((20, 40), TYPES[0], "channel", post=True, seed=2)
    leaves = [t.detach().requires_grad_() for t in tensors]
    grads = torch.autograd.grad(fused_hoad.residual_norm(*leaves), leaves, upstream)
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
                out = fused_hoad.residual_norm(*moved)
            ends.append(sum(float((o.double() * u.double()).sum()) for o, u in zip(out, upstream)))
        slope = (ends[0] - ends[1]) / (2 * e)
        assert abs(slope - float((g.double() * v.double()).sum())) <= 5e-3 * float(g.norm()), NAMES[k]
