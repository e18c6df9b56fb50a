"""Corners of the gated residual trunk's operators."""

from __future__ import annotations

import ctypes
import subprocess
import sys
import threading

import pytest
import torch

import fused_hoad
from fused_hoad import _native
from trunk_reference import assert_near, ffn, ffn_gradients, tolerance

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16]


# ---- the activation's derivative where it saturates ----


def slope_tolerance(g: float, dtype: torch.dtype) -> float:
    """e^{2|g|} is a power of 2 whose exponent 2|g| / ln 2 is rounded (2|g| 2^-24 of the result)
    times a rounded constant (half of that again); the power, the reciprocal and the products add
    less than 16 * 2^-24. bfloat16: the operand's and the result's rounding and one more."""
    return (3 * abs(g) + 16) * 2.0**-24 if dtype == torch.float32 else 3 * 2.0**-9


@pytest.mark.parametrize("dtype", TYPES)
def test_slope_of_saturated_units(dtype):
    """tanh' is even and keeps its digits on both sides: each row and each feature to its own."""
    values = [s * k for k in range(4, 13) for s in (1.0, -1.0)]
    exact = {g: float(torch.cosh(torch.tensor(g, dtype=torch.float64)) ** -2) for g in values}

    def make(*shape, fill):
        return torch.full(shape, fill, device="cuda", dtype=dtype, requires_grad=True)

    # rows: g = x, u = 1, dh = 1, so dx is the sum of 16 equal slopes
    x = torch.tensor(values, device="cuda").view(-1, 1).to(dtype).requires_grad_()
    wg, wu, wd, bu = make(16, 1, fill=1.0), make(16, 1, fill=0.0), make(1, 16, fill=1.0), make(16, fill=1.0)
    y = fused_hoad.gated_feed_forward(x, wg, wu, wd, None, bu, activation="tanh")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for g, got in zip(values, dx.view(-1).tolist()):
        assert abs(got - 16 * exact[g]) <= slope_tolerance(g, dtype) * 16 * exact[g], (g, got)
    # features: 16 of each g, as biases, one token
    bg = torch.tensor(values, device="cuda").repeat_interleave(16).to(dtype).requires_grad_()
    hidden = bg.numel()
    one = make(1, 1, fill=1.0)
    wg, wu, wd, bu = make(hidden, 1, fill=0.0), make(hidden, 1, fill=0.0), make(1, hidden, fill=1.0), \
        make(hidden, fill=1.0)
    y = fused_hoad.gated_feed_forward(one, wg, wu, wd, bg, bu, activation="tanh")
    for grad in torch.autograd.grad(y, [wg, bg], torch.ones_like(y)):
        by_value = grad.view(-1, 16)
        for g, got in zip(values, by_value.double().tolist()):
            for v in got:
                assert abs(v - exact[g]) <= slope_tolerance(g, dtype) * exact[g], (g, v)
        assert torch.equal(by_value[0::2], by_value[1::2])


# ---- batches without rows ----


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,gate_shape", [((2, 0, 48), (2, 1, 48)), ((3, 5, 0, 40), (3, 5, 1, 40)),
                                              ((0, 4, 48), (1, 1, 48)), ((4, 0, 48), (48,))])
def test_gate_gradient_of_no_rows(shape, gate_shape, dtype):
    """Every group's gate has a gradient of zero, whatever was in its memory before."""
    width = shape[-1]
    residual, branch = (torch.zeros(shape, device="cuda", dtype=dtype, requires_grad=True) for _ in range(2))
    weight, gate = (torch.ones(s, device="cuda", dtype=dtype, requires_grad=True) for s in ((width,), gate_shape))
    scale = torch.ones(1, device="cuda", requires_grad=True)
    outs = fused_hoad.residual_norm(residual, branch, weight, weight, gate, scale)
    used = [torch.full((n,), 7.0, device="cuda") for n in (64, 128, 256, 512, 1024) for _ in range(20)]
    del used  # the gradients' memory comes from here
    grads = torch.autograd.grad([o.sum() for o in outs], [weight, gate, scale, residual])
    for g, t in zip(grads, (weight, gate, scale, residual)):
        assert g.shape == t.shape and not g.any()


# ---- parameters that change between a forward and its backward ----


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_step_before_a_backward_is_noticed(bits):
    x, w, d = (torch.randn(s, device="cuda", requires_grad=True) for s in ((5, 8), (16, 8), (8, 16)))
    weight = torch.ones(8, device="cuda", requires_grad=True)
    optimizer = fused_hoad.AdamW([w, d, weight], state_bits=bits)

    def loss():
        return fused_hoad.residual_norm(x, fused_hoad.gated_feed_forward(x, w, w, d), weight)[1].sum()

    loss().backward()
    late = loss()
    versions = [t._version for t in (w, d, weight)]
    optimizer.step()
    assert all(t._version > v for t, v in zip((w, d, weight), versions))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        late.backward()


def test_adamw_step_raises_versions_of_all_it_writes():
    p, g = torch.randn(300, device="cuda"), torch.randn(300, device="cuda")
    codes = [torch.zeros(300, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(2, device="cuda") for _ in range(2)]
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    written = [p, *codes, *scales, step]
    before, of_grad = [t._version for t in written], g._version
    fused_hoad.adamw_step([p], [g], [codes[0]], [codes[1]], step, exp_avg_scales=[scales[0]],
                          exp_avg_sq_scales=[scales[1]])
    assert all(t._version == v + 1 for t, v in zip(written, before)) and g._version == of_grad
    with torch.inference_mode():  # inference tensors have no version
        q, m, v = (torch.zeros(8, device="cuda") for _ in range(3))
        fused_hoad.adamw_step([q], [torch.ones(8, device="cuda")], [m], [v], step)
        assert q.any()


# ---- forward-mode derivatives ----


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as forward

    x, w, d = (torch.randn(s, device="cuda") for s in ((5, 8), (16, 8), (8, 16)))
    c = torch.ones(8, device="cuda")
    ffn_of = fused_hoad.gated_feed_forward
    want, normed = ffn_of(x, w, w, d), fused_hoad.rms_norm(x, c)
    with forward.dual_level():
        dual_x, dual_d, dual_c = (forward.make_dual(t, torch.ones_like(t)) for t in (x, d, c))
        for call in (lambda: ffn_of(dual_x, w, w, d), lambda: ffn_of(x, w, w, dual_d),
                     lambda: ffn_of(x, w, w, d, None, None, dual_c),
                     lambda: fused_hoad.residual_norm(x, dual_x, c),
                     lambda: fused_hoad.residual_norm(x, x, c, gate=dual_c),
                     lambda: fused_hoad.rms_norm(dual_x, c), lambda: fused_hoad.rms_norm(x, dual_c)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # the gradient of a backward would lose its tangent just so
        leaf = x.clone().requires_grad_()
        for y in (ffn_of(leaf, w, w, d), fused_hoad.rms_norm(leaf, c)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, forward.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert torch.equal(ffn_of(x, w, w, d), want)  # no tangents here
        with torch.inference_mode():
            assert torch.equal(fused_hoad.rms_norm(x, c), normed)


# ---- factors next to an infinity ----


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["silu", "tanh"])
def test_an_infinite_unit_keeps_to_its_column(activation, dtype):
    """A feature whose g or u is infinite: the other features' gradients are what they were."""
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens, width, hidden, bad = 40, 32, 48, 21
    x, wg, wu = ((torch.randn(s, generator=g, device="cuda") * 0.5).to(dtype)
                 for s in ((tokens, width), (hidden, width), (hidden, width)))
    wd = torch.randn(width, hidden, generator=g, device="cuda").to(dtype)
    bg, bu = (torch.randn(hidden, generator=g, device="cuda").to(dtype) for _ in range(2))
    grad = torch.randn(tokens, width, generator=g, device="cuda").to(dtype)
    keep = [k for k in range(hidden) if k != bad]
    for which in (bg, bu):
        old = which[bad].clone()
        which[bad] = float("inf")
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd, bg, bu)]
        y = fused_hoad.gated_feed_forward(*leaves, activation=activation)
        got = torch.autograd.grad(y, leaves[1:], grad)
        which[bad] = old
        wide = [t.double() for t in (x, wg, wu, wd, bg, bu)]
        want = ffn_gradients(grad.double(), *wide, None, activation)
        for name, a, b in zip(("w_gate", "w_up", "w_down", "b_gate", "b_up"), got, want[1:]):
            a, b = (a[:, keep], b[:, keep]) if name == "w_down" else (a[keep], b[keep])
            size = torch.full_like(b, float(b.square().mean().sqrt()))
            assert_near(a, b, tolerance(dtype, tokens), f"d_{name}", size)


# ---- FP32 operands whose low bits are all set ----


@pytest.mark.parametrize("value", [1 + 2**-7 - 2**-23, 1 + 2**-8 - 2**-23, 2 - 2**-23,
                                   -(1 + 2**-7 + 2**-15 - 2**-23)])
@pytest.mark.parametrize("activation", ["silu", "tanh"])
def test_operands_with_all_low_bits_set(activation, value):
    """One product a result: what is left out of the products of pieces is not averaged away."""
    tensors = [torch.full(s, value, device="cuda") for s in ((130, 1), (1, 1), (1, 1), (1, 1))]
    grad = torch.full((130, 1), abs(value), device="cuda")
    tol = tolerance(torch.float32, 1)
    wide = [t.double() for t in tensors]
    with torch.no_grad():
        y = fused_hoad.gated_feed_forward(*tensors, activation=activation)
    assert_near(y, ffn(*wide, activation=activation), tol, "y")
    leaves = [t.requires_grad_() for t in tensors]
    y = fused_hoad.gated_feed_forward(*leaves, activation=activation)
    got = torch.autograd.grad(y, leaves, grad)
    want = ffn_gradients(grad.double(), *wide, None, None, None, activation)
    # the sums over the tokens add 130 equal values: their own rounding
    for name, a, b, terms in zip(("x", "w_gate", "w_up", "w_down"), got, want, (2, 130, 130, 130)):
        assert_near(a, b, tolerance(torch.float32, terms), "d_" + name)


def test_operands_at_the_ends_of_the_range():
    """The largest numbers do not round up to infinity in their pieces."""
    largest, least = torch.finfo(torch.float32).max, 2.0**-126
    x = torch.tensor([[largest], [-largest], [largest / 3], [2.0**127], [1.0]], device="cuda").repeat(30, 1)
    wg = torch.tensor([[least]], device="cuda")
    wu, wd = torch.tensor([[0.0]], device="cuda"), torch.tensor([[1.0]], device="cuda")
    bu = torch.tensor([1.0], device="cuda")
    with torch.no_grad():
        y = fused_hoad.gated_feed_forward(x, wg, wu, wd, None, bu, activation="tanh")
    want = ffn(x.double(), wg.double(), wu.double(), wd.double(), None, bu.double(), activation="tanh")
    assert_near(y, want, tolerance(torch.float32, 1), "y")


# ---- sizes asked for by a C caller ----


@pytest.mark.parametrize("change", [dict(gate_rows=0), dict(gate_rows=-1), dict(gate_rows=-(2**62)),
                                    dict(rows=-1), dict(width=0), dict(dtype=7), dict(eps=-1.0)])
def test_workspace_size_of_a_refused_norm(change):
    """0, as the calls' own refusal; a host process that asks is not ended by it."""
    fields = dict(rows=4, width=8, residual_dtype=0, dtype=0, residual=4096, branch=4096,
                  pre_weight=4096, gate=4096, residual_stride=8, branch_stride=8, gate_rows=2,
                  residual_scale=1.0, eps=1e-6)  # addresses that are not read

    def size(**changed):
        problem = _native.NormProblem(**{**fields, **changed})
        return _native.library().fhb_residual_norm_workspace_bytes(ctypes.byref(problem))

    assert size() > 0 and size(**change) == 0


# ---- two host threads ----


def norm_call(width, rows=200):
    """A call of the C ABI on tensors and a stream of its own."""
    stream = torch.cuda.Stream()
    x, b, total, normed = (torch.randn(rows, width, device="cuda") for _ in range(4))
    weight = torch.ones(width, device="cuda")
    torch.cuda.synchronize()
    problem = _native.NormProblem(
        rows=rows, width=width, residual_dtype=0, dtype=0, residual=x.data_ptr(), branch=b.data_ptr(),
        pre_weight=weight.data_ptr(), residual_stride=width, branch_stride=width, gate_rows=rows,
        residual_scale=1.0, eps=1e-6)
    keep = (stream, x, b, total, normed, weight)

    def call():
        return _native.library().fhb_residual_norm(
            ctypes.byref(problem), keep[3].data_ptr(), keep[4].data_ptr(), None, stream.cuda_stream)

    return call


def test_two_threads_with_rows_of_different_bytes():
    """Both calls use one kernel, with 160 and 192 KB of shared memory."""
    failed = []

    def work(call):
        for _ in range(4000):
            code = call()
            if code != 0:
                failed.append(code)

    threads = [threading.Thread(target=work, args=(norm_call(w),)) for w in (5120, 8192, 5120, 8192)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, (len(failed), failed[:3])
    assert fused_hoad.read_device_status(0) == 0


FIRST_CALLS = """
import ctypes, sys, threading
sys.path[:0] = {path!r}
import torch
from fused_hoad import _native

def call(results, k):
    torch.cuda.set_device(0)
    stream = torch.cuda.Stream()
    t = [torch.full(s, 0.5, device="cuda") for s in ((64, 32), (16, 32), (16, 32), (32, 16), (64, 32))]
    p = _native.FfnProblem(tokens=64, width=32, hidden=16, out_width=32, dtype=0, activation=1,
                           x=t[0].data_ptr(), w_gate=t[1].data_ptr(), w_up=t[2].data_ptr(),
                           w_down=t[3].data_ptr(), x_stride=32, w_gate_stride=32, w_up_stride=32,
                           w_down_stride=16)
    torch.cuda.synchronize()
    barrier.wait(60)
    lib = _native.library()
    size = lib.fhb_ffn_workspace_bytes(ctypes.byref(p), 0)
    room = torch.empty(size, device="cuda", dtype=torch.uint8)
    code = lib.fhb_ffn_forward(ctypes.byref(p), t[4].data_ptr(), None, room.data_ptr(), size,
                               stream.cuda_stream)
    torch.cuda.synchronize()
    g = 32 * 0.25
    want = 16 * 0.5 * g * g / (1 + 2.718281828459045 ** -g)
    results[k] = (code, bool(torch.allclose(t[4], torch.full_like(t[4], want), rtol=1e-5)))

barrier, results = threading.Barrier(4), [None] * 4
threads = [threading.Thread(target=call, args=(results, k)) for k in range(4)]
for t in threads: t.start()
for t in threads: t.join()
assert results == [(0, True)] * 4, results
"""


def test_first_calls_of_several_threads():
    """What a product sets up with its first call, in a process of its own."""
    script = FIRST_CALLS.format(path=[p for p in sys.path if p])
    run = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


# ---- waits that give up ----


def test_a_row_that_never_lands():
    """The wait gives up and says so, the copies on their way are waited for, no more are started,
    and the context stays usable."""
    library = _native.library()
    assert fused_hoad.read_device_status(0) == 0
    rows, out = torch.zeros(768, device="cuda"), torch.full((3,), -1.0, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert library.fhb_debug_staged_wait_selftest(rows.data_ptr(), None, stream) == 1
    assert library.fhb_debug_staged_wait_selftest(rows.data_ptr() + 4, out.data_ptr(), stream) == 2
    assert library.fhb_debug_staged_wait_selftest(rows.data_ptr(), out.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    assert out.tolist() == [1.0, float(0b110), 0.0]
    assert fused_hoad.read_device_status(0) == 1  # FHB_STATUS_STAGE_TIMEOUT
    x = torch.randn(700, 2048, device="cuda")
    y = fused_hoad.rms_norm(x, torch.ones(2048, device="cuda"), 0.0)
    assert torch.allclose(y.square().mean(1), torch.ones(700, device="cuda"), rtol=1e-4)
    assert fused_hoad.read_device_status(0) == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_products_wait_for_their_last_copies_and_sums(dtype):
    """Every product ends by waiting for the copies and sums of its last ring slots: a wait on a
    phase that never comes would set the status word and take a second. One CTA a tile and pairs,
    fewer blocks of K than slots and many times more, parts of K, several products a launch."""
    assert fused_hoad.read_device_status(0) == 0
    for tokens, width, hidden in [(9, 8, 8), (100, 64, 64), (130, 72, 40), (300, 1000, 24), (520, 64, 1030),
                                  (2000, 512, 512), (4100, 520, 1100), (33, 4000, 64), (20000, 64, 256)]:
        leaves = [torch.randn(s, device="cuda").to(dtype).requires_grad_()
                  for s in ((tokens, width), (hidden, width), (hidden, width), (width, hidden))]
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        start.record()
        y = fused_hoad.gated_feed_forward(*leaves)
        torch.autograd.grad(y, leaves, torch.ones_like(y))
        end.record()
        end.synchronize()
        assert start.elapsed_time(end) < 500.0, (tokens, width, hidden)
    assert fused_hoad.read_device_status(0) == 0


# ---- a trunk's residual scales ----


@pytest.mark.parametrize("bits", [32, 8])
def test_scales_of_a_bfloat16_trunk_move(bits):
    """Steps of 1e-3 add up next to 1, where bfloat16's own are 2^-8 and 2^-7."""
    torch.manual_seed(0)
    trunk = fused_hoad.GatedResidualTrunk(2, 32, 64, 2).cuda().bfloat16()
    optimizer = fused_hoad.AdamW(trunk.parameters(), lr=1e-3, weight_decay=0.0, state_bits=bits)
    x = torch.rand(500, 2, device="cuda").bfloat16()
    for k in range(3):
        optimizer.zero_grad(set_to_none=True)
        trunk(x).float().square().mean().backward()
        before = [s.detach().clone() for s in trunk.scale]
        assert all(s.grad.dtype == torch.float32 and bool(s.grad) for s in trunk.scale)
        optimizer.step()
        for s, b in zip(trunk.scale, before):
            assert s.dtype == torch.float32 and 0 < float((s - b).abs()) <= 1.1e-3


# ---- memory ----


@pytest.mark.parametrize("dtype", TYPES)
def test_workspaces_hold_what_is_written(dtype):
    """Without gradients a call needs h, and with them nothing that it keeps; the calls stay inside
    what they ask for."""
    tokens, width, hidden = 4096, 256, 1024
    tensors = [torch.randn(s, device="cuda").mul_(0.05).to(dtype)
               for s in ((tokens, width), (hidden, width), (hidden, width), (width, hidden))]
    problem = _native.FfnProblem(
        tokens=tokens, width=width, hidden=hidden, out_width=width, dtype=int(dtype == torch.bfloat16),
        activation=1, x=tensors[0].data_ptr(), w_gate=tensors[1].data_ptr(), w_up=tensors[2].data_ptr(),
        w_down=tensors[3].data_ptr(), x_stride=width, w_gate_stride=width, w_up_stride=width,
        w_down_stride=hidden)
    library, at = _native.library(), ctypes.byref(problem)
    value = 6 if dtype == torch.float32 else 2  # bytes of an operand's value
    packed = 6 * sum(t.numel() for t in tensors) if dtype == torch.float32 else 0
    h = tokens * hidden * value
    plain, saving = (library.fhb_ffn_workspace_bytes(at, k) for k in (0, 2))
    parts = plain - packed - h  # FP32 sums of parts of K, if any
    assert 0 <= parts <= 8 * tokens * width * 4 and saving == plain - h
    assert library.fhb_ffn_workspace_bytes(at, 3) == library.fhb_ffn_workspace_bytes(at, -1) == 0
    with torch.no_grad():
        want = fused_hoad.gated_feed_forward(*tensors)
    stream = torch.cuda.current_stream().cuda_stream
    for size, keeps in ((plain, 0), (saving, library.fhb_ffn_saved_bytes(at))):
        room, saved = (torch.full((n + 4096,), 77, device="cuda", dtype=torch.uint8) for n in (size, keeps))
        y = torch.empty_like(want)
        place = saved.data_ptr() if keeps else None
        assert library.fhb_ffn_forward(at, y.data_ptr(), place, room.data_ptr(), max(size - 1, 0), stream) in (
            (3,) if size else (0,))
        assert library.fhb_ffn_forward(at, y.data_ptr(), place, room.data_ptr(), size, stream) == 0
        assert torch.equal(y, want)
        assert (room[size:] == 77).all() and (saved[keeps:] == 77).all()
    # the same through the call with gradients: its peak is y, what it keeps and the workspace
    leaf = tensors[0].clone().requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    y = fused_hoad.gated_feed_forward(leaf, *tensors[1:])
    grown = torch.cuda.max_memory_allocated() - before
    assert grown <= y.numel() * y.element_size() + library.fhb_ffn_saved_bytes(at) + saving + 2**21


@pytest.mark.parametrize("tokens,width,hidden", [(1, 1024, 8000), (1, 4096, 6000), (1, 4096, 6200),
                                                 (2, 4096, 3000), (2, 4096, 3200), (3, 1024, 512)])
def test_few_tokens_on_both_sides_of_the_dot_products(tokens, width, hidden):
    """bfloat16: the dot products' limit of tokens times weights lies between the sizes."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, wg, wu, wd = ((torch.randn(s, generator=g, device="cuda") * s[-1] ** -0.5).bfloat16()
                     for s in ((tokens, width), (hidden, width), (hidden, width), (width, hidden)))
    x = x * width**0.5
    with torch.no_grad():
        y = fused_hoad.gated_feed_forward(x, wg, wu, wd)
    want = ffn(x.double(), wg.double(), wu.double(), wd.double())
    rms = torch.full_like(want, float(want.square().mean().sqrt()))
    assert_near(y, want, tolerance(torch.bfloat16, hidden), "y", rms)
