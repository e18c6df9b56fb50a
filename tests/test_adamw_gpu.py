"""AdamW over many tensors: 32-bit states against torch.optim.AdamW's formula in 64 bits, 8-bit
states against the coded formula bit for bit, and the optimizer in a training loop."""

from __future__ import annotations

import copy

import pytest
import torch

import fused_hoad

pytestmark = pytest.mark.gpu
BLOCK = 256
SHAPES = [(1,), (7, 9), (256,), (255, 3), (4096, 5), (64, 64), (0, 3), (300000,)]


def normal(shape, std, seed, dtype=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def blocks(t):
    flat = t.reshape(-1)
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def encode(values, square):
    """The documented code, in float32 operations one by one."""
    rows = blocks(values.sqrt() if square else values)
    scale = (rows.abs().amax(1) * (1.0 / 448.0)).clamp(min=2.0**-126)
    units = rows / scale[:, None]
    if square:
        units = torch.where(rows > 0, units.clamp(min=2.0**-9), units)
    codes = units.to(torch.float8_e4m3fn).reshape(-1)[: values.numel()].view(values.shape)
    return codes, scale


def setup(dtypes, bits, shapes=SHAPES):
    params = [normal(s, 0.1, k, dtypes[k % len(dtypes)]) for k, s in enumerate(shapes)]
    ms = [normal(s, 0.01, 100 + k) for k, s in enumerate(shapes)]
    vs = [normal(s, 0.01, 200 + k).square() for k, s in enumerate(shapes)]
    scales = [None, None]
    if bits == 8:
        full = [t for t in range(len(shapes))]
        m_codes = [encode(ms[k], False) if ms[k].numel() else (ms[k].to(torch.float8_e4m3fn), torch.zeros(0, device="cuda")) for k in full]
        v_codes = [encode(vs[k], True) if vs[k].numel() else (vs[k].to(torch.float8_e4m3fn), torch.zeros(0, device="cuda")) for k in full]
        ms, vs = [c for c, _ in m_codes], [c for c, _ in v_codes]
        scales = [[s for _, s in m_codes], [s for _, s in v_codes]]
    return params, ms, vs, scales


def grads_of(params, seed):
    return [normal(p.shape, 0.02, seed + k, p.dtype) for k, p in enumerate(params)]


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,),
                                    (torch.float32, torch.bfloat16)])
def test_32_bit_states(dtypes):
    params, ms, vs, _ = setup(dtypes, 32)
    want = [[t.double() for t in group] for group in (params, ms, vs)]
    step = torch.full((1,), 4, dtype=torch.int64, device="cuda")
    lr, betas, eps, decay = 3e-3, (0.9, 0.98), 1e-7, 0.1
    for t in (5, 6):
        grads = grads_of(params, 10 * t)
        fused_hoad.adamw_step(params, grads, ms, vs, step, lr=lr, betas=betas, eps=eps,
                              weight_decay=decay)
        assert int(step) == t
        for k, g in enumerate(grads):
            p, m, v = (w[k] for w in want)
            m.mul_(betas[0]).add_(g.double(), alpha=1 - betas[0])
            v.mul_(betas[1]).add_(g.double().square(), alpha=1 - betas[1])
            p.mul_(1 - lr * decay)
            p.sub_(lr / (1 - betas[0] ** t) * m / ((v / (1 - betas[1] ** t)).sqrt() + eps))
            # five float32 roundings a step on the moments; the parameters' own rounding
            assert torch.allclose(ms[k].double(), m, rtol=0, atol=10 * 2.0**-24 * 0.1)
            assert torch.allclose(vs[k].double(), v, rtol=10 * 2.0**-24, atol=0)
            # at most sixteen float32 roundings; a bfloat16 parameter has its own
            unit = 2.0**-8 if params[k].dtype == torch.bfloat16 else 2.0**-20
            assert torch.allclose(params[k].double(), p, rtol=unit, atol=unit * 0.05)
            p.copy_(params[k].double())  # a bfloat16 parameter goes on from its rounded value


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16, torch.float32)])
def test_8_bit_states_are_the_coded_formula(dtypes):
    params, ms, vs, (sm, sv) = setup(dtypes, 8)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    for t in (1, 2, 3):
        grads = grads_of(params, 10 * t)
        before = [[x.clone() for x in group] for group in (params, ms, vs, sm, sv)]
        fused_hoad.adamw_step(params, grads, ms, vs, step, lr=1e-2, weight_decay=0.0,
                              exp_avg_scales=sm, exp_avg_sq_scales=sv)
        for k, g in enumerate(grads):
            p0, m0, v0, s0, q0 = (group[k] for group in before)
            if not g.numel():
                continue
            m0, v0 = fused_hoad.decode_states(m0, v0, s0, q0)
            m = m0 * 0.9 + g.float() * (1.0 - 0.9)
            v = v0 * 0.999 + (g.float() * g.float()) * (1.0 - 0.999)
            for (codes, scale), c, s in ((encode(m, False), ms[k], sm[k]),
                                         (encode(v, True), vs[k], sv[k])):
                assert torch.equal(scale, s)
                assert torch.equal(codes.view(torch.uint8), c.view(torch.uint8))
            wanted = p0.double() - 1e-2 / (1 - 0.9**t) * m.double() / (
                (v.double() / (1 - 0.999**t)).sqrt() + 1e-8)
            unit = 2.0**-8 if p0.dtype == torch.bfloat16 else 2.0**-20
            assert torch.allclose(params[k].double(), wanted, rtol=unit, atol=unit * 0.1)


def test_8_bit_zeros_and_ranges():
    """Zero gradients keep zero states; a value far below its block's largest keeps a second
    moment above zero; blocks do not see one another."""
    p = normal((1024,), 0.1, 0)
    g = torch.zeros(1024, device="cuda")
    g[256:512] = 1e-30
    g[300] = 1.0
    g[512:768] = 1e-4
    m, v = (torch.zeros(1024, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2))
    sm, sv = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    old = p.clone()
    fused_hoad.adamw_step([p], [g], [m], [v], step, weight_decay=0.0, exp_avg_scales=[sm],
                          exp_avg_sq_scales=[sv])
    assert torch.equal(p[:256], old[:256]) and torch.equal(p[768:], old[768:])
    _, second = fused_hoad.decode_states(m, v, sm, sv)
    assert not second[:256].any() and not second[768:].any()
    # (1e-30)^2 underflows to zero in float32, so the second moment is exactly zero there
    assert second[300] > 0 and float(second[256:300].max()) == 0.0
    assert torch.allclose(second[512:768], torch.full_like(second[512:768], 1e-8 * 1e-3), rtol=1e-5)
    g[:256] = 1e-15  # its square is a float32: next to 1.0 the code must not fall to zero
    g[0] = 1.0
    fused_hoad.adamw_step([p], [g], [m], [v], step, weight_decay=0.0, exp_avg_scales=[sm],
                          exp_avg_sq_scales=[sv])
    _, second = fused_hoad.decode_states(m, v, sm, sv)
    assert (second[:256] > 0).all()
    assert torch.isfinite(p).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_8_bit_not_finite_stays_in_its_block(value):
    p, g = normal((1000,), 0.1, 0), normal((1000,), 0.1, 1)
    g[600] = value
    m, v = (torch.zeros(1000, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2))
    sm, sv = torch.zeros(4, device="cuda"), torch.zeros(4, device="cuda")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    fused_hoad.adamw_step([p], [g], [m], [v], step, exp_avg_scales=[sm], exp_avg_sq_scales=[sv])
    first, second = fused_hoad.decode_states(m, v, sm, sv)
    block = torch.arange(1000, device="cuda") // 256 == 2
    assert torch.isnan(first[block]).all() and torch.isnan(second[block]).all()
    assert torch.isfinite(first[~block]).all() and torch.isfinite(second[~block]).all()
    assert torch.isfinite(p[~block]).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_unaligned_views(bits):
    """Hundreds of tensors, some of them views at odd offsets, are the same as one by one."""
    shapes = [(1 + 37 * k % 1900,) for k in range(500)]
    params, ms, vs, (sm, sv) = setup((torch.float32, torch.bfloat16), bits, shapes)
    odd = torch.zeros(1901, device="cuda")[1:]
    params[0] = odd
    ms_one, vs_one, params_one, scales_one = (copy.deepcopy(x) for x in (ms, vs, params, [sm, sv]))
    params_one[0] = params[0].clone()
    if bits == 32:
        ms[0], vs[0] = torch.zeros(1901, device="cuda")[1:], torch.zeros(1902, device="cuda")[2:]
    else:
        ms[0], vs[0] = (torch.zeros(1901, device="cuda", dtype=torch.float8_e4m3fn)[1:] for _ in range(2))
        sm[0], sv[0] = torch.zeros(8, device="cuda"), torch.zeros(8, device="cuda")
        scales_one[0][0], scales_one[1][0] = sm[0].clone(), sv[0].clone()
    ms_one[0], vs_one[0] = ms[0].clone(), vs[0].clone()
    grads = grads_of(params, 7)
    step = torch.full((1,), 2, dtype=torch.int64, device="cuda")
    kw = {} if bits == 32 else {"exp_avg_scales": sm, "exp_avg_sq_scales": sv}
    fused_hoad.adamw_step(params, grads, ms, vs, step, **kw)
    assert int(step) == 3
    for k in range(len(params)):
        one = torch.full((1,), 2, dtype=torch.int64, device="cuda")
        kw = {} if bits == 32 else {"exp_avg_scales": [scales_one[0][k]],
                                    "exp_avg_sq_scales": [scales_one[1][k]]}
        fused_hoad.adamw_step([params_one[k]], [grads[k]], [ms_one[k]], [vs_one[k]], one, **kw)
        assert torch.equal(params[k], params_one[k]), k
        assert torch.equal(ms[k].view(torch.uint8), ms_one[k].view(torch.uint8)), k
        assert torch.equal(vs[k].view(torch.uint8), vs_one[k].view(torch.uint8)), k


def test_nothing_to_do_advances_the_step():
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    fused_hoad.adamw_step([], [], [], [], step)
    assert int(step) == 1


def train(optimizer_of, model, points, steps, graph=False):
    want = fused_hoad.manufactured_solution(points).to(points.dtype)
    optimizer = optimizer_of(model.parameters())

    def loss_fn():
        return (model(points) - want).float().square().mean()

    if graph:
        replay = fused_hoad.cuda_graph_step(loss_fn, optimizer)
        for _ in range(steps - 3):
            loss = replay()
    else:
        for _ in range(steps):
            optimizer.zero_grad(set_to_none=True)
            loss = loss_fn()
            loss.backward()
            optimizer.step()
    return float(loss), optimizer


@pytest.mark.parametrize("bits,graph", [(32, False), (8, False), (32, True)])
def test_trunk_learns(bits, graph):
    """The three operators together: a gated residual trunk fits the manufactured solution."""
    torch.manual_seed(0)
    model = fused_hoad.GatedResidualTrunk(2, 64, 128, 3).cuda()
    points = fused_hoad.uniform_points(2048).cuda()
    start = float((model(points) - fused_hoad.manufactured_solution(points)).square().mean())
    loss, optimizer = train(lambda p: fused_hoad.AdamW(p, lr=2e-3, state_bits=bits), model,
                            points, 200, graph)
    assert loss < 0.02 * start, (start, loss)
    # a reloaded optimizer goes on with the same moments
    twin = copy.deepcopy(model)
    other = fused_hoad.AdamW(twin.parameters(), lr=1.0, state_bits=bits)
    other.load_state_dict(optimizer.state_dict())
    for p, q in zip(model.parameters(), twin.parameters()):
        q.grad = p.grad = torch.ones_like(p)
    optimizer.step()
    other.step()
    for p, q in zip(model.parameters(), twin.parameters()):
        assert torch.equal(p, q)


def test_trunk_in_bfloat16_follows_float32():
    torch.manual_seed(0)
    model = fused_hoad.GatedResidualTrunk(2, 64, 128, 3, activation="silu").cuda()
    points = fused_hoad.uniform_points(1000).cuda()
    with torch.no_grad():
        want = model(points)
        got = model.to(torch.bfloat16)(points.to(torch.bfloat16)).float()
    assert float((got - want).norm() / want.norm()) < 0.1


@pytest.mark.parametrize("dtype,bits", [(torch.float32, 32), (torch.bfloat16, 8)])
def test_fit_trunk_example(dtype, bits):
    from fused_hoad.fit_trunk import fit_trunk

    model, before, after, ms = fit_trunk(points=4096, blocks=2, hidden=128, steps=150, dtype=dtype,
                                         state_bits=bits)
    assert after < 0.1 * before and ms > 0
    assert next(model.parameters()).dtype == dtype
    assert fused_hoad.read_device_status(0) == 0
